// Keys and values held in 4 bits: the format of a pool, and what turns its bytes into numbers.
//
// A layer's pool is uint8 [pages][kv heads][page / 16][2][16 * (d / 2 + d / 32)], d 64 or 128. A unit is 16 tokens of one head: a plane of
// keys and one of values (17 d bytes in all, contiguous, a multiple of 64), each 16 rows of d / 2 bytes of codes and then 16 rows of
// d / 32 scales. A token's bytes hold nothing of another token, so tokens are stored in any order and at once.
//
//   value = (code - 8) * s          code 1 .. 15, one s for 32 neighbouring values
//   s     = half(byte << 7) * 2^e   e -6 for keys, -10 for values; byte 8 .. 247, so never subnormal and never infinite
//
// s is max|x| / 7 with three bits of mantissa kept (nearest, ties to even): a product code * s has at most 7 bits and is exact in
// bf16. Codes of four bits with a scale per 32 values keep 2% of the variance of normal values as noise (code rounding 0.3 s, s = 0.3 sigma).
//
// The nibbles of a row lie as the matrix instruction m16n8k16 wants them: a lane's registers are words of the row, masked. Keys: word
// (lane quarter q = c % 8 / 2, block b = c / 32) holds the eight values of its block that lanes with lane % 4 = q multiply;
// nibble (c % 32 / 8) + 4 (c % 2), so that a mask 0x000f000f leaves two neighbours. Values: word (lane group g = c % 8, u = c / 64), nibble
// c % 64 / 8. A row of 128 values has the halves of its lane groups exchanged for tokens with bit 1 set, which puts the rows
// that a warp reads at once in different banks.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kKv4Unit = 16;                              // tokens
constexpr int kKv4KeyExp = -6, kKv4ValueExp = -10;
__host__ __device__ constexpr int kv4_plane_bytes(int d) { return kKv4Unit * (d / 2 + d / 32); }
__host__ __device__ constexpr int kv4_unit_bytes(int d) { return 2 * kv4_plane_bytes(d); }

constexpr int kKv4MaxSeqs = 256;          // of a batch whose key axis is cut into equal shares: their unit counts are in shared memory

// The pool of one layer and where sequences lie in it.
struct Kv4Pool {
  const uint8_t* base;
  const int* block_table;      // [sequences][max_pages]
  long long pages;             // in the pool; entries outside it are reported and read as page 0
  int hkv, max_pages;
  int unit_shift;              // log2(units of a page)
  DeviceStatus* status;
};
// Unit `u` (16 tokens) of a sequence, for one kv head.
template <int D>
__device__ __forceinline__ const uint8_t* kv4_unit(const Kv4Pool& p, const int* table, int kv_head, int u, uint32_t kernel) {
  int page = table[u >> p.unit_shift];
  if (page < 0 || page >= p.pages) {
    report_status(p.status, kBadArgument, kernel, 41, static_cast<uint32_t>(page));
    page = 0;
  }
  const long long units = ((static_cast<long long>(page) * p.hkv + kv_head) << p.unit_shift) + (u & ((1 << p.unit_shift) - 1));
  return p.base + units * kv4_unit_bytes(D);
}
// Tokens of a sequence that its row of the block table can name.
__device__ __forceinline__ int kv4_length(const Kv4Pool& p, int len, uint32_t kernel) {
  const long long most = (static_cast<long long>(p.max_pages) << p.unit_shift) * kKv4Unit;
  if (len > most) {
    report_status(p.status, kBadArgument, kernel, 42, static_cast<uint32_t>(len));
    return static_cast<int>(most);
  }
  return len;
}

// First of the last `window` keys (at least one) below key `end`. Where queries outnumber keys `end` may be below 0, from which a window near
// 2^31 must not be taken off.
__device__ __forceinline__ int kv4_window_start(int end, int window) { return end > window ? end - window : 0; }

// Exponent of a capped score, cut where exp2 would overflow. A NaN stays one, which fminf would turn into the cut.
__device__ __forceinline__ float kv4_cut(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(126.f));
  return y;
}

// ---- numbers to bytes ---------------------------------------------------------------------------
// Scale byte of a block whose largest magnitude is amax, and the scale.
__device__ __forceinline__ uint32_t kv4_scale(float amax, int exp, float& s) {
  const float f = __fdiv_rn(amax, 7.f) * __uint_as_float(static_cast<uint32_t>(127 - exp) << 23);
  const uint32_t bits = __float_as_uint(f);
  // ties to even at three bits of mantissa; the exponent's bias goes from 127 to 15
  const int b = static_cast<int>((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20) - (112 << 3);
  const uint32_t byte = static_cast<uint32_t>(min(max(b, 8), 247));
  s = __uint_as_float((byte + ((112u + exp) << 3)) << 20);
  return byte;
}
// Code of a value: NaN is 8, as zero is.
__device__ __forceinline__ uint32_t kv4_code(float x, float s) {
  return static_cast<uint32_t>(min(max(__float2int_rn(__fdiv_rn(x, s)), -7), 7) + 8);
}

// ---- bytes to numbers, bf16 (exact) ----------------------------------------------------------------
// Scale byte i of a word as a bf16 pair.
template <bool kValues>
__device__ __forceinline__ __nv_bfloat162 kv4_scale_bf16(uint32_t word, int i) {
  constexpr uint32_t kBias = (127 - 15 + (kValues ? kKv4ValueExp : kKv4KeyExp)) << 7;
  const uint32_t b = (((word >> (8 * i)) & 0xffu) << 4) + kBias;
  const uint32_t both = b | (b << 16);
  return *reinterpret_cast<const __nv_bfloat162*>(&both);
}
// Two codes in the low four bits of the halves of x (other bits zero) times a scale: 128 + code is a bf16, and with
// off = -136 s the fused multiply-add has an exact result.
__device__ __forceinline__ uint32_t kv4_pair_bf16(uint32_t x, __nv_bfloat162 s, __nv_bfloat162 off) {
  const uint32_t biased = x | 0x43004300u;
  const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&biased), s, off);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 kv4_off_bf16(__nv_bfloat162 s) { return __hmul2(s, __float2bfloat162_rn(-136.f)); }

// One row as 16-byte pieces of eight bf16 values: put(piece, values). w: the row's d / 8 words in the order of memory (with the
// halves of 128 values put right); scales: its d / 32 bytes.
template <int D, typename Put>
__device__ __forceinline__ void kv4_key_row(const uint32_t (&w)[D / 8], uint32_t scales, Put put) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b) {
    const __nv_bfloat162 s = kv4_scale_bf16<false>(scales, b), off = kv4_off_bf16(s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = kv4_pair_bf16((w[q * (D / 32) + b] >> (4 * j)) & 0x000f000fu, s, off);
      put(4 * b + j, make_uint4(v[0], v[1], v[2], v[3]));
    }
  }
}
template <int D, typename Put>
__device__ __forceinline__ void kv4_value_row(const uint32_t (&w)[D / 8], uint32_t scales, Put put) {
#pragma unroll
  for (int u = 0; u < D / 64; ++u)
#pragma unroll
    for (int half = 0; half < 2; ++half) {      // nibbles 0 .. 3 and 4 .. 7: one block of 32 values each
      const __nv_bfloat162 s = kv4_scale_bf16<true>(scales, 2 * u + half), off = kv4_off_bf16(s);
      uint32_t m[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) m[g] = __byte_perm(w[2 * g * (D / 64) + u], w[(2 * g + 1) * (D / 64) + u], half ? 0x7632 : 0x5410);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t v[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) v[g] = kv4_pair_bf16((m[g] >> (4 * j)) & 0x000f000fu, s, off);
        put(8 * u + 4 * half + j, make_uint4(v[0], v[1], v[2], v[3]));
      }
    }
}
// Token `t` (0 .. 15) of a plane: its words and scales.
template <int D>
__device__ __forceinline__ void kv4_load_row(const uint8_t* plane, int t, bool values, uint32_t (&w)[D / 8], uint32_t& scales) {
  const int turn = D == 128 && values && (t & 2) ? 2 : 0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(plane + t * (D / 2) + (i ^ turn) * 16));
    w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
  }
  const uint8_t* sc = plane + kKv4Unit * (D / 2) + t * (D / 32);
  if (D == 128) scales = __ldg(reinterpret_cast<const unsigned int*>(sc));
  else scales = __ldg(reinterpret_cast<const unsigned short*>(sc));
}

// Host: what an entry point takes, or a negative code.
inline int kv4_unit_shift(int page) { return page == 16 ? 0 : page == 32 ? 1 : page == 64 ? 2 : page == 128 ? 3 : -1; }
inline bool kv4_pool_fits(const void* pool, int d, int page) {
  return (d == 64 || d == 128) && kv4_unit_shift(page) >= 0 && (reinterpret_cast<uintptr_t>(pool) & 15) == 0;
}

}  // namespace b200
