// One query token per sequence over a K/V cache held in 4 bits (format: kv4.cuh).
//
// Bound by the bytes of the cache only as long as a byte costs few instructions: at 6.5 TB/s a processor gets 24 bytes (45 values) a cycle and issues
// four warp instructions in it. So codes are never turned into numbers one by one; the tensor core multiplies registers that are masked words of a row:
//
//   S^T (keys x heads) = K Q^T     A = codes of 16 keys, B = queries, both in half precision: masked with 0x000f000f a word is two
//                                  subnormals code * 2^-24, with 0x00f000f0 two of code * 2^-20 (queries of those places are divided by 16; all
//                                  are times a power of two that keeps a bf16's bits). A block of 32 values has one scale per key: its
//                                  partial sums are multiplied by it in 32 bits. The offset 8 of the codes is in what the sums start from
//   O^T (values x heads) = V^T P^T A = 128 + codes of 16 values of 16 keys (four bits in the mantissa of a bf16 128), B = P^T times the
//                                  keys' scales of that block. The offset is a second product with a constant matrix of -136.
//                                  In bf16, since probabilities times scales have no bound from below: a first token that takes nearly
//                                  all of the weight and has values near zero leaves the rest to probabilities of 2^-24
//
// P^T is S^T after the softmax with its 8 x 8 blocks transposed (movmatrix). Rows of the tile are not the keys in order: row 2 i is key i and
// row 2 i + 1 key 7 - i of eight, which lets every shared-memory read of codes touch each bank once.
//
// Work: a unit is 16 tokens of one kv head. All units of all sequences and heads in a row are cut into equal shares, one per resident
// block, whatever the lengths; a share's first and last sequence may be other blocks' too, whose parts the second kernel
// joins (in the order of the blocks, so results do not depend on timing). Within a share every warp takes each eighth unit and has its own ring of
// bulk copies, so warps meet only where a sequence ends. Short sequences get one block each and no second kernel.
#include "kv4.cuh"
#include "mma_sync.cuh"

namespace b200 {

int num_sms();      // of the current device, see gemm_tcgen05.cu

constexpr int kDec4Warps = 8;
constexpr int kDec4Threads = kDec4Warps * 32;
constexpr int kDec4Stages = 4;
constexpr int kDec4MaxSeqs = 2048;         // of a batch that is cut into shares: their unit counts are in shared memory
constexpr float kDec4Gap = 8.f;            // the reference of the exponentials is raised once a score passes it by this many powers of two
constexpr float kDec4Log2e = 1.4426950408889634f;

struct DecodeKv4Params {
  const __nv_bfloat16* q;      // [sequences][hq][d]
  __nv_bfloat16* out;
  const int* kv_lens;
  Kv4Pool pool;
  float* parts;                // [blocks][2][heads of a chunk][d + 4]: sums, maximum, denominator
  int* prefix;                 // [sequences + 1] units before a sequence, for the second kernel
  int seqs, hq, group, chunks, chunk_heads;      // heads of a group are walked in `chunks` parts
  int window, blocks;
  float scale_log2, cap_in, cap_out;
};

__device__ __forceinline__ uint32_t scaled_bf16x2(uint32_t x, uint32_t s) {
  const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float dec4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Units of a sequence that its query sees, and the first of them.
__device__ __forceinline__ int dec4_units(const DecodeKv4Params& p, int len, int& first) {
  first = p.window > 0 ? max(0, len - p.window) / kKv4Unit : 0;
  return len > 0 ? (len + kKv4Unit - 1) / kKv4Unit - first : 0;
}

// Bytes of dynamic shared memory: rings, the warps' results of one tile of eight heads, the prefix.
__host__ __device__ constexpr int dec4_ring_bytes(int d) { return kDec4Warps * kDec4Stages * kv4_unit_bytes(d); }
__host__ __device__ constexpr int dec4_merge_bytes(int d) { return kDec4Warps * 8 * (d + 4) * 4; }

template <int D, int NT, bool kShares>
__global__ void __launch_bounds__(kDec4Threads, NT == 1 ? 2 : 1) attn_decode_kv4_kernel(const DecodeKv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr uint32_t kValueBias = ((127 - 15 + kKv4ValueExp) << 7) * 0x10001u;
  constexpr int kUnit = kv4_unit_bytes(D), kPlane = kv4_plane_bytes(D), kBlocks = D / 32, kWords = D / 32, kPitch = D + 4;
  __shared__ uint64_t full[kDec4Warps][kDec4Stages];
  __shared__ float merge_ml[kDec4Warps][8][2];
  __shared__ int warp_units[kDec4Warps];
  __shared__ uint32_t abort_word;
  float* merge = reinterpret_cast<float*>(smem + dec4_ring_bytes(D));
  int* prefix = reinterpret_cast<int*>(smem + dec4_ring_bytes(D) + dec4_merge_bytes(D));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  uint8_t* ring = smem + warp * kDec4Stages * kUnit;
  volatile uint32_t* abort_flag = &abort_word;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kDec4Stages; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) abort_word = 0;
  pdl_wait();
  pdl_trigger();
  const int heads_v = p.pool.hkv * p.chunks;         // kv heads, once for every part of their query heads

  // share [f0, f1) of the units in the order (sequence, head, unit)
  long long f0, f1;
  int only_seq = 0, only_units = 0, only_first = 0;
  if (kShares) {
    int run = 0;
    for (int base = 0; base < p.seqs; base += kDec4Threads) {
      const int s = base + threadIdx.x;
      int first, n = s < p.seqs ? dec4_units(p, kv4_length(p.pool, p.kv_lens[s], kKernelKv4), first) : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (lane == 31) warp_units[warp] = sum;
      __syncthreads();
      int before = run;
      for (int w = 0; w < kDec4Warps; ++w) {
        if (w < warp) before += warp_units[w];
        run += warp_units[w];
      }
      if (s < p.seqs) prefix[s] = before + sum - n;
      __syncthreads();
    }
    if (threadIdx.x == 0) prefix[p.seqs] = run;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= p.seqs; i += kDec4Threads) p.prefix[i] = prefix[i];
    const long long total = static_cast<long long>(run) * heads_v;
    f0 = total * blockIdx.x / p.blocks;
    f1 = total * (blockIdx.x + 1) / p.blocks;
  } else {
    only_seq = blockIdx.x / heads_v;
    only_units = dec4_units(p, kv4_length(p.pool, p.kv_lens[only_seq], kKernelKv4), only_first);
    f0 = 0;
    f1 = only_units;
    __syncthreads();
  }
  // (sequence, head, first unit of the share's order and how many) that a unit of the order belongs to
  auto find = [&](long long f, int& s, int& h, long long& at, int& n, int& first) {
    if (kShares) {
      int lo = 0, hi = p.seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<long long>(prefix[mid]) * heads_v <= f) lo = mid; else hi = mid;
      }
      s = lo;
      n = prefix[s + 1] - prefix[s];
      const long long seq_at = static_cast<long long>(prefix[s]) * heads_v;
      h = static_cast<int>((f - seq_at) / n);
      at = seq_at + static_cast<long long>(h) * n;
      dec4_units(p, kv4_length(p.pool, p.kv_lens[s], kKernelKv4), first);
    } else {
      s = only_seq; h = blockIdx.x - only_seq * heads_v; at = 0; n = only_units; first = only_first;
    }
  };
  // units of this warp: f0 + warp + 8 i, i below mine
  const int share = static_cast<int>(f1 - f0);
  const int mine = share > warp ? (share - warp + kDec4Warps - 1) / kDec4Warps : 0;
  const uint8_t* src = nullptr;                      // lane j: address of unit 32 (i / 32) + j of the warp
  auto addresses = [&](int i0) {
    const int i = i0 + lane;
    if (i >= mine) return;
    int s, h, n, first;
    long long at;
    const long long f = f0 + warp + static_cast<long long>(i) * kDec4Warps;
    find(f, s, h, at, n, first);
    src = kv4_unit<D>(p.pool, p.pool.block_table + static_cast<long long>(s) * p.pool.max_pages, h / p.chunks, first + static_cast<int>(f - at), kKernelKv4);
  };
  auto fetch = [&](int i) {
    if (i >= mine) return;
    if ((i & 31) == 0 && i > 0) addresses(i);
    if ((i & 31) == lane) {
      uint64_t* bar = &full[warp][i % kDec4Stages];
      mbar_arrive_expect_tx(bar, kUnit);
      bulk_load(ring + (i % kDec4Stages) * kUnit, src, kUnit, bar);
    }
  };
  addresses(0);
#pragma unroll
  for (int i = 0; i < kDec4Stages; ++i) fetch(i);

  bool ok = true;
  int i = 0;
  long long f = f0;
  bool empty = !kShares && f0 == f1;                 // a sequence without keys: zeros
  while (f < f1 || empty) {
    int s, h, n, first;
    long long at;
    find(f, s, h, at, n, first);
    const long long stop = empty ? f1 : min(at + n, f1);
    const int kv_head = h / p.chunks, head0 = kv_head * p.group + (h - kv_head * p.chunks) * p.chunk_heads;
    const int heads = min(p.chunk_heads, (kv_head + 1) * p.group - head0);
    const int len = empty ? 0 : kv4_length(p.pool, p.kv_lens[s], kKernelKv4);
    const int start = p.window > 0 ? max(0, len - p.window) : 0;

    // queries of heads 8 t + g in half precision, with a power of two taken out so that the largest is in [2^12, 2^13)
    uint32_t qb[NT][D / 16][2];
    float init[NT][kBlocks][2], factor[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const bool on = 8 * t + g < heads;
      const __nv_bfloat16* qh = p.q + (static_cast<long long>(s) * p.hq + head0 + (on ? 8 * t + g : 0)) * D;
      float amax = 0.f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          qb[t][m][r] = on ? *reinterpret_cast<const uint32_t*>(qh + m * 16 + r * 8 + tq * 2) : 0u;
          const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qb[t][m][r]));
          amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = amax > 0.f ? min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 12, -100), 85) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      float sum[kBlocks];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) sum[b] = 0.f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qb[t][m][r]));
          const float sh = r ? down * 0.0625f : down;                   // places 8 .. 15 meet codes times 16
          qb[t][m][r] = pack_f16x2(v.x * sh, v.y * sh);
          const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&qb[t][m][r]));
          sum[m / 2] += (w.x + w.y) * (r ? 16.f : 1.f);
        }
      // what the partial sums start from: -8 * 2^-24 * sum of the block's queries, for the two heads of this lane's results
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        float x = sum[b];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        x *= -4.76837158203125e-7f;
        init[t][b][0] = __shfl_sync(0xffffffffu, x, 8 * tq);
        init[t][b][1] = __shfl_sync(0xffffffffu, x, 8 * tq + 4);
      }
      // codes are times 2^24, scales (as fp32 with bits byte << 20 under an exponent of 96) times 2^(16 + key exponent)
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        factor[t][j] = __shfl_sync(0xffffffffu, up, 8 * tq + 4 * j) * __uint_as_float(static_cast<uint32_t>(127 + 24 + 16 + kKv4KeyExp) << 23);
    }
    float o[NT][D / 16][4], mx[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][m][j] = 0.f;
      mx[t][0] = mx[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }

    for (; ok; ++i) {
      const long long fi = f0 + warp + static_cast<long long>(i) * kDec4Warps;
      if (fi >= stop) break;
      const int slot = i % kDec4Stages;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][slot], (i / kDec4Stages) & 1, abort_flag))) { ok = false; break; }
      const uint8_t* unit = ring + slot * kUnit;
      const int key0 = (first + static_cast<int>(fi - at)) * kKv4Unit;
      const bool whole = key0 >= start && key0 + kKv4Unit <= len;
      const int ka = (g & 1) ? 7 - (g >> 1) : g >> 1;                   // keys of rows g and g + 8: ka, ka + 8
      // ---- scores
      float sc[NT][4];
      {
        uint32_t wa[kWords], wb[kWords], sa, sb;
        if (D == 128) {
          const uint4 a = *reinterpret_cast<const uint4*>(unit + ka * 64 + tq * 16), b = *reinterpret_cast<const uint4*>(unit + (ka + 8) * 64 + tq * 16);
          wa[0] = a.x; wa[1] = a.y; wa[kWords - 2] = a.z; wa[kWords - 1] = a.w;
          wb[0] = b.x; wb[1] = b.y; wb[kWords - 2] = b.z; wb[kWords - 1] = b.w;
          sa = *reinterpret_cast<const uint32_t*>(unit + 8 * D + ka * 4);
          sb = *reinterpret_cast<const uint32_t*>(unit + 8 * D + (ka + 8) * 4);
        } else {
          const uint2 a = *reinterpret_cast<const uint2*>(unit + ka * 32 + tq * 8), b = *reinterpret_cast<const uint2*>(unit + (ka + 8) * 32 + tq * 8);
          wa[0] = a.x; wa[1] = a.y;
          wb[0] = b.x; wb[1] = b.y;
          sa = *reinterpret_cast<const uint16_t*>(unit + 8 * D + ka * 2);
          sb = *reinterpret_cast<const uint16_t*>(unit + 8 * D + (ka + 8) * 2);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const uint32_t xa = wa[b], xb = wb[b], ya = xa >> 8, yb = xb >> 8;
          const uint32_t a0[4] = {xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u};
          const uint32_t a1[4] = {ya & 0x000f000fu, yb & 0x000f000fu, ya & 0x00f000f0u, yb & 0x00f000f0u};
          const float fa = __uint_as_float((((b < 3 ? sa << (20 - 8 * b) : sa >> 4)) & 0x0ff00000u) | 0x30000000u);
          const float fb = __uint_as_float((((b < 3 ? sb << (20 - 8 * b) : sb >> 4)) & 0x0ff00000u) | 0x30000000u);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float acc[4] = {init[t][b][0], init[t][b][1], init[t][b][0], init[t][b][1]};
            mma_f16_16816(acc, a0, qb[t][2 * b][0], qb[t][2 * b][1]);
            mma_f16_16816(acc, a1, qb[t][2 * b + 1][0], qb[t][2 * b + 1][1]);
            sc[t][0] = fmaf(acc[0], fa, sc[t][0]);
            sc[t][1] = fmaf(acc[1], fa, sc[t][1]);
            sc[t][2] = fmaf(acc[2], fb, sc[t][2]);
            sc[t][3] = fmaf(acc[3], fb, sc[t][3]);
          }
        }
      }
      uint32_t pt[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = sc[t][j] * factor[t][j & 1];
          if (p.cap_out == 0.f) {
            sc[t][j] = x * p.scale_log2;
          } else {                                    // cap tanh(x) = cap - 2 cap / (exp(2 x) + 1)
            const float e = dec4_exp2(fminf(x * p.cap_in, 126.f));
            sc[t][j] = p.cap_out - __fdividef(2.f * p.cap_out, e + 1.f);
          }
          if (!whole) {
            const int key = key0 + ka + (j & 2) * 4;
            if (key < start || key >= len) sc[t][j] = -INFINITY;
          }
        }
        const bool over = fmaxf(sc[t][0], sc[t][2]) > mx[t][0] + kDec4Gap || fmaxf(sc[t][1], sc[t][3]) > mx[t][1] + kDec4Gap;
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(sc[t][j], sc[t][2 + j]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (top > mx[t][j]) {
              const float alpha = dec4_exp2(mx[t][j] - top);
              mx[t][j] = top;
              l[t][j] *= alpha;
#pragma unroll
              for (int m = 0; m < D / 16; ++m) {
                o[t][m][j] *= alpha;
                o[t][m][2 + j] *= alpha;
              }
            }
          }
        }
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = dec4_exp2(sc[t][j] - mx[t][j & 1]);
        l[t][0] += e[0] + e[2];
        l[t][1] += e[1] + e[3];
        pt[t][0] = transpose8x8(pack_bf16x2(e[0], e[1]));
        pt[t][1] = transpose8x8(pack_bf16x2(e[2], e[3]));
      }
      // ---- values: keys tq, 7 - tq and the same plus 8
      {
        const uint8_t* vp = unit + kPlane;
        const int r0 = tq, r1 = 7 - tq;
        uint32_t w[4][D / 64], s4[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = (r & 1 ? r1 : r0) + (r >> 1) * 8;
          if (D == 128) {
            const uint2 x = *reinterpret_cast<const uint2*>(vp + row * 64 + ((g ^ ((row & 2) << 1)) << 3));
            w[r][0] = x.x; w[r][D / 64 - 1] = x.y;
            s4[r] = *reinterpret_cast<const uint32_t*>(vp + 8 * D + row * 4);
          } else {
            w[r][0] = *reinterpret_cast<const uint32_t*>(vp + row * 32 + g * 4);
            s4[r] = *reinterpret_cast<const uint16_t*>(vp + 8 * D + row * 2);
          }
        }
        const uint32_t offset[4] = {0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};        // -136
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const uint32_t sel = b == 0 ? 0x4404u : b == 1 ? 0x5414u : b == 2 ? 0x6424u : 0x7434u;
          // scale bytes of a pair of keys on top of the halves, then where a bf16 has them
          const uint32_t p0 = ((__byte_perm(s4[0], s4[1], sel) & 0xff00ff00u) >> 4) + kValueBias, p1 = ((__byte_perm(s4[2], s4[3], sel) & 0xff00ff00u) >> 4) + kValueBias;
          uint32_t a[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) {              // byte j of this block's half of the words: values of two products' rows g and g + 8
              const uint32_t x = __byte_perm(w[2 * r][b / 2], w[2 * r + 1][b / 2], (b & 1 ? 0x7632 : 0x5410) + (j ? 0x0101 : 0));
              a[j][2 * r] = (x & 0x000f000fu) | 0x43004300u;
              a[j][2 * r + 1] = ((x >> 4) & 0x000f000fu) | 0x43004300u;
            }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint32_t b0 = scaled_bf16x2(pt[t][0], p0), b1 = scaled_bf16x2(pt[t][1], p1);
            mma_bf16_16816(o[t][2 * b], offset, b0, b1);
            mma_bf16_16816(o[t][2 * b], a[0], b0, b1);
            mma_bf16_16816(o[t][2 * b + 1], offset, b0, b1);
            mma_bf16_16816(o[t][2 * b + 1], a[1], b0, b1);
          }
        }
      }
      __syncwarp();
      fetch(i + kDec4Stages);
    }

    // ---- join the warps' results, eight heads at a time
    const bool part = kShares && !(at >= f0 && at + n <= f1);
    float* dst_part = kShares ? p.parts + (static_cast<long long>(blockIdx.x) * 2 + (at < f0 ? 0 : 1)) * p.chunk_heads * (D + 4) : nullptr;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[t][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (g == 0) {
          merge_ml[warp][2 * tq + j][0] = mx[t][j];
          merge_ml[warp][2 * tq + j][1] = sum;
        }
      }
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* row = merge + (warp * 8 + 2 * tq + j) * kPitch + m * 16 + g;
          row[0] = o[t][m][j];
          row[8] = o[t][m][2 + j];
        }
      __syncthreads();
      const int hh = threadIdx.x >> 5;                // a head per warp
      if (8 * t + hh < heads) {
        float top = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < kDec4Warps; ++w) top = fmaxf(top, merge_ml[w][hh][0]);
        float wt[kDec4Warps];
#pragma unroll
        for (int w = 0; w < kDec4Warps; ++w) {
          wt[w] = merge_ml[w][hh][0] == top ? 1.f : dec4_exp2(merge_ml[w][hh][0] - top);      // a warp without keys: 0, or all are
          den += wt[w] * merge_ml[w][hh][1];
        }
        for (int c = lane * 4; c < D; c += 128) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kDec4Warps; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(merge + (w * 8 + hh) * kPitch + c);
            acc.x = fmaf(x.x, wt[w], acc.x);
            acc.y = fmaf(x.y, wt[w], acc.y);
            acc.z = fmaf(x.z, wt[w], acc.z);
            acc.w = fmaf(x.w, wt[w], acc.w);
          }
          if (part) {
            *reinterpret_cast<float4*>(dst_part + (8 * t + hh) * (D + 4) + c) = acc;
          } else {
            const float inv = den == 0.f ? 0.f : 1.f / den;
            *reinterpret_cast<uint2*>(p.out + (static_cast<long long>(s) * p.hq + head0 + 8 * t + hh) * D + c) =
                make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          }
        }
        if (part && lane == 0) *reinterpret_cast<float2*>(dst_part + (8 * t + hh) * (D + 4) + D) = make_float2(top, den);
      }
      __syncthreads();
    }
    f = stop;
    empty = false;
  }
  if (!ok) {
    // copies in flight end before the block does
    for (int j = i; j < min(i + kDec4Stages, mine); ++j) mbar_wait(&full[warp][j % kDec4Stages], (j / kDec4Stages) & 1, abort_flag, 1 << 22);
    if (lane == 0) report_status(p.pool.status, kWaitTimeout, kKernelKv4, 43, blockIdx.x);
  }
}

// Joins the parts of sequences that several blocks share; zeros for those without keys. One block per (sequence, part of a kv head's heads),
// one warp per head.
template <int D>
__global__ void __launch_bounds__(256) join_decode_kv4_kernel(const DecodeKv4Params p) {
  pdl_wait();
  pdl_trigger();
  const int heads_v = p.pool.hkv * p.chunks, s = blockIdx.x / heads_v, h = blockIdx.x - s * heads_v;
  const long long total = static_cast<long long>(p.prefix[p.seqs]) * heads_v;
  const int n = p.prefix[s + 1] - p.prefix[s];
  const long long at = static_cast<long long>(p.prefix[s]) * heads_v + static_cast<long long>(h) * n;
  const int kv_head = h / p.chunks, head0 = kv_head * p.group + (h - kv_head * p.chunks) * p.chunk_heads;
  const int heads = min(p.chunk_heads, (kv_head + 1) * p.group - head0);
  // block of unit f: the last whose share starts at or before it
  const int c0 = n > 0 ? static_cast<int>(((at + 1) * p.blocks - 1) / total) : 0, c1 = n > 0 ? static_cast<int>(((at + n) * p.blocks - 1) / total) : 0;
  if (n > 0 && c0 == c1) return;                     // one block had all of it
  const int lane = threadIdx.x & 31;
  for (int hh = threadIdx.x >> 5; hh < heads; hh += 8) {
    __nv_bfloat16* out = p.out + (static_cast<long long>(s) * p.hq + head0 + hh) * D;
    // the first part is the second one of its block: the sequence starts in that share
    auto part = [&](int c) { return p.parts + ((static_cast<long long>(c) * 2 + (c == c0 ? 1 : 0)) * p.chunk_heads + hh) * (D + 4); };
    float top = -INFINITY, den = 0.f;
    if (n > 0) {
      for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, part(c)[D]);
      top = warp_max(top);
    }
    constexpr int kEach = D / 32;                    // values of a lane
    float acc[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) acc[j] = 0.f;
    if (n > 0)
#pragma unroll 4
      for (int c = c0; c <= c1; ++c) {
        const float* x = part(c);
        const float2 ml = *reinterpret_cast<const float2*>(x + D);
        const float w = ml.x == top ? 1.f : dec4_exp2(ml.x - top);
        den = fmaf(w, ml.y, den);
#pragma unroll
        for (int j = 0; j < kEach; j += 2) {
          const float2 v = *reinterpret_cast<const float2*>(x + lane * kEach + j);
          acc[j] = fmaf(w, v.x, acc[j]);
          acc[j + 1] = fmaf(w, v.y, acc[j + 1]);
        }
      }
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int j = 0; j < kEach; j += 2) *reinterpret_cast<uint32_t*>(out + lane * kEach + j) = pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
  }
}

// How a batch is cut: blocks of the first kernel, 0 for one block per sequence and head.
static int dec4_blocks(int seqs, int heads_v, int chunk_heads, int max_kv_len) {
  const long long units = (static_cast<long long>(max_kv_len) + kKv4Unit - 1) / kKv4Unit, pairs = static_cast<long long>(seqs) * heads_v;
  if (units <= 4 * kDec4Warps || seqs > kDec4MaxSeqs) return 0;
  const long long room = (chunk_heads > 8 ? 1ll : 2ll) * num_sms(), shares = (pairs * units + 2 * kDec4Warps - 1) / (2 * kDec4Warps);
  return static_cast<int>(shares < room ? shares : room);
}
static void dec4_chunks(int group, int& chunks, int& heads) {
  chunks = (group + 15) / 16;
  heads = (group + chunks - 1) / chunks;
}

}  // namespace b200

using namespace b200;

// Bytes of workspace for these sizes (0: none is used).
B200_API long long b200_attn_decode_kv4_workspace(int seqs, int hq, int hkv, int d, int max_kv_len) {
  if (seqs <= 0 || hkv < 1 || hq < hkv || hq % hkv) return 0;
  int chunks, heads;
  dec4_chunks(hq / hkv, chunks, heads);
  const int blocks = dec4_blocks(seqs, hkv * chunks, heads, max_kv_len);
  return blocks == 0 ? 0 : static_cast<long long>(blocks) * 2 * heads * (d + 4) * 4 + (seqs + 1ll) * 4;
}

// q, out [sequences][hq][d] bf16. window > 0: the last `window` keys. max_kv_len chooses how the work is cut, nothing else; the workspace
// (16-byte aligned) is of the size that b200_attn_decode_kv4_workspace gives for the same sizes. Returns the number of launches.
B200_API int b200_attn_decode_kv4(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, int seqs, int hq,
                                  int hkv, int d, int page, int max_pages, long long pages, int max_kv_len, int window, float scale,
                                  float softcap, void* workspace, long long workspace_bytes, void* status, cudaStream_t stream) {
  if (seqs <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || max_pages < 1 || pages < 1 || !kv4_pool_fits(pool, d, page)) return -2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) return -4;
  DecodeKv4Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.kv_lens = kv_lens;
  p.pool = Kv4Pool{static_cast<const uint8_t*>(pool), block_table, pages, hkv, max_pages, kv4_unit_shift(page), static_cast<DeviceStatus*>(status)};
  p.seqs = seqs; p.hq = hq; p.group = hq / hkv;
  dec4_chunks(p.group, p.chunks, p.chunk_heads);
  p.window = window;
  p.scale_log2 = scale * kDec4Log2e;
  if (softcap > 0.f) {
    p.cap_in = 2.f * kDec4Log2e * scale / softcap;
    p.cap_out = softcap * kDec4Log2e;
  }
  const long long pairs = static_cast<long long>(seqs) * hkv * p.chunks;
  if (pairs >= (1ll << 31)) return -3;
  if (window > 0 && window < max_kv_len) max_kv_len = window + kKv4Unit;
  p.blocks = dec4_blocks(seqs, hkv * p.chunks, p.chunk_heads, max_kv_len);
  const bool shares = p.blocks > 0;
  if (shares) {
    const long long floats = static_cast<long long>(p.blocks) * 2 * p.chunk_heads * (d + 4);
    if (!workspace || workspace_bytes < floats * 4 + (seqs + 1ll) * 4) return -5;
    p.parts = static_cast<float*>(workspace);
    p.prefix = reinterpret_cast<int*>(p.parts + floats);
  }
  const int fixed = dec4_ring_bytes(d) + dec4_merge_bytes(d), smem = fixed + (shares ? (seqs + 1) * 4 : 0);
  static PerDeviceOnce once[8];
  auto go = [&](auto kernel, PerDeviceOnce& o) -> cudaError_t {
    if (o.first_time()) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed + (kDec4MaxSeqs + 1) * 4);
      if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(static_cast<unsigned>(shares ? p.blocks : pairs)), dim3(kDec4Threads), smem, stream, p);
  };
  const bool two = p.chunk_heads > 8;
  cudaError_t e;
  if (d == 128) {
    if (shares) e = two ? go(attn_decode_kv4_kernel<128, 2, true>, once[0]) : go(attn_decode_kv4_kernel<128, 1, true>, once[1]);
    else e = two ? go(attn_decode_kv4_kernel<128, 2, false>, once[2]) : go(attn_decode_kv4_kernel<128, 1, false>, once[3]);
  } else {
    if (shares) e = two ? go(attn_decode_kv4_kernel<64, 2, true>, once[4]) : go(attn_decode_kv4_kernel<64, 1, true>, once[5]);
    else e = two ? go(attn_decode_kv4_kernel<64, 2, false>, once[6]) : go(attn_decode_kv4_kernel<64, 1, false>, once[7]);
  }
  if (e != cudaSuccess) return -static_cast<int>(e) - 300;
  if (!shares) return 1;
  e = d == 128 ? launch_pdl(join_decode_kv4_kernel<128>, dim3(static_cast<unsigned>(pairs)), dim3(256), 0, stream, p)
               : launch_pdl(join_decode_kv4_kernel<64>, dim3(static_cast<unsigned>(pairs)), dim3(256), 0, stream, p);
  return e == cudaSuccess ? 2 : -static_cast<int>(e) - 400;
}
