// Writing the 4-bit K/V cache (format: kv4.cuh) and reading whole sequences back.
//
//  * rope_kv4    packed q | k | v rows of a projection: optional RMS norm of the heads of q and k, rotation, q to a dense matrix, k
//                and v in blocks of 32 to their pages
//  * kv4_gather  sequences as dense bf16 rows, for what the attention kernels do not take
//
// Angles are position * frequency in 64 bits (the product is exact up to position 2^29): in 32 bits a position of 100000 would leave
// 8 bits behind the point. Sums of squares are in 64 bits as well, and products of the rotation are rounded one by one, so that
// what a token is held as does not depend on the order of anything. Both are work per angle and per row, not per byte.
#include "kv4.cuh"

namespace b200 {

struct RopeKv4Params {
  const __nv_bfloat16* qkv;        // [tokens][(hq + 2 hkv) d], or null: part
  __nv_bfloat16* q_out;            // [tokens][hq][d]
  uint8_t* pool;
  __nv_bfloat16 *k_out, *v_out;    // [tokens][hkv][d] as the cache holds them, or null
  const int* positions;
  const long long* slots;          // page * page size + offset; < 0: not stored; null: nothing is
  const __nv_bfloat16 *q_norm_w, *k_norm_w;
  const float* inv_freq;           // [rot / 2]
  long long slots_end;             // slots of the pool
  int tokens, hq, hkv, rot, style, page, block_tokens;
  float eps;
  SplitPartials part;
  DeviceStatus* status;
};

constexpr int kRope4Blocks = 4;      // of 256 threads a processor

template <bool kPart>
__device__ __forceinline__ float kv4_input(const RopeKv4Params& p, int t, int feature, int ld) {
  return kPart ? split_sum(p.part, t, feature) : __bfloat162float(p.qkv[static_cast<long long>(t) * ld + feature]);
}

// D / 8 lanes share a row (a head of a token), eight neighbouring values each. A block works out the angles of its tokens once and walks
// rows; blocks along y share a token's rows where tokens are few.
template <int D, bool kPart>
__global__ void __launch_bounds__(256, kRope4Blocks) rope_kv4_kernel(const RopeKv4Params p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kLanes = D / 8;
  extern __shared__ __align__(16) float turns[];     // [block_tokens][2][rot / 2 or a few more] cos, sin
  const int heads = p.hq + 2 * p.hkv, ld = heads * D, half = p.rot >> 1, pitch = (half + 3) & ~3;
  const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.tokens - t0);
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int tt = i / half, j = i - tt * half;
    double s, c;
    sincos(p.positions[t0 + tt] * static_cast<double>(p.inv_freq[j]), &s, &c);
    turns[2 * tt * pitch + j] = static_cast<float>(c);
    turns[(2 * tt + 1) * pitch + j] = static_cast<float>(s);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, u = threadIdx.x & (kLanes - 1), c0 = u * 8;
  const int step = 256 / kLanes * gridDim.y, first = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes;
  const int warp_first = first - lane / kLanes;      // the row of the warp's first lane: every lane makes the same rounds
  // the next row is on its way while one is worked on
  const auto row = [&](int t, int r) {
    return __ldg(reinterpret_cast<const uint4*>(p.qkv + static_cast<long long>(t) * ld + min(first + r, heads - 1) * D + c0));
  };
  uint4 next = make_uint4(0u, 0u, 0u, 0u);
  if (!kPart) next = row(t0, 0);
  for (int tt = 0; tt < nt; ++tt) {
    const int t = t0 + tt;
    const float *cosv = turns + 2 * tt * pitch, *sinv = cosv + pitch;
    const long long slot = p.slots ? p.slots[t] : -1;
    const bool stored = slot >= 0 && slot < p.slots_end;
    if (slot >= p.slots_end && threadIdx.x == 0 && blockIdx.y == 0) report_status(p.status, kBadArgument, kKernelKv4, 1, static_cast<uint32_t>(t));
    for (int r = 0; warp_first + r < heads; r += step) {
      const bool on = first + r < heads;
      const int h = on ? first + r : heads - 1;
      const int kind = h < p.hq ? 0 : h < p.hq + p.hkv ? 1 : 2;
      float v[8];
      if (kPart) {
        split_sum8(p.part, t, h * D + c0, v);
      } else {
        const uint4 raw = next;
        if (warp_first + r + step < heads) next = row(t, r + step);
        else if (tt + 1 < nt) next = row(t + 1, 0);
        const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __bfloat1622float2(b[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
      const __nv_bfloat16* w = kind == 0 ? p.q_norm_w : kind == 1 ? p.k_norm_w : nullptr;
      float rstd = 1.f;
      if (p.q_norm_w || p.k_norm_w) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += static_cast<double>(v[i]) * v[i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w) {
          rstd = static_cast<float>(1.0 / sqrt(ss / D + p.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], rstd), __bfloat162float(w[c0 + i]));
        }
      }
      if (p.rot > 0) {                               // rows of v take part in the exchange, not in the rotation
        if (p.style == 1) {
          if (kind != 2) {
#pragma unroll
            for (int i = 0; i < 8; i += 2)
              if (c0 + i < p.rot) {
                const float a = v[i], b = v[i + 1], fc = cosv[(c0 + i) >> 1], fs = sinv[(c0 + i) >> 1];
                v[i] = __fsub_rn(__fmul_rn(a, fc), __fmul_rn(b, fs));
                v[i + 1] = __fadd_rn(__fmul_rn(b, fc), __fmul_rn(a, fs));
              }
          }
        } else {
          float other[8];
          const bool aligned = (half & 7) == 0;
          if (aligned) {                     // partners are the eight values of another lane of the row
            const int q = c0 < half ? u + (half >> 3) : c0 < p.rot ? u - (half >> 3) : u;
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, v[i], q, kLanes);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int e = c0 + i, q = e < half ? e + half : e - half;
              other[i] = 0.f;
              if (e < p.rot && kind != 2) {
                other[i] = kv4_input<kPart>(p, t, h * D + q, ld);
                if (w) other[i] = __fmul_rn(__fmul_rn(other[i], rstd), __bfloat162float(w[q]));
              }
            }
          }
          if (kind != 2 && c0 < p.rot) {
            if (aligned) {                           // a - b is a + (-b), to the bit
              const bool low = c0 < half;
              const float *fc = cosv + (low ? c0 : c0 - half), *fs = sinv + (low ? c0 : c0 - half);
#pragma unroll
              for (int i = 0; i < 8; i += 4) {
                const float4 c = *reinterpret_cast<const float4*>(fc + i), n = *reinterpret_cast<const float4*>(fs + i);
                const float ca[4] = {c.x, c.y, c.z, c.w}, sa[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float turned = __fmul_rn(other[i + j], sa[j]);
                  v[i + j] = __fadd_rn(__fmul_rn(v[i + j], ca[j]), low ? -turned : turned);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int e = c0 + i;
                if (e >= p.rot) continue;
                const float fc = cosv[e < half ? e : e - half], fs = sinv[e < half ? e : e - half];
                v[i] = e < half ? __fsub_rn(__fmul_rn(v[i], fc), __fmul_rn(other[i], fs)) : __fadd_rn(__fmul_rn(v[i], fc), __fmul_rn(other[i], fs));
              }
            }
          }
        }
      }
      if (on && kind == 0)
        *reinterpret_cast<uint4*>(p.q_out + (static_cast<long long>(t) * p.hq + h) * D + c0) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      if (!__any_sync(0xffffffffu, on && kind != 0)) continue;
      // blocks of 32: four lanes
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      float s;
      const bool val = kind == 2;
      const uint32_t byte = kv4_scale(amax, val ? kKv4ValueExp : kKv4KeyExp, s);
      uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = kv4_code(v[i], s);
      // keys: this lane's pairs are nibbles u % 4 and 4 + u % 4 of the words of the four lane quarters; values: its eight codes are
      // nibble u % 8 of the words of the eight lane groups. The lanes of a block (of 64 values) exchange halves until
      // each has one word.
      uint32_t word[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = 0;
      if (val) {
#pragma unroll
        for (int i = 0; i < 8; ++i) word[i] = code[i] << (4 * (u & 7));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) word[i] = (code[2 * i] | (code[2 * i + 1] << 16)) << (4 * (u & 3));
      }
      {
        uint32_t sum[4];
        const bool hi = (u & 4) != 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, hi ? word[i] : word[4 + i], 4);
          sum[i] = val ? (hi ? word[4 + i] : word[i]) | got : word[i];
        }
        const bool hi2 = (u & 2) != 0;
        uint32_t two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, hi2 ? sum[i] : sum[2 + i], 2);
          two[i] = (hi2 ? sum[2 + i] : sum[i]) | got;
        }
        const bool hi1 = (u & 1) != 0;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, hi1 ? two[0] : two[1], 1);
        word[0] = (hi1 ? two[1] : two[0]) | got;
      }
      if (!on || kind == 0) continue;
      const int hk = h - p.hq - (val ? p.hkv : 0);
      if (stored) {
        const long long page = slot / p.page;
        const int off = static_cast<int>(slot - page * p.page), tok = off & 15;
        uint8_t* plane = p.pool + ((page * p.hkv + hk) * (p.page >> 4) + (off >> 4)) * kv4_unit_bytes(D) + (val ? kv4_plane_bytes(D) : 0);
        int at;                                      // word of the row
        if (val) at = ((u & 7) ^ (D == 128 && (tok & 2) ? 4 : 0)) * (D / 64) + (u >> 3);
        else at = (u & 3) * (D / 32) + (u >> 2);
        *reinterpret_cast<uint32_t*>(plane + tok * (D / 2) + at * 4) = word[0];
        if ((u & 3) == 0) plane[kKv4Unit * (D / 2) + tok * (D / 32) + (u >> 2)] = static_cast<uint8_t>(byte);
      }
      __nv_bfloat16* dense = val ? p.v_out : p.k_out;
      if (dense) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (static_cast<int>(code[i]) - 8) * s;
        *reinterpret_cast<uint4*>(dense + (static_cast<long long>(t) * p.hkv + hk) * D + c0) =
            make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
      }
    }
  }
}

// Four lanes per (token, head): each reads the row's codes whole (16-byte words hold a value of every block, so the lanes take the same
// addresses) and writes every fourth piece of eight values, so that the four write 64 bytes side by side. Two scattered
// 4-byte words a lane and a piece a thread took 118 us where this takes 75 (33000 tokens of 8 heads; 58 at the rate of a plain copy).
template <int D>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const Kv4Pool p, const int* __restrict__ cu_kv, int seqs, int total,
                                                         __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v) {
  pdl_wait();
  pdl_trigger();
  constexpr int kQuads = D / 32;                     // 16-byte words of a row's codes, and pieces of a lane
  const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 2;      // (token, head)
  const int part = threadIdx.x & 3;
  const long long token = row / p.hkv;
  if (token >= total) return;
  const int head = static_cast<int>(row - token * p.hkv);
  int lo = 0, hi = seqs;                             // the last sequence that starts at or before this token
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_kv[mid] <= token) lo = mid; else hi = mid;
  }
  const int pos = static_cast<int>(token - cu_kv[lo]);
  uint4* ko = reinterpret_cast<uint4*>(k + row * D) + part;
  uint4* vo = reinterpret_cast<uint4*>(v + row * D) + part;
  if (pos < 0 || token >= cu_kv[seqs] || pos >= kv4_length(p, pos + 1, kKernelKv4)) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) ko[4 * i] = vo[4 * i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const uint8_t* unit = kv4_unit<D>(p, p.block_table + static_cast<long long>(lo) * p.max_pages, head, pos >> 4, kKernelKv4);
  const int t = pos & 15;
  uint32_t kw[4 * kQuads], vw[4 * kQuads], ks, vs;
  const uint4* kr = reinterpret_cast<const uint4*>(unit + t * (D / 2));
  const uint4* vr = reinterpret_cast<const uint4*>(unit + kv4_plane_bytes(D) + t * (D / 2));
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {
    const uint4 a = __ldg(kr + i), b = __ldg(vr + (D == 128 && (t & 2) ? i ^ 2 : i));
    kw[4 * i] = a.x, kw[4 * i + 1] = a.y, kw[4 * i + 2] = a.z, kw[4 * i + 3] = a.w;
    vw[4 * i] = b.x, vw[4 * i + 1] = b.y, vw[4 * i + 2] = b.z, vw[4 * i + 3] = b.w;
  }
  const uint8_t* scales = unit + kKv4Unit * (D / 2) + t * (D / 32);
  if (D == 128) {
    ks = __ldg(reinterpret_cast<const uint32_t*>(scales));
    vs = __ldg(reinterpret_cast<const uint32_t*>(scales + kv4_plane_bytes(D)));
  } else {
    ks = __ldg(reinterpret_cast<const uint16_t*>(scales));
    vs = __ldg(reinterpret_cast<const uint16_t*>(scales + kv4_plane_bytes(D)));
  }
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {                 // piece 4 i + part, of block i
    uint32_t o[4];
    {
      const __nv_bfloat162 s = kv4_scale_bf16<false>(ks, i), off = kv4_off_bf16(s);
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = kv4_pair_bf16((kw[q * kQuads + i] >> (4 * part)) & 0x000f000fu, s, off);
      ko[4 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    {
      const __nv_bfloat162 s = kv4_scale_bf16<true>(vs, i), off = kv4_off_bf16(s);
      const int shift = 4 * (part + (i & 1) * 4);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t a = vw[2 * g * (D / 64) + (i >> 1)] >> shift, b = vw[(2 * g + 1) * (D / 64) + (i >> 1)] >> shift;
        o[g] = kv4_pair_bf16((a & 15u) | ((b & 15u) << 16), s, off);
      }
      vo[4 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

}  // namespace b200

using namespace b200;

// See the header comment. d 64 or 128, page 16, 32, 64 or 128, rot even and at most d, everything on 16-byte boundaries. A slot
// behind the pool's end is not stored and is reported in the status word.
B200_API int b200_rope_kv4(const void* qkv, void* q_out, void* pool, void* k_out, void* v_out, const int* positions, const long long* slots,
                           const void* q_norm_w, const void* k_norm_w, const float* inv_freq, int tokens, int hq, int hkv, int d, int rot,
                           int style, int page, long long pages, float eps, const float* part_ws, int part_splits,
                           int part_bn, const void* part_bias, void* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (hq < 1 || hkv < 1 || pages < 0 || !kv4_pool_fits(pool, d, page)) return -2;
  if (rot < 0 || rot > d || (rot & 1) || (style != 0 && style != 1) || (rot > 0 && !inv_freq)) return -3;
  uintptr_t all = 0;
  for (const void* x : {qkv, static_cast<const void*>(q_out), static_cast<const void*>(k_out), static_cast<const void*>(v_out), static_cast<const void*>(part_ws), part_bias})
    all |= reinterpret_cast<uintptr_t>(x);
  if (all & 15) return -4;
  if (static_cast<long long>(hq + 2 * hkv) * d >= (1ll << 31)) return -2;
  RopeKv4Params p{};
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.pool = static_cast<uint8_t*>(pool);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.positions = positions;
  p.slots = slots;
  p.q_norm_w = static_cast<const __nv_bfloat16*>(q_norm_w);
  p.k_norm_w = static_cast<const __nv_bfloat16*>(k_norm_w);
  p.inv_freq = inv_freq;
  p.slots_end = pages * page;
  p.tokens = tokens; p.hq = hq; p.hkv = hkv; p.rot = rot; p.style = style; p.page = page;
  p.eps = eps;
  p.part = SplitPartials{part_ws, part_splits, part_bn, static_cast<const __nv_bfloat16*>(part_bias)};
  p.status = static_cast<DeviceStatus*>(status);
  const int rows = 256 / (d / 8), chunks = (hq + 2 * hkv + rows - 1) / rows;
  p.block_tokens = tokens >= 148 * 8 ? 4 : 1;        // more tokens a block once every processor has several
  const dim3 grid((tokens + p.block_tokens - 1) / p.block_tokens, p.block_tokens == 1 ? chunks : 1);
  const size_t smem = static_cast<size_t>(p.block_tokens) * 2 * ((rot / 2 + 3) & ~3) * sizeof(float);
  cudaError_t e;
  if (d == 128) e = part_ws ? launch_pdl(rope_kv4_kernel<128, true>, grid, dim3(256), smem, stream, p) : launch_pdl(rope_kv4_kernel<128, false>, grid, dim3(256), smem, stream, p);
  else e = part_ws ? launch_pdl(rope_kv4_kernel<64, true>, grid, dim3(256), smem, stream, p) : launch_pdl(rope_kv4_kernel<64, false>, grid, dim3(256), smem, stream, p);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}

// k, v [total][hkv][d] bf16: rows cu_kv[s] .. cu_kv[s + 1] are the first tokens of sequence s.
B200_API int b200_kv4_gather(const void* pool, const int* block_table, const int* cu_kv, void* k, void* v, int seqs, int total, int hkv,
                             int d, int page, int max_pages, long long pages, void* status, cudaStream_t stream) {
  if (total <= 0 || seqs <= 0) return 0;
  if (hkv < 1 || max_pages < 1 || pages < 1 || !kv4_pool_fits(pool, d, page)) return -2;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return -4;
  const Kv4Pool p{static_cast<const uint8_t*>(pool), block_table, pages, hkv, max_pages, kv4_unit_shift(page), static_cast<DeviceStatus*>(status)};
  const long long blocks = (static_cast<long long>(total) * hkv * 4 + 255) / 256;
  if (blocks >= (1ll << 31)) return -2;
  const dim3 grid(static_cast<unsigned>(blocks));
  const cudaError_t e = d == 128 ? launch_pdl(kv4_gather_kernel<128>, grid, dim3(256), 0, stream, p, cu_kv, seqs, total, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v))
                                 : launch_pdl(kv4_gather_kernel<64>, grid, dim3(256), 0, stream, p, cu_kv, seqs, total, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v));
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}
