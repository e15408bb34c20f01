// Rotary positions on several axes: every pair of a head's channels turns by the position of one axis (time, row, column of a
// picture or film), next to the RMS norm of the heads of q and k ahead of it and the store of k and v behind it.
//
//   angle(t, j) = positions[axes[j]][t] * inv_freq[j]         (a, b) -> (a cos - b sin, b cos + a sin)
//
// Angles are the tokens', not the heads': a block works out those of its tokens once, as whole and broken turns in 64 bits, since a position of
// 100000 would leave 32 bits 7 bits behind the point; what is left of the turn, at most half of it, goes through the 32-bit functions.
#include "common.cuh"

namespace b200 {

int num_sms();      // of the current device, see gemm_tcgen05.cu

struct RopeAxesParams {
  const __nv_bfloat16* qkv;        // [tokens][(hq + 2 hkv) d]
  __nv_bfloat16* q_out;            // [tokens][hq][d]
  __nv_bfloat16 *k_cache, *v_cache;  // [pages][hkv][page][d], or null
  __nv_bfloat16 *k_out, *v_out;    // [tokens][hkv][d], or null
  const int* positions;            // [n_axes][tokens]
  const int* axes;                 // [rot / 2]
  const float* inv_freq;           // [rot / 2]
  const long long* slots;          // page * page size + offset; < 0: not stored; null: nothing is
  const __nv_bfloat16 *q_norm_w, *k_norm_w;
  long long slots_end;             // slots of the pool
  int tokens, n_axes, hq, hkv, d, rot, style, page, block_tokens;
  float eps;
  DeviceStatus* status;
};

__device__ __forceinline__ float2 axes_turn(const RopeAxesParams& p, int t, int j) {
  const int a = p.axes[j];
  if (static_cast<unsigned>(a) >= static_cast<unsigned>(p.n_axes)) {
    report_status(p.status, kBadArgument, kKernelRopeAxes, 1, static_cast<uint32_t>(j));
    return make_float2(1.f, 0.f);
  }
  const double turns = p.positions[static_cast<long long>(a) * p.tokens + t] * static_cast<double>(p.inv_freq[j]) * 0.15915494309189533577;
  float s, c;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c, s);
}

// Row of token t in a cache of one head's pages, -1: not stored.
__device__ __forceinline__ long long axes_row(const RopeAxesParams& p, int t, bool tell) {
  const long long slot = p.slots ? p.slots[t] : -1;
  if (slot < 0) return -1;
  if (slot >= p.slots_end) {
    if (tell) report_status(p.status, kBadArgument, kKernelRopeAxes, 2, static_cast<uint32_t>(t));
    return -1;
  }
  return slot / p.page * p.hkv * p.page + slot % p.page;
}

template <int V>
struct AxesVec;
template <>
struct AxesVec<8> { using T = uint4; };
template <>
struct AxesVec<4> { using T = uint2; };

template <int V>
__device__ __forceinline__ void axes_store(__nv_bfloat16* dst, const float (&v)[V]) {
  typename AxesVec<V>::T raw;
  uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<typename AxesVec<V>::T*>(dst) = raw;
}

template <int V>
__device__ __forceinline__ void axes_unpack(const typename AxesVec<V>::T& raw, float (&v)[V]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// `lanes` lanes share a head (as many as it has units of work; a power of two of them where a norm's sum is exchanged), two vectors of V neighbouring
// values each: with split halves the two that turn together, else neighbours (what lies behind the rotated part always so). A thread keeps its place
// in the head and walks the heads of a few tokens, the next vectors on their way while some are turned, the first ones while the angles are worked out.
// 8192 tokens of 32 + 16 heads of 128 with norms: 48.1 us, bound by instructions (issued in 75 % of the cycles; 4.2 TB/s). With a division per vector and norm
// weights loaded one by one 56.6; without the sines 46.2. Of 4900 patches, 48 heads of 80, nothing stored: 15.5 us (4.8 TB/s).
template <int V>
__global__ void __launch_bounds__(256, 4) rope_axes_kernel(const RopeAxesParams p, int lanes) {
  using Vec = typename AxesVec<V>::T;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) float axes_table[];      // [block_tokens][cos of rot / 2, then sin; each part padded to 4], norm weights of q, of k
  __shared__ long long cache_row[8];
  const int heads = p.hq + 2 * p.hkv, half = p.rot >> 1, pitch = (half + 3) & ~3;
  const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.tokens - t0);
  const int units = p.d / (2 * V), split = half / V;       // units whose two vectors turn together
  const int each = 256 / lanes, mine = threadIdx.x / lanes, u = threadIdx.x - mine * lanes;
  const int h0 = blockIdx.y * each + mine, step = each * gridDim.y, rounds = (heads - static_cast<int>(blockIdx.y) * each + step - 1) / step;
  const bool on = mine < each && u < units, turns = on && u * V < half, norms = p.q_norm_w || p.k_norm_w;
  const int at = min(u, units - 1), ca = (p.style == 0 && at < split ? at : 2 * at) * V, cb = p.style == 0 && at < split ? ca + half : ca + V;
  const __nv_bfloat16* src = p.qkv + (static_cast<long long>(t0) * heads + min(h0, heads - 1)) * p.d;
  Vec na = __ldg(reinterpret_cast<const Vec*>(src + ca)), nb = __ldg(reinterpret_cast<const Vec*>(src + cb));
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, j = i - t * half;
    const float2 cs = axes_turn(p, t0 + t, j);
    axes_table[2 * t * pitch + j] = cs.x;
    axes_table[(2 * t + 1) * pitch + j] = cs.y;
  }
  float* const weights = axes_table + 2 * p.block_tokens * pitch;
  if (norms)
    for (int i = threadIdx.x; i < 2 * p.d; i += 256) {
      const __nv_bfloat16* w = i < p.d ? p.q_norm_w : p.k_norm_w;
      weights[i] = w ? __bfloat162float(w[i < p.d ? i : i - p.d]) : 0.f;
    }
  if (threadIdx.x < nt) cache_row[threadIdx.x] = axes_row(p, t0 + threadIdx.x, blockIdx.y == 0);
  __syncthreads();
  const auto floats = [](const float* from, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(from + i);
      v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
    }
  };
  for (int tt = 0; tt < nt; ++tt) {
    const int t = t0 + tt;
    const float* cosv = axes_table + 2 * tt * pitch + u * V;
    const long long stored = cache_row[tt];
    for (int r = 0, h = h0; r < rounds; ++r, h += step) {
      const int kind = h < p.hq ? 0 : (h < p.hq + p.hkv ? 1 : 2);
      float a[V], b[V];
      axes_unpack<V>(na, a);
      axes_unpack<V>(nb, b);
      if (r + 1 < rounds || tt + 1 < nt) {
        const bool same = r + 1 < rounds;
        src = p.qkv + (static_cast<long long>(same ? t : t + 1) * heads + min(same ? h + step : h0, heads - 1)) * p.d;
        na = __ldg(reinterpret_cast<const Vec*>(src + ca));
        nb = __ldg(reinterpret_cast<const Vec*>(src + cb));
      }
      if (norms) {
        float ss = 0.f;
        if (on) {
#pragma unroll
          for (int i = 0; i < V; ++i) ss += a[i] * a[i] + b[i] * b[i];
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (kind == 0 ? p.q_norm_w != nullptr : kind == 1 && p.k_norm_w) {
          const float rstd = rsqrtf(ss / p.d + p.eps);
          const float* nw = weights + kind * p.d;
          float w[V];
          floats(nw + ca, w);
#pragma unroll
          for (int i = 0; i < V; ++i) a[i] = a[i] * rstd * w[i];
          floats(nw + cb, w);
#pragma unroll
          for (int i = 0; i < V; ++i) b[i] = b[i] * rstd * w[i];
        }
      }
      if (turns && kind != 2) {
        float cs[V], sn[V];
        if ((u + 1) * V <= half && (half & 3) == 0) {
          floats(cosv, cs);
          floats(cosv + pitch, sn);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const bool real = u * V + i < half;
            cs[i] = real ? cosv[i] : 1.f;
            sn[i] = real ? cosv[pitch + i] : 0.f;
          }
        }
        if (p.style == 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * cs[i] - y * sn[i];
            b[i] = y * cs[i] + x * sn[i];
          }
        } else {
          // pairs (2 i, 2 i + 1) of the unit's 2 V neighbours: the first V / 2 pairs lie in a, the others in b
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
            a[2 * i] = x * cs[i] - y * sn[i];
            a[2 * i + 1] = y * cs[i] + x * sn[i];
            b[2 * i] = z * cs[V / 2 + i] - w * sn[V / 2 + i];
            b[2 * i + 1] = w * cs[V / 2 + i] + z * sn[V / 2 + i];
          }
        }
      }
      if (!on || h >= heads) continue;
      __nv_bfloat16 *dst = nullptr, *dense = nullptr;
      if (kind == 0) {
        dst = p.q_out + (static_cast<long long>(t) * p.hq + h) * p.d;
      } else {
        const int hk = kind == 1 ? h - p.hq : h - p.hq - p.hkv;
        __nv_bfloat16* cache = kind == 1 ? p.k_cache : p.v_cache;
        if (cache && stored >= 0) dst = cache + (stored + static_cast<long long>(hk) * p.page) * p.d;
        dense = kind == 1 ? p.k_out : p.v_out;
        if (dense) dense += (static_cast<long long>(t) * p.hkv + hk) * p.d;
      }
      if (dst) {
        axes_store<V>(dst + ca, a);
        axes_store<V>(dst + cb, b);
      }
      if (dense) {
        axes_store<V>(dense + ca, a);
        axes_store<V>(dense + cb, b);
      }
    }
  }
}

// The same for heads whose halves are no multiple of four values (or not aligned to them): a warp a head, value by value.
__global__ void __launch_bounds__(256) rope_axes_any_kernel(const RopeAxesParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float rows[8][256];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, heads = p.hq + 2 * p.hkv, half = p.rot >> 1;
  const long long unit = static_cast<long long>(blockIdx.x) * 8 + wid;
  if (unit >= static_cast<long long>(p.tokens) * heads) return;
  const int t = static_cast<int>(unit / heads), h = static_cast<int>(unit - static_cast<long long>(t) * heads);
  const int kind = h < p.hq ? 0 : (h < p.hq + p.hkv ? 1 : 2);
  float* row = rows[wid];
  float ss = 0.f;
  for (int c = lane; c < p.d; c += 32) {
    row[c] = __bfloat162float(p.qkv[unit * p.d + c]);
    ss += row[c] * row[c];
  }
  const __nv_bfloat16* nw = kind == 0 ? p.q_norm_w : (kind == 1 ? p.k_norm_w : nullptr);
  if (nw) {
    const float rstd = rsqrtf(warp_sum(ss) / p.d + p.eps);
    for (int c = lane; c < p.d; c += 32) row[c] = row[c] * rstd * __bfloat162float(nw[c]);
  }
  __syncwarp();
  if (kind != 2) {
    for (int j = lane; j < half; j += 32) {
      const int ca = p.style == 0 ? j : 2 * j, cb = p.style == 0 ? j + half : 2 * j + 1;
      const float2 cs = axes_turn(p, t, j);
      const float x = row[ca], y = row[cb];
      row[ca] = x * cs.x - y * cs.y;
      row[cb] = y * cs.x + x * cs.y;
    }
    __syncwarp();
  }
  __nv_bfloat16 *dst = nullptr, *dense = nullptr;
  if (kind == 0) {
    dst = p.q_out + (static_cast<long long>(t) * p.hq + h) * p.d;
  } else {
    const int hk = kind == 1 ? h - p.hq : h - p.hq - p.hkv;
    __nv_bfloat16* cache = kind == 1 ? p.k_cache : p.v_cache;
    const long long at = axes_row(p, t, lane == 0);
    if (cache && at >= 0) dst = cache + (at + static_cast<long long>(hk) * p.page) * p.d;
    dense = kind == 1 ? p.k_out : p.v_out;
    if (dense) dense += (static_cast<long long>(t) * p.hkv + hk) * p.d;
  }
  for (int c = lane; c < p.d; c += 32) {
    const __nv_bfloat16 y = __float2bfloat16(row[c]);
    if (dst) dst[c] = y;
    if (dense) dense[c] = y;
  }
}

template <int V>
static cudaError_t launch_rope_axes(RopeAxesParams p, cudaStream_t stream) {
  const bool norm = p.q_norm_w || p.k_norm_w;
  int lanes = p.d / (2 * V);
  if (norm)
    for (lanes = 1; lanes * 2 * V < p.d;) lanes *= 2;
  const int each = 256 / lanes, chunks = (p.hq + 2 * p.hkv + each - 1) / each;
  p.block_tokens = p.tokens >= num_sms() * 8 ? 4 : 1;      // more tokens a block once every processor has several
  return launch_pdl(rope_axes_kernel<V>, dim3((p.tokens + p.block_tokens - 1) / p.block_tokens, p.block_tokens == 1 ? chunks : 1), dim3(256),
                    (p.block_tokens * 2 * (((p.rot >> 1) + 3) & ~3) + (norm ? 2 * p.d : 0)) * sizeof(float), stream, p, lanes);
}

}  // namespace b200

using namespace b200;

// See the header comment and RopeAxesParams. d even, at most 256; rot even, at most d. A slot behind the pool's end is not stored and a pair
// whose axis does not exist is not turned; both are reported in the status word.
B200_API int b200_rope_axes(const void* qkv, void* q_out, void* k_cache, void* v_cache, void* k_out, void* v_out, const int* positions,
                            const int* axes, const float* inv_freq, const long long* slots, const void* q_norm_w, const void* k_norm_w,
                            int tokens, int n_axes, int hq, int hkv, int d, int rot, int style, int page, long long pages, float eps,
                            void* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (hq < 1 || hkv < 1 || d < 2 || d > 256 || (d & 1) || rot < 0 || rot > d || (rot & 1) || (style != 0 && style != 1)) return -2;
  if (rot > 0 && (n_axes < 1 || !positions || !axes || !inv_freq)) return -3;
  if ((k_cache || v_cache) && (page < 1 || pages < 0 || !k_cache || !v_cache)) return -4;
  if (static_cast<long long>(hq + 2ll * hkv) * d >= (1ll << 31)) return -2;
  RopeAxesParams p{};
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_cache = static_cast<__nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<__nv_bfloat16*>(v_cache);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.positions = positions; p.axes = axes; p.inv_freq = inv_freq; p.slots = slots;
  p.q_norm_w = static_cast<const __nv_bfloat16*>(q_norm_w);
  p.k_norm_w = static_cast<const __nv_bfloat16*>(k_norm_w);
  p.slots_end = k_cache ? pages * page : 0;
  p.tokens = tokens; p.n_axes = n_axes; p.hq = hq; p.hkv = hkv; p.d = d; p.rot = rot; p.style = style; p.page = page;
  p.eps = eps;
  p.status = static_cast<DeviceStatus*>(status);
  uintptr_t all = 0;
  for (const void* x : {qkv, static_cast<const void*>(q_out), static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    all |= reinterpret_cast<uintptr_t>(x);
  const auto fits = [&](int v) {
    return d % (2 * v) == 0 && all % (2 * v) == 0 && (style == 1 || ((rot >> 1) % v == 0 && (d - rot) % (2 * v) == 0));
  };
  cudaError_t e;
  if (fits(8)) {
    e = launch_rope_axes<8>(p, stream);
  } else if (fits(4)) {
    e = launch_rope_axes<4>(p, stream);
  } else {
    const long long blocks = (static_cast<long long>(tokens) * (hq + 2 * hkv) + 7) / 8;
    if (blocks >= (1ll << 31)) return -2;
    e = launch_pdl(rope_axes_any_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p);
  }
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}
