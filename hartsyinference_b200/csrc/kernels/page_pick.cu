// The pages that queries attend to, chosen by a cheap score (formats: picked.cuh).
//
//  * key_bounds   after a forward pass has stored its keys: largest and smallest value of every channel over the keys of each page that became
//                 full, in 8 bits with a common power of two
//  * pick_pages   for each run of queries and key head: the `first` pages, the `last` up to the run's own and what lies behind, and the `top` of
//                 the largest score between them. With a the codes of a query head (8 bits and a power of two of their own)
//                   score(page) = max over queries of 2^(e_q + e_page) * sum_c max(a_c high_c, a_c low_c),
//                 a bound of every product of a with a key of the page. max(a h, a l) is a+ h + a- l, so the sum is an integer product of 2 D
//                 codes: mma.sync on 8-bit integers, exact, below 2^22 and scaled by a power of two. What is kept does not depend on any order.
#include "picked.cuh"

namespace b200 {

struct BoundsParams {
  const __nv_bfloat16* k;      // [pages][hkv][page][D]
  uint8_t* bounds;             // [pages][hkv][2 D + 16]
  const int *block_table, *kv_lens, *cu_q;
  long long pages, units;
  int seqs, hkv, page_shift, max_pages, per_seq;
  DeviceStatus* status;
};

// A warp per page and head; four channels a lane, D / 4 lanes a key.
template <int D>
__global__ void __launch_bounds__(256) key_bounds_kernel(const BoundsParams p) {
  pdl_wait();
  pdl_trigger();
  const long long unit = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const int lane = threadIdx.x & 31, page = 1 << p.page_shift;
  const int h = static_cast<int>(unit % p.hkv), seq = static_cast<int>(unit / p.hkv / p.per_seq), j = static_cast<int>(unit / p.hkv % p.per_seq);
  const int q_len = p.cu_q ? p.cu_q[seq + 1] - p.cu_q[seq] : 1;
  const int kv_len = static_cast<int>(min(static_cast<long long>(p.kv_lens[seq]), static_cast<long long>(p.max_pages) << p.page_shift));
  const int at = (max(0, kv_len - q_len) >> p.page_shift) + j;
  if (q_len <= 0 || kv_len <= 0 || at >= kv_len >> p.page_shift) return;
  const int id = p.block_table[static_cast<long long>(seq) * p.max_pages + at];
  if (id < 0 || id >= p.pages) {
    if (lane == 0) report_status(p.status, kBadArgument, kKernelPicked, 1, static_cast<uint32_t>(seq));
    return;
  }
  constexpr int kLanes = D / 4, kRows = 32 / kLanes;
  const int c = (lane & (kLanes - 1)) * 4;
  const __nv_bfloat16* src = p.k + (static_cast<long long>(id) * p.hkv + h) * page * D + c;
  float high[4], low[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { high[i] = -INFINITY; low[i] = INFINITY; }
  for (int t0 = lane / kLanes; t0 < page; t0 += 8 * kRows) {
    uint2 raw[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) raw[u] = *reinterpret_cast<const uint2*>(src + min(t0 + u * kRows, page - 1) * D);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw[u]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2 f = __bfloat1622float2(b[i]);
        f.x = f.x == f.x ? f.x : 0.f;
        f.y = f.y == f.y ? f.y : 0.f;
        high[2 * i] = fmaxf(high[2 * i], f.x);
        low[2 * i] = fminf(low[2 * i], f.x);
        high[2 * i + 1] = fmaxf(high[2 * i + 1], f.y);
        low[2 * i + 1] = fminf(low[2 * i + 1], f.y);
      }
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int o = kLanes; o < 32; o <<= 1) {
      high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], o));
      low[i] = fminf(low[i], __shfl_xor_sync(0xffffffffu, low[i], o));
    }
    top = fmaxf(top, fmaxf(fabsf(high[i]), fabsf(low[i])));
  }
  top = warp_max(top);
  const int e = bounds_exponent(top);
  const float f = bounds_pow2(-e);
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(ceilf(high[i] * f), -127.f), 127.f))) & 0xffu) << (8 * i);
    lo |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(floorf(low[i] * f), -127.f), 127.f))) & 0xffu) << (8 * i);
  }
  uint8_t* dst = p.bounds + (static_cast<long long>(id) * p.hkv + h) * (2 * D + kBoundsTail);
  if (lane < kLanes) {
    *reinterpret_cast<uint32_t*>(dst + c) = hi;
    *reinterpret_cast<uint32_t*>(dst + D + c) = lo;
  }
  if (lane == 0) *reinterpret_cast<uint4*>(dst + 2 * D) = make_uint4(static_cast<uint32_t>(e + kBoundsBias), 0u, 0u, 0u);
}

// ------------------------------------------------------------------------------------------ the choice
constexpr int kPickThreads = 256, kPickWarps = 8, kPickBins = 256;
constexpr int kPickRows = 128;          // queries of a run, heads counted

struct PickParams {
  const __nv_bfloat16* q;      // [tokens][hq][D]
  const uint8_t* bounds;       // [pages][hkv][2 D + 16]
  const int *block_table, *kv_lens, *cu_q;
  int* out;                    // [rows][hkv][width]
  long long pages;
  int seqs, hq, hkv, run, page_shift, max_pages, top, first, last, width, parts, cap;
  DeviceStatus* status;
};

struct PickShared {
  unsigned hist[2][kPickBins];
  unsigned meet[2];                 // smallest and largest key of this block
  unsigned counts[2];               // this block's selected and tied ones
  unsigned warp_a[kPickWarps], warp_b[kPickWarps];
  unsigned bin, want, in_bin;
  float2 row[kPickRows];            // 2^e and 0, or 0 and -inf for rows that pad
};

__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pick_peer(const void* local, int block) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(block));
  return r;
}
__device__ __forceinline__ unsigned pick_peer_load(const void* local, int block) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(pick_peer(local, block)) : "memory");
  return v;
}

// Barrier over the blocks of a row.
__device__ __forceinline__ void pick_sync(int parts) {
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
}

// A cluster of `parts` blocks per row of runs and key head; each scores a share of the pages.
template <int D>
__global__ void __launch_bounds__(kPickThreads) pick_pages_kernel(const PickParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t pick_smem[];
  PickShared& sh = *reinterpret_cast<PickShared*>(pick_smem);
  constexpr int kPitch = 2 * D + 64;      // of a query's codes: rows of eight lanes keep apart in the banks
  uint8_t* codes = pick_smem + (sizeof(PickShared) + 15) / 16 * 16;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, group = p.hq / p.hkv;
  const int row = blockIdx.x / p.parts, rank = blockIdx.x % p.parts, h = blockIdx.y;
  const int tiles = (p.run * group + 15) / 16;
  float* scores = reinterpret_cast<float*>(codes + tiles * 16 * kPitch);
  int* out = p.out + (static_cast<long long>(row) * p.hkv + h) * p.width;
  const RunOfRow r = run_of_row(p.cu_q, p.kv_lens, p.seqs, p.run, row, static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x7fffffffll)));
  const int end = r.begin + r.tokens - 1;
  if (r.tokens <= 0 || end < 0) {
    if (rank == 0)
      for (int i = threadIdx.x; i < p.width; i += kPickThreads) out[i] = -1;
    return;
  }
  const int page0 = max(r.begin, 0) >> p.page_shift, page1 = end >> p.page_shift;
  const int hi = max(p.first, page0 - p.last + 1), n = hi - p.first;       // pages first .. hi are scored
  if (n <= p.top) {                                                        // every page is kept
    if (rank == 0)
      for (int i = threadIdx.x; i < p.width; i += kPickThreads) out[i] = i <= page1 ? i : -1;
    return;
  }
  // (from here on first < hi <= page1)
  if (rank == 0) {
    const int tail = page1 - hi + 1;
    for (int i = threadIdx.x; i < p.first; i += kPickThreads) out[i] = i;
    for (int i = p.first + p.top + threadIdx.x; i < p.width; i += kPickThreads) {
      const int j = i - p.first - p.top;
      out[i] = j < tail ? hi + j : -1;
    }
  }
  if (p.top == 0) return;

  // ---- codes of the queries: a+ against the largest values, a- against the smallest
  for (int i = wid; i < tiles * 16; i += kPickWarps) {
    constexpr int kEach = D / 32;
    const bool real = i < r.tokens * group && r.begin + i / group >= 0;
    float v[kEach], amax = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) v[k] = 0.f;
    if (real) {
      const __nv_bfloat16* src = p.q + (static_cast<long long>(r.q_off + i / group) * p.hq + h * group + i % group) * D + lane * kEach;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        v[k] = __bfloat162float(src[k]);
        v[k] = v[k] == v[k] ? v[k] : 0.f;
        amax = fmaxf(amax, fabsf(v[k]));
      }
    }
    const int e = bounds_exponent(warp_max(amax));
    const float f = bounds_pow2(-e);
    uint8_t* dst = codes + i * kPitch + lane * kEach;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int a = static_cast<int>(fminf(fmaxf(rintf(v[k] * f), -127.f), 127.f));
      dst[k] = static_cast<uint8_t>(max(a, 0));
      dst[D + k] = static_cast<uint8_t>(min(a, 0));
    }
    if (lane == 0) sh.row[i] = real ? make_float2(bounds_pow2(e), 0.f) : make_float2(0.f, -INFINITY);
  }
  __syncthreads();

  // ---- scores of this block's share
  const int per = (n + p.parts - 1) / p.parts, a0 = min(n, rank * per), mine = min(n, a0 + per) - a0;
  const int* ids = p.block_table + static_cast<long long>(r.seq) * p.max_pages + p.first + a0;
  const int g = lane >> 2, kq = lane & 3;
  for (int base = wid * 32; base < mine; base += kPickWarps * 32) {
    // operands: channels are taken in an order of their own, 16 bytes a lane of every 64; sums do not mind
    uint4 b[4][2 * D / 64];
    float unit[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      const int at = min(base + nb * 8 + g, mine - 1);
      int id = ids[at];
      const bool ok = id >= 0 && id < p.pages;
      if (!ok) {
        report_status(p.status, kBadArgument, kKernelPicked, 2, static_cast<uint32_t>(r.seq));
        id = 0;
      }
      const uint8_t* src = p.bounds + (static_cast<long long>(id) * p.hkv + h) * (2 * D + kBoundsTail);
#pragma unroll
      for (int c = 0; c < 2 * D / 64; ++c) b[nb][c] = __ldg(reinterpret_cast<const uint4*>(src + c * 64 + kq * 16));
      unit[nb] = ok ? bounds_pow2(min(50, max(-50, static_cast<int>(__ldg(src + 2 * D)) - kBoundsBias))) : 0.f;
    }
    float best[4][2];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) best[nb][0] = best[nb][1] = -INFINITY;
    for (int mt = 0; mt < tiles; ++mt) {
      int acc[4][4];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) acc[nb][0] = acc[nb][1] = acc[nb][2] = acc[nb][3] = 0;
      const uint8_t* src = codes + (mt * 16 + g) * kPitch + kq * 16;
#pragma unroll
      for (int c = 0; c < 2 * D / 64; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(src + c * 64), y = *reinterpret_cast<const uint4*>(src + 8 * kPitch + c * 64);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          mma_s8_16832(acc[nb], x.x, y.x, x.y, y.y, b[nb][c].x, b[nb][c].y);
          mma_s8_16832(acc[nb], x.z, y.z, x.w, y.w, b[nb][c].z, b[nb][c].w);
        }
      }
      const float2 f0 = sh.row[mt * 16 + g], f1 = sh.row[mt * 16 + 8 + g];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          best[nb][i] = fmaxf(best[nb][i], fmaxf(fmaf(static_cast<float>(acc[nb][i]), f0.x, f0.y), fmaf(static_cast<float>(acc[nb][2 + i]), f1.x, f1.y)));
    }
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) best[nb][i] = fmaxf(best[nb][i], __shfl_xor_sync(0xffffffffu, best[nb][i], o));
      // column g of the tile is with the lanes of quarter g / 2
      const float x = __shfl_sync(0xffffffffu, best[nb][0], g >> 1), y = __shfl_sync(0xffffffffu, best[nb][1], g >> 1);
      const int at = base + nb * 8 + g;
      if (kq == nb && at < mine) scores[at] = unit[nb] > 0.f ? (g & 1 ? y : x) * unit[nb] : -INFINITY;
    }
  }
  __syncthreads();

  // ---- the `top` largest: keys order like scores; digits of 8 bits of what they lie above the smallest
  const auto key_of = [&](int i) {
    const unsigned u = __float_as_uint(scores[i]);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
  };
  unsigned least = 0xffffffffu, most = 0u;
  for (int i = threadIdx.x; i < mine; i += kPickThreads) {
    const unsigned k = key_of(i);
    least = min(least, k);
    most = max(most, k);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) { sh.warp_a[wid] = least; sh.warp_b[wid] = most; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPickWarps; ++w) { least = min(least, sh.warp_a[w]); most = max(most, sh.warp_b[w]); }
    sh.meet[0] = least;
    sh.meet[1] = most;
  }
  pick_sync(p.parts);
  if (p.parts > 1) {
    least = 0xffffffffu;
    most = 0u;
    for (int k = 0; k < p.parts; ++k) {
      least = min(least, pick_peer_load(&sh.meet[0], k));
      most = max(most, pick_peer_load(&sh.meet[1], k));
    }
  } else {
    least = sh.meet[0];
    most = sh.meet[1];
  }
  int shift = 32 - __clz(static_cast<int>(most - least));        // bits that differ
  unsigned prefix = 0u, want = static_cast<unsigned>(p.top);
  for (int pass = 0;; ++pass) {
    const int bits = min(8, shift);
    shift -= bits;
    unsigned* hist = sh.hist[pass & 1];
    hist[threadIdx.x] = 0u;                                        // 256 threads, 256 bins
    __syncthreads();
    for (int i = threadIdx.x; i < mine; i += kPickThreads) {
      const unsigned k = key_of(i) - least, digit = (k >> shift) & ((1u << bits) - 1u);
      if ((static_cast<unsigned long long>(k) >> (shift + bits)) == prefix) atomicAdd(hist + digit, 1u);
    }
    pick_sync(p.parts);
    unsigned count = 0;
    if (p.parts > 1) {
      for (int k = 0; k < p.parts; ++k) count += pick_peer_load(hist + threadIdx.x, k);
    } else {
      count = hist[threadIdx.x];
    }
    // how many lie in this bin and above it
    unsigned upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_down_sync(0xffffffffu, upto, o);
      if (lane + o < 32) upto += x;
    }
    if (lane == 0) sh.warp_a[wid] = upto;
    __syncthreads();
    for (int w = wid + 1; w < kPickWarps; ++w) upto += sh.warp_a[w];
    if (upto >= want && upto - count < want) {
      sh.bin = threadIdx.x;
      sh.want = want - (upto - count);
      sh.in_bin = count;
    }
    __syncthreads();
    prefix = (prefix << bits) | sh.bin;
    want = sh.want;
    const bool done = sh.in_bin == want || shift == 0;
    if (done) break;                     // (the same in every block of the row)
  }

  // ---- kept: larger prefixes, and the first `want` of the equal ones
  const int seg = ((mine + kPickWarps - 1) / kPickWarps + 31) & ~31, s0 = min(mine, wid * seg), s1 = min(mine, s0 + seg);
  unsigned over = 0, tied = 0;
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < s1 ? (key_of(i) - least) >> shift : 0u;
    over += __popc(__ballot_sync(0xffffffffu, i < s1 && k > prefix));
    tied += __popc(__ballot_sync(0xffffffffu, i < s1 && k == prefix));
  }
  if (lane == 0) { sh.warp_a[wid] = over; sh.warp_b[wid] = tied; }
  __syncthreads();
  unsigned over0 = 0, tied0 = 0;
  for (int w = 0; w < wid; ++w) { over0 += sh.warp_a[w]; tied0 += sh.warp_b[w]; }
  if (threadIdx.x == kPickThreads - 1) { sh.counts[0] = over0 + over; sh.counts[1] = tied0 + tied; }
  pick_sync(p.parts);
  if (p.parts > 1)
    for (int k = 0; k < rank; ++k) {
      over0 += pick_peer_load(&sh.counts[0], k);
      tied0 += pick_peer_load(&sh.counts[1], k);
    }
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < s1 ? (key_of(i) - least) >> shift : 0u, below = (1u << lane) - 1u;
    const unsigned more = __ballot_sync(0xffffffffu, i < s1 && k > prefix), same = __ballot_sync(0xffffffffu, i < s1 && k == prefix);
    const unsigned o = over0 + __popc(more & below), t = tied0 + __popc(same & below);
    const bool kept = (more >> lane & 1u) || ((same >> lane & 1u) && t < want);
    if (kept) out[p.first + o + min(t, want)] = p.first + a0 + i;
    over0 += __popc(more);
    tied0 += __popc(same);
  }
  if (p.parts > 1) cluster_sync_all();     // nobody leaves while a peer may still read its words
}

template <int D>
static int launch_pick(const PickParams& p, int rows, int smem, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (configured.first_time() && cudaFuncSetAttribute(pick_pages_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return -200;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * p.parts, p.hkv);
  cfg.blockDim = dim3(kPickThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_b200_pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, pick_pages_kernel<D>, p);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}

}  // namespace b200

using namespace b200;

static int picked_page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

// k [pages][hkv][page][d] bf16, bounds [pages][hkv][2 d + 16]; block_table [seqs][max_pages], kv_lens [seqs], cu_q [seqs + 1] or null (one new
// token a sequence), max_q_len: no sequence has more. Pages that hold one of a sequence's last q_len keys and are full are bounded.
B200_API int b200_key_bounds(const void* k, void* bounds, const int* block_table, const int* kv_lens, const int* cu_q, int seqs, int max_q_len,
                             int hkv, int d, int page, int max_pages, long long pages, void* status, cudaStream_t stream) {
  if (seqs <= 0 || max_q_len <= 0 || max_pages <= 0) return 0;
  BoundsParams p{};
  p.page_shift = picked_page_shift(page);
  if (p.page_shift < 0 || hkv < 1 || pages < 1 || (d != 64 && d != 128)) return -2;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(bounds)) & 15) return -4;
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.bounds = static_cast<uint8_t*>(bounds);
  p.block_table = block_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
  p.pages = pages;
  p.seqs = seqs; p.hkv = hkv; p.max_pages = max_pages;
  const long long most = (static_cast<long long>(max_q_len) + page - 1) >> p.page_shift;       // pages that so many tokens fill
  p.per_seq = static_cast<int>(most < max_pages ? most : max_pages);
  p.units = static_cast<long long>(seqs) * p.per_seq * hkv;
  p.status = static_cast<DeviceStatus*>(status);
  const long long blocks = (p.units + 7) / 8;
  if (blocks >= (1ll << 31)) return -3;
  const dim3 grid(static_cast<unsigned>(blocks));
  const cudaError_t e = d == 128 ? launch_pdl(key_bounds_kernel<128>, grid, dim3(256), 0, stream, p) : launch_pdl(key_bounds_kernel<64>, grid, dim3(256), 0, stream, p);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}

// q [tokens][hq][d] bf16, out int32 [rows][hkv][width] (see picked.cuh), rows = (tokens + seqs (run - 1)) / run,
// width >= first + top + last + (run + page - 2) / page.
B200_API int b200_pick_pages(const void* q, const void* bounds, const int* block_table, const int* kv_lens, const int* cu_q, int* out, int seqs,
                             int rows, int hq, int hkv, int d, int page, int max_pages, long long pages, int run, int top, int first, int last,
                             int width, void* status, cudaStream_t stream) {
  if (rows <= 0 || seqs <= 0) return 0;
  PickParams p{};
  p.page_shift = picked_page_shift(page);
  if (p.page_shift < 0 || hkv < 1 || hq < 1 || hq % hkv || pages < 1 || max_pages < 1 || (d != 64 && d != 128) || hkv > 65535) return -2;
  if (run < 1 || static_cast<long long>(run) * (hq / hkv) > kPickRows || (!cu_q && (run != 1 || rows != seqs))) return -3;
  if (top < 0 || first < 0 || last < 1 || static_cast<long long>(first) + top + last + (run + page - 2) / page > width) return -5;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(bounds)) & 15) return -4;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.bounds = static_cast<const uint8_t*>(bounds);
  p.block_table = block_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
  p.out = out;
  p.pages = pages;
  p.seqs = seqs; p.hq = hq; p.hkv = hkv; p.run = run; p.max_pages = max_pages;
  p.top = top; p.first = first; p.last = last; p.width = width;
  p.status = static_cast<DeviceStatus*>(status);
  const int codes = (run * (hq / hkv) + 15) / 16 * 16 * (2 * d + 64), fixed = (static_cast<int>(sizeof(PickShared)) + 15) / 16 * 16 + codes;
  // blocks of a row: until the processors have two each, as long as a block has 256 pages to score; at least as many as hold the scores
  p.parts = 1;
  while (p.parts < 8 && static_cast<long long>(rows) * hkv * p.parts < num_sms() && max_pages > p.parts * 256) p.parts *= 2;
  while (p.parts < 8 && fixed + static_cast<long long>((max_pages + p.parts - 1) / p.parts) * 4 > 100000) p.parts *= 2;
  p.cap = (max_pages + p.parts - 1) / p.parts;
  if (fixed + 4ll * p.cap > 232448) return -6;
  if (static_cast<long long>(rows) * p.parts >= (1ll << 31)) return -3;
  return d == 128 ? launch_pick<128>(p, rows, fixed + 4 * p.cap, stream) : launch_pick<64>(p, rows, fixed + 4 * p.cap, stream);
}
