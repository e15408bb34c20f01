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

int make_kmajor_map(CUtensorMap* out, const void* base, int elem_bytes, long long rows, long long k, long long ld, int box_rows);

struct BoundsParams {
  const __nv_bfloat16* k;      // [pages][hkv][page][D]
  uint8_t* bounds;             // [pages][hkv][2 D + 16]
  const int *block_table, *kv_lens, *cu_q;
  long long pages, units;
  int seqs, hkv, page_shift, max_pages, per_seq;
  DeviceStatus* status;
};

// A warp per page and head; four channels a lane, D / 4 lanes a key. Bound by latency: a warp has few loads and one page. The pages of 2048 new tokens, 8 heads
// of 128, take 3.1 us, one token of 16 sequences 1.3.
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
constexpr int kPickThreads = 512, kPickWarps = 16, kPickBins = 2048;
constexpr int kPickRows = 128;          // queries of a run, heads counted
constexpr int kPickStep = 16;           // pages that a warp scores at a time

struct PickParams {
  const __nv_bfloat16* q;      // [tokens][hq][D]
  const uint8_t* bounds;       // [pages][hkv][2 D + 16]
  const int *block_table, *kv_lens, *cu_q;
  int* out;                    // [rows][hkv][width]
  long long pages;
  int seqs, rows, tokens, hq, hkv, run, page_shift, max_pages, top, first, last, width, parts;
  int pairs;                   // rows of runs of twice as many queries
  DeviceStatus* status;
};

struct PickShared {
  unsigned hist[kPickBins];
  unsigned least[8 * kPickWarps], most[8 * kPickWarps];      // smallest and largest key of every warp of the row's blocks
  unsigned warp_a[kPickWarps], warp_b[kPickWarps];
  unsigned counts[2];               // this block's selected and tied ones
  unsigned bin, want, in_bin, listed;
  unsigned list[32];                // keys of a bin that is nearly all that is left
  __align__(16) float row[kPickRows];       // of a query: 2^e
};

// What a row of runs chooses between: pages first .. first + n are scored, if there are more of them than `top`.
struct PickRange {
  RunOfRow run;
  int n;
};

__device__ __forceinline__ RunOfRow pick_run(const PickParams& p, int row, int runs = 1) {
  return run_of_row(p.cu_q, p.kv_lens, p.seqs, runs * p.run, row, static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x7fffffffll)), p.tokens);
}

// The pages that are kept whatever the scores, of run x.run (written by the block of rank 0); false: nothing is left to choose.
__device__ __forceinline__ bool pick_range(const PickParams& p, int* out, bool writes, PickRange& x) {
  const int end = x.run.begin + x.run.tokens - 1;
  if (x.run.tokens <= 0 || end < 0) {
    if (writes)
      for (int i = threadIdx.x; i < p.width; i += blockDim.x) out[i] = -1;
    return false;
  }
  const int page0 = max(x.run.begin, 0) >> p.page_shift, page1 = end >> p.page_shift;
  const int hi = max(p.first, page0 - p.last + 1);
  x.n = hi - p.first;
  if (x.n <= p.top) {                                                        // every page is kept
    if (writes)
      for (int i = threadIdx.x; i < p.width; i += blockDim.x) out[i] = i <= page1 ? i : -1;
    return false;
  }
  // (from here on first < hi <= page1)
  if (writes) {
    const int tail = page1 - hi + 1;
    for (int i = threadIdx.x; i < p.first; i += blockDim.x) out[i] = i;
    for (int i = p.first + p.top + threadIdx.x; i < p.width; i += blockDim.x) {
      const int j = i - p.first - p.top;
      out[i] = j < tail ? hi + j : -1;
    }
  }
  return p.top > 0;
}

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
__device__ __forceinline__ void pick_peer_store(const void* local, int block, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(pick_peer(local, block)), "r"(v) : "memory");
}

// Sums are below 2^22, so 1.5 * 2^23 + sum is a float with the sum in its last bits, and that number taken off again leaves the sum as a float, exactly
// (conversions take four times as long; so do roundings, which the same addition makes).
constexpr float kPickLarge = 12582912.f;
constexpr int kPickLargeBits = 0x4b400000;
__device__ __forceinline__ float pick_float(int sum) { return __int_as_float(sum + kPickLargeBits) - kPickLarge; }
// Two sums at a time, times two factors.
__device__ __forceinline__ float2 pick_scaled2(int a, int b, float2 f) {
  float2 r;
  asm("{\n\t"
      ".reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %4};\n\t"
      "mov.b64 z, {%5, %6};\n\t"
      "add.rn.f32x2 x, x, y;\n\t"
      "mul.rn.f32x2 x, x, z;\n\t"
      "mov.b64 {%0, %1}, x;\n\t"
      "}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(__int_as_float(a + kPickLargeBits)), "f"(__int_as_float(b + kPickLargeBits)), "f"(-kPickLarge), "f"(f.x), "f"(f.y));
  return r;
}
// Code of a channel: v times f, a power of two, to the nearest whole number from -127 to 127.
__device__ __forceinline__ int pick_code(float v, float f) {
  return __float_as_int(fminf(fmaxf(v * f, -127.f), 127.f) + kPickLarge) - kPickLargeBits;
}

// Keys order like scores.
__device__ __forceinline__ unsigned pick_key(float score) {
  const unsigned u = __float_as_uint(score);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The `top` largest of more than `top` scores, of which this block holds the `mine` from number `a0` on, ties to the lowest number: first + number, in order, to
// out[0 .. top). `least` and `most` bound all keys. Digits of what keys lie above the smallest, as many as it takes: 11 bits where one block holds all
// scores; 9 in a cluster, whose blocks read one another's counts. Once a digit leaves 32 keys at most, every warp ranks them by itself. All threads of all blocks
// of the row, or `kThreads` threads (tid) of a block that share barrier `bar`; sh.hist is zero before, for all of them to see.
template <bool kCluster, int kThreads>
__device__ __forceinline__ void pick_select(PickShared& sh, int tid, int bar, const float* scores, int mine, int a0, int rank, int parts, int top, unsigned least, unsigned most,
                                            int first, int* out) {
  constexpr int kWarps = kThreads / 32, kDigit = kCluster ? 9 : 11, kBins = 1 << kDigit, kEach = kBins / kThreads;
  const int lane = tid & 31, wid = tid >> 5;
  const auto sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(kThreads) : "memory"); };
  int shift = 32 - __clz(static_cast<int>(most - least));        // bits that differ
  unsigned prefix = 0u, want = static_cast<unsigned>(top);
  for (int pass = 0;; ++pass) {
    const int bits = min(kDigit, shift);
    shift -= bits;
    unsigned* hist = sh.hist + (kCluster ? (pass & 1) * kBins : 0);      // (a peer may still read those of the pass before)
    if (pass >= (kCluster ? 2 : 1)) {
      if (kEach >= 4) {
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) reinterpret_cast<uint4*>(hist)[i * kThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
      } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) hist[i * kThreads + tid] = 0u;
      }
      sync();
    }
#pragma unroll 4
    for (int i = tid; i < mine; i += kThreads) {
      const unsigned k = pick_key(scores[i]) - least;
      if ((static_cast<unsigned long long>(k) >> (shift + bits)) == prefix) atomicAdd(hist + ((k >> shift) & ((1u << bits) - 1u)), 1u);
    }
    if (kCluster) cluster_sync_all();
    else sync();
    // a thread owns neighbouring bins; how many lie in them and above
    unsigned own[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (kCluster) {
        own[i] = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < parts) own[i] += pick_peer_load(hist + tid * kEach + i, k);
      } else if (i % 4 == 0) {                 // (four bins at a time: one by one the lanes would meet in the banks)
        const uint4 x = *reinterpret_cast<const uint4*>(hist + tid * kEach + i);
        own[i] = x.x; own[i + 1] = x.y; own[i + 2] = x.z; own[i + 3] = x.w;
      }
      sum += own[i];
    }
    unsigned upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_down_sync(0xffffffffu, upto, o);
      if (lane + o < 32) upto += x;
    }
    if (lane == 0) sh.warp_a[wid] = upto;
    sync();
    upto += __reduce_add_sync(0xffffffffu, lane > wid && lane < kWarps ? sh.warp_a[lane] : 0u);
    unsigned above = upto - sum;
    if (above < want && upto >= want) {
#pragma unroll
      for (int i = kEach - 1; i >= 0; --i) {
        if (above < want && above + own[i] >= want) {
          sh.bin = tid * kEach + i;
          sh.want = want - above;
          sh.in_bin = own[i];
          sh.listed = 0;
        }
        above += own[i];
      }
    }
    sync();
    prefix = (prefix << bits) | sh.bin;
    want = sh.want;
    const unsigned left = sh.in_bin;
    if (left == want || shift == 0) break;           // (alike in all blocks)
    if (left > 32) continue;
#pragma unroll 4
    for (int i = tid; i < mine; i += kThreads) {
      const unsigned k = pick_key(scores[i]) - least;
      if (k >> shift == prefix) sh.list[atomicAdd(&sh.listed, 1u)] = k;
    }
    if (kCluster) cluster_sync_all();
    else sync();
    unsigned key = 0;
    if (kCluster) {
      unsigned to = lane < parts ? pick_peer_load(&sh.listed, lane) : 0u, from;
      const unsigned count = to;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, to, o);
        if (lane >= o) to += x;
      }
      from = to - count;
      for (int k = 0; k < parts; ++k) {
        const int a = static_cast<int>(__shfl_sync(0xffffffffu, from, k)), b = static_cast<int>(__shfl_sync(0xffffffffu, to, k));
        if (lane >= a && lane < b) key = pick_peer_load(sh.list + (lane - a), k);
      }
    } else if (lane < static_cast<int>(left)) {
      key = sh.list[lane];
    }
    unsigned larger = 0, alike = 0;
    for (int i = 0; i < static_cast<int>(left); ++i) {
      const unsigned x = __shfl_sync(0xffffffffu, key, i);
      larger += x > key;
      alike += x == key;
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, lane < static_cast<int>(left) && larger < want && larger + alike >= want)) - 1;
    prefix = __shfl_sync(0xffffffffu, key, at);
    want -= __shfl_sync(0xffffffffu, larger, at);
    shift = 0;
    break;
  }
  // kept: larger prefixes, and the first `want` of the equal ones
  const int seg = ((mine + kWarps - 1) / kWarps + 31) & ~31, s0 = min(mine, wid * seg), s1 = min(mine, s0 + seg);
  unsigned over = 0, tied = 0;
#pragma unroll 4
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < s1 ? (pick_key(scores[i]) - least) >> shift : 0u;
    over += __popc(__ballot_sync(0xffffffffu, i < s1 && k > prefix));
    tied += __popc(__ballot_sync(0xffffffffu, i < s1 && k == prefix));
  }
  if (lane == 0) { sh.warp_a[wid] = over; sh.warp_b[wid] = tied; }
  sync();
  unsigned over0 = __reduce_add_sync(0xffffffffu, lane < wid ? sh.warp_a[lane] : 0u), tied0 = __reduce_add_sync(0xffffffffu, lane < wid ? sh.warp_b[lane] : 0u);
  if (kCluster) {
    if (tid == kThreads - 1) { sh.counts[0] = over0 + over; sh.counts[1] = tied0 + tied; }
    cluster_sync_all();
    unsigned x = 0, y = 0;
    if (lane < rank) { x = pick_peer_load(&sh.counts[0], lane); y = pick_peer_load(&sh.counts[1], lane); }
    over0 += __reduce_add_sync(0xffffffffu, x);
    tied0 += __reduce_add_sync(0xffffffffu, y);
  }
#pragma unroll 4
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < s1 ? (pick_key(scores[i]) - least) >> shift : 0u, below = (1u << lane) - 1u;
    const unsigned more = __ballot_sync(0xffffffffu, i < s1 && k > prefix), same = __ballot_sync(0xffffffffu, i < s1 && k == prefix);
    const unsigned o = over0 + __popc(more & below), t = tied0 + __popc(same & below);
    const bool kept = (more >> lane & 1u) || ((same >> lane & 1u) && t < want);
    if (kept) out[o + min(t, want)] = first + a0 + i;
    over0 += __popc(more);
    tied0 += __popc(same);
  }
}

// A cluster of `parts` blocks per row of runs and key head; each scores a share of the pages, a warp 16 at a time. Pages are rows of the product
// and queries (with their heads) its columns, eight a tile: groups of up to eight heads fill one, and the maximum over them is two exchanges. The bounds of the
// next 16 pages are on their way into registers while some are multiplied. One token of 16 sequences of 2000 to 6000 tokens, 32 heads on 8: 6.7 us, of which the
// loads' latencies one after the other (length, page number, bounds) and the choice's barriers are the most; 16.8 with queries as
// rows, 256 threads and digits of 8 bits. One token behind 131072, 64 heads on 8: 14.9 us, the cluster's counts among them (1.2 TB/s).
template <int D>
__global__ void __launch_bounds__(kPickThreads, 1) pick_pages_kernel(const PickParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t pick_smem[];
  PickShared& sh = *reinterpret_cast<PickShared*>(pick_smem);
  constexpr int kPitch = 2 * D + 64;      // of a query's codes: rows of eight lanes keep apart in the banks
  constexpr int kC = 2 * D / 64, kRow = 2 * D + kBoundsTail;
  uint8_t* codes = pick_smem + (sizeof(PickShared) + 15) / 16 * 16;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, group = p.hq / p.hkv;
  const int row = blockIdx.x / p.parts, rank = blockIdx.x % p.parts, h = blockIdx.y;
  const int tiles = (p.run * group + 7) / 8;
  float* scores = reinterpret_cast<float*>(codes + tiles * 8 * kPitch);
  int* out = p.out + (static_cast<long long>(row) * p.hkv + h) * p.width;
  PickRange x{pick_run(p, row), 0};
  if (!pick_range(p, out, rank == 0, x)) return;                 // (alike in all blocks of a cluster)
  const RunOfRow& r = x.run;

  // ---- the first bounds on their way
  const int per = (x.n + p.parts - 1) / p.parts, a0 = min(x.n, rank * per), mine = min(x.n, a0 + per) - a0;
  const int* ids = p.block_table + static_cast<long long>(r.seq) * p.max_pages + p.first + a0;
  const int g = lane >> 2, kq = lane & 3;
  constexpr int kAll = kPickWarps * kPickStep;
  // of pages g and g + 8 of a step; channels are taken in an order of their own, 16 bytes a lane of every 64: sums do not mind
  int id[2];
  const auto load_ids = [&](int base) {
#pragma unroll
    for (int i = 0; i < 2; ++i) id[i] = ids[min(base + i * 8 + g, mine - 1)];
  };
  const auto load_bounds = [&](uint4 (&to)[2][kC], float (&u)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool ok = id[i] >= 0 && id[i] < p.pages;
      if (!ok) report_status(p.status, kBadArgument, kKernelPicked, 2, static_cast<uint32_t>(r.seq));
      const uint8_t* src = p.bounds + (static_cast<long long>(ok ? id[i] : 0) * p.hkv + h) * kRow;
#pragma unroll
      for (int c = 0; c < kC; ++c) to[i][c] = __ldg(reinterpret_cast<const uint4*>(src + c * 64 + kq * 16));
      u[i] = ok ? bounds_pow2(min(50, max(-50, static_cast<int>(__ldg(src + 2 * D)) - kBoundsBias))) : 0.f;
    }
  };
  uint4 a[2][kC];
  float unit[2];
  int base = wid * kPickStep;
  if (base < mine) {
    load_ids(base);
    load_bounds(a, unit);
    load_ids(base + kAll);
  }

  for (int i = threadIdx.x; i < kPickBins / 4; i += kPickThreads) reinterpret_cast<uint4*>(sh.hist)[i] = make_uint4(0u, 0u, 0u, 0u);

  // ---- codes of the queries: a+ against the largest values, a- against the smallest
  for (int i = wid; i < tiles * 8; i += kPickWarps) {
    constexpr int kEach = D / 32;
    // (rows that pad, and queries in front of the first key, repeat one that counts)
    const int token = min(max(i / group, -r.begin), r.tokens - 1);
    float v[kEach], amax = 0.f;
    const __nv_bfloat16* src = p.q + (static_cast<long long>(r.q_off + token) * p.hq + h * group + i % group) * D + lane * kEach;
#pragma unroll
    for (int k = 0; k < kEach; k += 2) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + k));
      v[k] = f.x == f.x ? f.x : 0.f;
      v[k + 1] = f.y == f.y ? f.y : 0.f;
      amax = fmaxf(amax, fmaxf(fabsf(v[k]), fabsf(v[k + 1])));
    }
    const int e = bounds_exponent(warp_max(amax));
    const float f = bounds_pow2(-e);
    uint32_t up = 0, down = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int c = pick_code(v[k], f);
      up |= static_cast<uint32_t>(max(c, 0)) << (8 * k);
      down |= (static_cast<uint32_t>(min(c, 0)) & 0xffu) << (8 * k);
    }
    uint8_t* dst = codes + i * kPitch + lane * kEach;
    if (kEach == 4) {
      *reinterpret_cast<uint32_t*>(dst) = up;
      *reinterpret_cast<uint32_t*>(dst + D) = down;
    } else {
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(up);
      *reinterpret_cast<uint16_t*>(dst + D) = static_cast<uint16_t>(down);
    }
    if (lane == 0) sh.row[i] = bounds_pow2(e);
  }
  if (p.parts > 1) cluster_sync_all();          // (the peers' memory is there)
  else __syncthreads();

  // ---- scores of this block's share
  unsigned least = 0xffffffffu, most = 0u;
  for (; base < mine; base += kAll) {
    uint4 next[2][kC];
    float next_unit[2];
    if (base + kAll < mine) {
      load_bounds(next, next_unit);
      load_ids(base + 2 * kAll);
    }
    float best[2] = {-INFINITY, -INFINITY};
    for (int t = 0; t < tiles; ++t) {
      int acc[2][4];                           // even and odd halves of the channels
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0;
      const uint8_t* src = codes + (t * 8 + g) * kPitch + kq * 16;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const uint4 b = *reinterpret_cast<const uint4*>(src + c * 64);
        mma_s8_16832(acc[0], a[0][c].x, a[1][c].x, a[0][c].y, a[1][c].y, b.x, b.y);
        mma_s8_16832(acc[1], a[0][c].z, a[1][c].z, a[0][c].w, a[1][c].w, b.z, b.w);
      }
      const float2 f = *reinterpret_cast<const float2*>(sh.row + t * 8 + 2 * kq);      // of queries 2 kq and 2 kq + 1
#pragma unroll
      for (int i = 0; i < 2; ++i)
        best[i] = fmaxf(best[i], fmaxf(pick_float(acc[0][2 * i] + acc[1][2 * i]) * f.x,
                                       pick_float(acc[0][2 * i + 1] + acc[1][2 * i + 1]) * f.y));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
      best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
      const int at = base + i * 8 + g;
      if (kq == 0 && at < mine) {
        const float score = unit[i] > 0.f ? best[i] * unit[i] : -INFINITY;
        const unsigned k = pick_key(score);
        least = min(least, k);
        most = max(most, k);
        scores[at] = score;
      }
    }
    if (base + kAll < mine) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unit[i] = next_unit[i];
#pragma unroll
        for (int c = 0; c < kC; ++c) a[i][c] = next[i][c];
      }
    }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  const int slot = rank * kPickWarps + wid;
  if (p.parts > 1) {
    if (lane < p.parts) {
      pick_peer_store(sh.least + slot, lane, least);
      pick_peer_store(sh.most + slot, lane, most);
    }
    cluster_sync_all();
  } else {
    if (lane == 0) {
      sh.least[slot] = least;
      sh.most[slot] = most;
    }
    __syncthreads();
  }
  least = 0xffffffffu;
  most = 0u;
  for (int i = lane; i < p.parts * kPickWarps; i += 32) {
    least = min(least, sh.least[i]);
    most = max(most, sh.most[i]);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (p.parts > 1) {
    pick_select<true, kPickThreads>(sh, threadIdx.x, 0, scores, mine, a0, rank, p.parts, p.top, least, most, p.first, out + p.first);
    cluster_sync_all();                        // nobody leaves while a peer may still read its words
  } else {
    pick_select<false, kPickThreads>(sh, threadIdx.x, 0, scores, mine, 0, 0, 1, p.top, least, most, p.first, out + p.first);
  }
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

// The same for runs whose queries (with their heads) are many, on the 5th-generation tensor cores: a block scores 128 pages at a time for two neighbouring
// runs of a sequence, up to 128 queries each. Pages are rows of the product, so a thread of the epilogue owns a page and takes the maximum over a run's queries by itself.
//   warp 0        TMA producer: the codes of 128 pages into one of three stages, four pages a gather
//   warp 1        one thread issues the products
//   warp 3        rows of no run
//   warps 8..15   scores: a page a thread, its 16 to 128 sums of one of the runs from one of two halves of TMEM; then half of the block chooses for each run
// 2048 queries of 64 heads on 8, runs of 16, behind 30720: 135 us, 3.5 blocks a processor one after the other. A block takes about 11 us for its start, the coding of
// the queries and the choice, and 1.4 a tile: the way from a gather (16 bytes of such rows a processor and cycle) over products and TMEM to the maxima, whose instructions are 0.4 of
// them. A tile serves two runs (one: 218 us; mma.sync, whose 8-bit products have a fifth of the rate, 307); loads of 32 columns ahead of the maxima 159, a fourth stage 150, gathers
// from rows of 256 bytes 150, all against 146.
constexpr int kPtThreads = 512, kPtTile = 128, kPtStages = 3;

struct PickTcShared {
  uint64_t a_full[kPtStages], a_empty[kPtStages], s_full[2], s_empty[2];
  uint64_t drain;                   // all products have been carried out
  uint32_t tmem_base, abort_flag;
};

// Four rows of a tensor of bytes, 128 of each from column c on; completion counts bytes on `bar`.
__device__ __forceinline__ void pick_gather4(void* dst, const CUtensorMap* m, uint64_t* bar, int c, const int (&row)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3])
      : "memory");
}

template <int D>
__global__ void __launch_bounds__(kPtThreads, 1) pick_pages_tc_kernel(const PickParams p, const __grid_constant__ CUtensorMap tm) {
  pdl_wait();
  extern __shared__ uint8_t pick_raw[];
  constexpr int kAtoms = 2 * D / 128, kRow = 2 * D + kBoundsTail, kStage = kPtTile * 2 * D, kAtom = 2 * kPickRows * 128;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pick_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, group = p.hq / p.hkv;
  const int pair = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv, cols = (p.run * group + 15) & ~15;
  uint8_t* stages = smem;                                    // [3][atom][128 pages][128 bytes]; the choice works here afterwards
  uint8_t* codes = stages + kPtStages * kStage;              // [atom][256 queries][128 bytes]
  float* factor = reinterpret_cast<float*>(codes + kAtoms * kAtom);              // of a query: 2^e
  PickTcShared& bars = *reinterpret_cast<PickTcShared*>(factor + 2 * kPickRows);
  float* scores = reinterpret_cast<float*>(&bars + 1);       // [2][pages]
  const auto out_of = [&](int i) { return p.out + (static_cast<long long>(i) * p.hkv + h) * p.width; };
  // rows of no run: one warp of a block looks some up, beside the others' work
  const auto leave_out = [&] {
    for (int row = pair; row < p.rows; row += p.pairs) {
      if (pick_run(p, row).tokens > 0) continue;
      for (int i = lane; i < p.width; i += 32) out_of(row)[i] = -1;
    }
  };
  // the runs of this block: two neighbouring ones of a sequence, which are one of twice as many queries
  PickRange x[2];
  int rows[2], runs = 0;
  {
    PickRange y{pick_run(p, pair, 2), 0};
    RunOfRow& r = y.run;
    const int first_q = p.cu_q ? p.cu_q[r.seq] : r.seq, rest = r.tokens - p.run;
    const int row = static_cast<int>((first_q + static_cast<long long>(r.seq) * (p.run - 1)) / p.run) + (r.q_off - first_q) / p.run;
    r.tokens = min(r.tokens, p.run);
    if (r.tokens > 0 && pick_range(p, out_of(row), true, y)) { x[runs] = y; rows[runs++] = row; }
    if (rest > 0) {
      r.q_off += p.run;
      r.begin += p.run;
      r.tokens = rest;
      if (pick_range(p, out_of(row + 1), true, y)) { x[runs] = y; rows[runs++] = row + 1; }
    }
    if (runs == 0) {
      if (wid == 3) leave_out();
      return;
    }
    if (runs == 1) { x[1] = x[0]; rows[1] = rows[0]; }
  }
  const int n = max(x[0].n, x[1].n), n_tiles = (n + kPtTile - 1) / kPtTile;
  const int* ids = p.block_table + static_cast<long long>(x[0].run.seq) * p.max_pages + p.first;

  // the queries on their way: D / 8 lanes a query, 16 bytes each
  constexpr int kQLanes = D / 8, kQueries = 32 / kQLanes, kRounds = kPickRows / (16 * kQueries);
  const int u = lane % kQLanes, inverse = (65536 + group - 1) / group;      // i / group for i < 128 is a product and a shift
  uint4 raw[2][kRounds];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const RunOfRow& r = x[w].run;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      // (rows that pad, and queries in front of the first key, repeat one that counts)
      const int i = (k * 16 + wid) * kQueries + lane / kQLanes, at = i * inverse >> 16, token = min(max(at, -r.begin), r.tokens - 1);
      raw[w][k] = __ldg(reinterpret_cast<const uint4*>(p.q + (static_cast<long long>(r.q_off + token) * p.hq + h * group + i - at * group) * D + u * 8));
    }
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPtStages; ++i) {
      mbar_init(&bars.a_full[i], 4);
      mbar_init(&bars.a_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.s_empty[i], 4 * runs);
    }
    mbar_init(&bars.drain, 1);
    bars.abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm);
  }
  if (wid == 2) {
    tmem_alloc(&bars.tmem_base, 512);
    tmem_relinquish();
  }
  volatile uint32_t* abort_flag = &bars.abort_flag;
  __syncthreads();
  pdl_trigger();                                             // (not before this block has its TMEM: a kernel that starts early may take what it waits for, and wait for this grid)
  // rows of the pool of bounds: of four neighbouring pages of a tile (one that is no page lies behind the end and arrives as zeros)
  const int quad = (wid & 3) * 8 + (lane & 7);
  const auto rows_of = [&](int j, int (&to)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = ids[min(j * kPtTile + quad * 4 + i, n - 1)];
      to[i] = id >= 0 && id < p.pages ? id * p.hkv + h : static_cast<int>(p.pages * p.hkv);
    }
  };
  const auto gather = [&](int j, const int (&from)[4]) {
    const int s = j % kPtStages;
    if (lane == 0) mbar_arrive_expect_tx(&bars.a_full[s], kStage / 4);
    __syncwarp();
    if (lane < 8) {
#pragma unroll
      for (int a = 0; a < kAtoms; ++a) pick_gather4(stages + s * kStage + a * (kPtTile * 128) + quad * 512, &tm, &bars.a_full[s], a * 128, from);
    }
  };
  int next[4];
  if (wid >= 4 && wid < 8) {                                 // the first tiles are on their way while the queries are coded
    int from[kPtStages][4];
#pragma unroll
    for (int j = 0; j < kPtStages; ++j) rows_of(min(j, n_tiles - 1), from[j]);
    rows_of(kPtStages < n_tiles ? kPtStages : 0, next);
#pragma unroll
    for (int j = 0; j < kPtStages; ++j)
      if (j < n_tiles) gather(j, from[j]);
  }

  // ---- codes of the queries
  {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (w >= runs) break;
#pragma unroll
      for (int k = 0; k < kRounds; ++k) {
        const int i = (k * 16 + wid) * kQueries + lane / kQLanes, at = w * cols + i;
        const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw[w][k]);
        float v[8], amax = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 f = __bfloat1622float2(b[y]);
          v[2 * y] = f.x == f.x ? f.x : 0.f;
          v[2 * y + 1] = f.y == f.y ? f.y : 0.f;
          amax = fmaxf(amax, fmaxf(fabsf(v[2 * y]), fabsf(v[2 * y + 1])));
        }
#pragma unroll
        for (int o = kQLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int e = bounds_exponent(amax);
        const float f = bounds_pow2(-e);
        uint2 up = make_uint2(0u, 0u), down = make_uint2(0u, 0u);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int c = pick_code(v[y], f), d = pick_code(v[4 + y], f);
          up.x |= static_cast<uint32_t>(max(c, 0)) << (8 * y);
          down.x |= (static_cast<uint32_t>(min(c, 0)) & 0xffu) << (8 * y);
          up.y |= static_cast<uint32_t>(max(d, 0)) << (8 * y);
          down.y |= (static_cast<uint32_t>(min(d, 0)) & 0xffu) << (8 * y);
        }
        if (i >= cols) continue;
        const auto place = [&](int byte) {
          return reinterpret_cast<uint2*>(codes + (byte >> 7) * kAtom + at * 128 + ((((byte >> 4) & 7) ^ (at & 7)) << 4) + (byte & 15));
        };
        *place(u * 8) = up;
        *place(D + u * 8) = down;
        if (u == 0) factor[at] = bounds_pow2(e);
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);
  unsigned least = 0xffffffffu, most = 0u;

  if (wid >= 4 && wid < 8) {
    bool ok = true;
    int sent = min(kPtStages, n_tiles);
    const auto read = [&](int j) {                           // whether the products of tile j have read its stage
      return __all_sync(0xffffffffu, mbar_wait(&bars.a_empty[j % kPtStages], static_cast<uint32_t>((j / kPtStages) & 1), abort_flag)) != 0;
    };
    for (; sent < n_tiles && (ok = read(sent - kPtStages)); ++sent) {
      gather(sent, next);
      if (sent + 1 < n_tiles) rows_of(sent + 1, next);
    }
    for (int j = max(0, n_tiles - kPtStages); j < n_tiles && ok; ++j) ok = read(j);      // until the last tiles have been read, or somebody gives up
    if (!ok) {
      if (lane == 0) report_status(p.status, kWaitTimeout, kKernelPicked, 22, blockIdx.x);
      // copies on their way land before the shared memory is given back
      uint32_t none = 0;
      for (int i = max(0, sent - kPtStages); i < sent; ++i) mbar_wait(&bars.a_full[i % kPtStages], static_cast<uint32_t>((i / kPtStages) & 1), &none);
    }
  } else if (wid == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc(128, runs * cols, kFmtS8, kFmtS8, 2);
      for (int j = 0; j < n_tiles; ++j) {
        const int s = j % kPtStages;
        if (!mbar_wait(&bars.a_full[s], static_cast<uint32_t>((j / kPtStages) & 1), abort_flag) ||
            (j >= 2 && !mbar_wait(&bars.s_empty[j & 1], static_cast<uint32_t>(((j >> 1) - 1) & 1), abort_flag))) {
          report_status(p.status, kWaitTimeout, kKernelPicked, 23, blockIdx.x);
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int a = 0; a < kAtoms; ++a) {
          const uint64_t ad = make_desc_sw128(smem_u32(stages + s * kStage + a * (kPtTile * 128)));
          const uint64_t bd = make_desc_sw128(smem_u32(codes + a * kAtom));
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_i8_ss(tmem_base + (j & 1) * 256, ad + 2 * k, bd + 2 * k, idesc, (a | k) != 0);
        }
        tc_commit(&bars.s_full[j & 1]);
        tc_commit(&bars.a_empty[s]);
      }
      // no product reads shared memory or writes TMEM when they are given back, whoever gave up
      uint32_t none = 0;
      tc_commit(&bars.drain);
      mbar_wait(&bars.drain, 0, &none);
    }
    __syncwarp();
  } else if (wid == 3) {
    leave_out();
  } else if (wid >= 8 && wid < 8 + 4 * runs) {
    const int w = (wid - 8) >> 2, mine = threadIdx.x & 127;  // run, page of a tile = TMEM lane
    const uint32_t column = tmem_base + (static_cast<uint32_t>((wid & 3) * 32) << 16) + w * cols;
    const float* const mult = factor + w * cols;
    float* const to = scores + w * p.max_pages;
    // the exponent of the tile's page, one tile ahead, and the page's number two ahead
    const int count = x[w].n;
    const auto id_of = [&](int j) { return ids[min(j * kPtTile + mine, count - 1)]; };
    // (a loaded value is first looked at a tile later: a test of it here would wait for it)
    const auto exponent_of = [&](int id) {
      return static_cast<int>(__ldg(p.bounds + (static_cast<long long>(id >= 0 && id < p.pages ? id : 0) * p.hkv + h) * kRow + 2 * D));
    };
    int id = id_of(0), behind = id_of(1), exponent = exponent_of(id);
    for (int j = 0; j < n_tiles; ++j) {
      const int ahead = exponent_of(behind), far = id_of(j + 2);
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.s_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag))) {
        if (lane == 0) report_status(p.status, kWaitTimeout, kKernelPicked, 24, blockIdx.x);
        break;
      }
      tc_fence_after_sync();
      float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      // 64 columns a time (those behind the run's are read, not used; the last ones end with TMEM)
      for (int c0 = 0; c0 < cols; c0 += 64) {
        uint32_t s[64];
        tmem_ld_32x32(column + (j & 1) * 256 + c0, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        if (c0 + 32 < cols) tmem_ld_32x32(column + (j & 1) * 256 + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld_wait();
        if (c0 + 64 >= cols) {                               // the products of the tile after the next may take these columns
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.s_empty[j & 1]);
        }
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          if (i % 16 == 0 && c0 + i >= cols) break;
          const float4 f = *reinterpret_cast<const float4*>(mult + c0 + i);
          const float2 a = pick_scaled2(static_cast<int>(s[i]), static_cast<int>(s[i + 1]), make_float2(f.x, f.y));
          const float2 b = pick_scaled2(static_cast<int>(s[i + 2]), static_cast<int>(s[i + 3]), make_float2(f.z, f.w));
          best[(i >> 1) & 2] = fmaxf(best[(i >> 1) & 2], fmaxf(a.x, a.y));
          best[((i >> 1) & 2) + 1] = fmaxf(best[((i >> 1) & 2) + 1], fmaxf(b.x, b.y));
        }
      }
      const int at = j * kPtTile + mine;
      if (at < count) {
        const bool ok = id >= 0 && id < p.pages;
        if (!ok) report_status(p.status, kBadArgument, kKernelPicked, 2, static_cast<uint32_t>(x[0].run.seq));
        const float unit = bounds_pow2(min(50, max(-50, exponent - kBoundsBias)));
        const float score = ok ? fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])) * unit : -INFINITY;
        const unsigned k = pick_key(score);
        least = min(least, k);
        most = max(most, k);
        to[at] = score;
      }
      exponent = ahead;
      id = behind;
      behind = far;
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (wid == 2) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
  const int w = wid >> 3;                                    // the run that this half of the block chooses for
  if (*abort_flag) {                                         // nothing is chosen
    if (w < runs)
      for (int i = threadIdx.x & 255; i < p.top; i += 256) out_of(rows[w])[p.first + i] = -1;
    return;
  }
  PickShared* sh = reinterpret_cast<PickShared*>(stages);    // [2] (the last products have been waited for)
  for (int i = threadIdx.x & 255; i < kPickBins / 4; i += 256) reinterpret_cast<uint4*>(sh[w].hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (wid >= 8 && lane == 0) {
    sh[(wid - 8) >> 2].least[wid & 3] = least;
    sh[(wid - 8) >> 2].most[wid & 3] = most;
  }
  __syncthreads();
  if (w >= runs) return;
  least = __reduce_min_sync(0xffffffffu, sh[w].least[lane & 3]);
  most = __reduce_max_sync(0xffffffffu, sh[w].most[lane & 3]);
  pick_select<false, 256>(sh[w], threadIdx.x & 255, 1 + w, scores + w * p.max_pages, x[w].n, 0, 0, 1, p.top, least, most, p.first, out_of(rows[w]) + p.first);
}

template <int D>
static int launch_pick_tc(const PickParams& p, int smem, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (configured.first_time() && cudaFuncSetAttribute(pick_pages_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return -200;
  CUtensorMap tm;
  const int rc = make_kmajor_map(&tm, p.bounds, 1, p.pages * p.hkv, 2 * D, 2 * D + kBoundsTail, 1);
  if (rc) return rc;
  const cudaError_t e = launch_pdl(pick_pages_tc_kernel<D>, dim3(static_cast<unsigned>(p.pairs) * p.hkv), dim3(kPtThreads), smem, stream, p, tm);
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
                             int rows, int tokens, int hq, int hkv, int d, int page, int max_pages, long long pages, int run, int top, int first, int last,
                             int width, void* status, cudaStream_t stream) {
  if (rows <= 0 || seqs <= 0) return 0;
  PickParams p{};
  p.page_shift = picked_page_shift(page);
  if (p.page_shift < 0 || hkv < 1 || hq < 1 || hq % hkv || pages < 1 || max_pages < 1 || (d != 64 && d != 128) || hkv > 65535) return -2;
  if (run < 1 || static_cast<long long>(run) * (hq / hkv) > kPickRows || (!cu_q && (run != 1 || rows != seqs || tokens != seqs))) return -3;
  if (top < 0 || first < 0 || last < 1 || static_cast<long long>(first) + top + last + (run + page - 2) / page > width) return -5;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(bounds)) & 15) return -4;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.bounds = static_cast<const uint8_t*>(bounds);
  p.block_table = block_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
  p.out = out;
  p.pages = pages;
  p.seqs = seqs; p.rows = rows; p.tokens = tokens; p.hq = hq; p.hkv = hkv; p.run = run; p.max_pages = max_pages;
  p.top = top; p.first = first; p.last = last; p.width = width;
  p.status = static_cast<DeviceStatus*>(status);
  // Tiles of 128 queries pay from 17 on, once there are more rows than processors: below that the other kernel's blocks share a row, and few queries leave most
  // of a tile empty. us, tiles / mma.sync, heads of 128 (queries of a run, rows x key heads, pages): 8, 200, 200 11.8 / 12.0; 8, 1000, 200 42 / 38; 8, 1000, 1000 70 / 73;
  // 16, 1000, 200 42 / 40; 16, 1000, 1000 70 / 78; 24, 160, 1000 19 / 25; 24, 300, 500 25 / 25; 32, 600, 270 33 / 34; 32, 2000, 1920 182 / 285; 64, 304, 270 23 / 25;
  // 64, 64, 1880 28 / 21; 128, 152, 270 15 / 25; 128, 32, 1880 33 / 21; 128, 504, 1920 67 / 157; heads of 64: 28, 500, 1920 43 / 62; 56, 76, 270 12 / 9;
  // 112, 126, 1920 32 / 27.
  // The scores of two runs lie in shared memory, 8 bytes for every column of the block table, however few of them a sequence uses (how many that is only the device
  // knows): heads of 128 leave room for 8300 columns, and under wider tables the other kernel chooses (2048 queries of 64 heads behind 30720: 140 us under 8048 columns, 285 under 9048).
  const long long smem_tc = 1024 + (kPtStages * kPtTile + 2 * kPickRows) * 2 * d + 2 * kPickRows * 4 + static_cast<int>(sizeof(PickTcShared)) + 8ll * max_pages;
  if (run * (hq / hkv) > 16 && static_cast<long long>(rows) * hkv > num_sms() && smem_tc <= 232448 && static_cast<long long>(rows) * hkv < (1ll << 31) && pages * hkv < (1ll << 31)) {
    p.pairs = static_cast<int>((tokens + static_cast<long long>(seqs) * (2 * run - 1)) / (2 * run));
    return d == 128 ? launch_pick_tc<128>(p, static_cast<int>(smem_tc), stream) : launch_pick_tc<64>(p, static_cast<int>(smem_tc), stream);
  }
  const int fixed = (static_cast<int>(sizeof(PickShared)) + 15) / 16 * 16 + (run * (hq / hkv) + 7) / 8 * 8 * (2 * d + 64);
  // blocks of a row: as long as every processor has one at most and a block 256 pages to score; at least as many as hold the scores
  p.parts = 1;
  while (p.parts < 8 && static_cast<long long>(rows) * hkv * p.parts * 2 <= num_sms() && max_pages > p.parts * 256) p.parts *= 2;
  const auto scores = [&] { return 4ll * ((max_pages + p.parts - 1) / p.parts); };
  while (p.parts < 8 && fixed + scores() > 232448) p.parts *= 2;
  if (fixed + scores() > 232448) return -6;
  if (static_cast<long long>(rows) * p.parts >= (1ll << 31)) return -3;
  const int smem = fixed + static_cast<int>(scores());
  return d == 128 ? launch_pick<128>(p, rows, smem, stream) : launch_pick<64>(p, rows, smem, stream);
}
