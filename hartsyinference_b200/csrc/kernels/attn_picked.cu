// Attention over chosen pages (rows of page numbers: picked.cuh), for decoded tokens, a few queries, and runs of a prompt that have a cap or few columns.
//
// A block owns 8 or more columns, a column being a query head of a token of one run, all on one key head, and walks the chosen pages in units of
// 16 keys, every warp units of its own. Products are mma.sync with the keys as rows (S = K Q^T, O^T = V^T P^T): eight columns fill a tile of eight,
// and an accumulator of O costs half of what it would with columns as rows. K and V come straight from the pages into
// registers: the channels of K are taken in the order in which 16-byte loads deal them to the lanes (Q likewise; sums do not mind), those of V
// fall into tiles so that a lane's 16 bytes are four pairs of rows, which two neighbouring keys' words make by byte permutes. P is turned by
// movmatrix. Nothing goes through shared memory but Q and, once, the warps' results, so no barrier stands between a load and its use.
// Rows of up to 24 columns are walked by each warp alone (35 us for 16 x 5 tokens of 32 heads on 8, 20 columns, over 2112 keys, where the registers leave a
// processor one block; in blocks of fewer columns, each reading all pages, 46), longer ones by two or four warps at a time, each with columns of its own, over the
// same units: their loads of a unit are asked for about the same time, and nothing is kept for them but in L2.
// Maxima and sums are in 32 bits, of unrounded probabilities. P is rounded to bf16 once, since the second product takes what V is held in: at most 2^-8 of a
// probability, which leaves results up to 0.0022 of their norm from 64 bits where their own rounding leaves 0.0017.
//
// A row whose pages are too many for one block's warps is shared by a cluster of up to eight blocks (every eighth page each), which meet
// through distributed shared memory: one launch, no scratch.
//
// One token of 64 sequences, 64 heads on 8, 2096 keys each: 89 us, 6.2 TB/s of keys and values. One token behind 131001, 32 heads on 8, 4096 keys: 11.5 us, the
// latencies of pages chosen, page numbers, keys, values and the join one after the other.
#include <math.h>

#include "picked.cuh"

namespace b200 {

struct PickedParams {
  const __nv_bfloat16* q;      // [tokens][hq][D]
  const __nv_bfloat16 *k, *v;  // [pages][hkv][page][D]
  __nv_bfloat16* out;          // [tokens][hq][D]
  const int* picked;           // [rows][hkv][width]
  const int *block_table, *kv_lens, *cu_q;
  long long pages;
  int seqs, tokens, hq, hkv, run, page_shift, max_pages, width, parts, cap;
  float scale_log2, cap_in, cap_out;   // softcap: cap_out - 2 cap_out / (1 + 2^(cap_in s)), or cap_out = 0
  DeviceStatus* status;
};

constexpr int kPkThreads = 256, kPkWarps = 8;

__device__ __forceinline__ float pk_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pk_turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void pk_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 pk_load(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Whether one of two bf16 is not finite.
__device__ __forceinline__ bool pk_not_finite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ float pk_peer(const float* local, int block) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(block));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// Shared memory: list of pages, limits of the columns, Q; the results of warps, then of the block, lie over Q.
template <int D, int NT, int CG>
struct PkLayout {
  static constexpr int kCols = 8 * NT;                           // of a warp
  static constexpr int kAll = kCols * CG;                        // of the block
  static constexpr int kQPitch = 2 * D + 64;                     // bytes; eight lanes' pieces of 16 bytes keep apart
  static constexpr int kOPitch = D + 4;                          // floats
  static constexpr int kWarpO = kCols * kOPitch;                 // floats of a warp's O
  static constexpr int head(int cap) { return (cap * 8 + kAll * 4 + 15) / 16 * 16; }
  static constexpr int bytes(int cap) {
    const int q = kAll * kQPitch, join = kPkWarps * (kWarpO + 2 * kCols) * 4;
    return head(cap) + (q > join ? q : join);
  }
};

template <int D, int NT, int CG>
__global__ void __launch_bounds__(kPkThreads, NT == 1 ? 2 : 1) attn_picked_kernel(const PickedParams p) {
  pdl_wait();
  pdl_trigger();
  using L = PkLayout<D, NT, CG>;
  constexpr int kK = D / 32, kHalves = D / 64;
  extern __shared__ __align__(16) uint8_t pk_smem[];
  int2* list = reinterpret_cast<int2*>(pk_smem);                 // page id (-1: none), first key
  int* limits = reinterpret_cast<int*>(pk_smem + p.cap * 8);
  uint8_t* work = pk_smem + L::head(p.cap);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, g = lane >> 2, kq = lane & 3, group = p.hq / p.hkv;
  const int row = blockIdx.x / p.parts, rank = blockIdx.x % p.parts, h = blockIdx.y;
  const int mate = wid % CG, walker = wid / CG;                  // whose columns, whose units
  constexpr int kWalkers = kPkWarps / CG;
  const RunOfRow r = run_of_row(p.cu_q, p.kv_lens, p.seqs, p.run, row, static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x7fffffffll)), p.tokens);
  const int cols = r.tokens * group;
  if (r.tokens <= 0) return;                        // (alike in all blocks of a cluster)
  const int end = r.begin + r.tokens;                            // keys that the run's last query sees

  const int* mine = p.picked + (static_cast<long long>(row) * p.hkv + h) * p.width;
  const int n = (p.width - rank + p.parts - 1) / p.parts;        // every parts-th entry
  for (int i = threadIdx.x; i < n; i += kPkThreads) {
    const int at = mine[rank + i * p.parts];
    int id = -1;
    if (at >= 0 && at < p.max_pages && at <= (end - 1) >> p.page_shift) {
      id = p.block_table[static_cast<long long>(r.seq) * p.max_pages + at];
      if (id < 0 || id >= p.pages) {
        report_status(p.status, kBadArgument, kKernelPicked, 3, static_cast<uint32_t>(r.seq));
        id = -1;
      }
    }
    list[i] = make_int2(id, id < 0 ? 0 : at << p.page_shift);
  }
  for (int c = threadIdx.x; c < L::kAll; c += kPkThreads) limits[c] = c < cols ? r.begin + c / group + 1 : 0;
  for (int i = threadIdx.x; i < L::kAll * (D / 8); i += kPkThreads) {
    const int c = i / (D / 8), x = i - c * (D / 8);
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (c < cols) w = *reinterpret_cast<const uint4*>(p.q + (static_cast<long long>(r.q_off + c / group) * p.hq + h * group + c % group) * D + x * 8);
    *reinterpret_cast<uint4*>(work + c * L::kQPitch + x * 16) = w;
  }
  __syncthreads();

  const uint8_t* const mine_q = work + mate * L::kCols * L::kQPitch;
  const int* const mine_limits = limits + mate * L::kCols;
  const int free_keys = r.begin + mate * L::kCols / group + 1;   // keys that every column of the warp sees
  const int unit_shift = p.page_shift - 4, units = n << unit_shift;
  int lim[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[t][i] = mine_limits[t * 8 + 2 * kq + i];
  float o[kHalves][4][NT][4];                                    // [half][tile][columns][row g | row g + 8 of two columns]
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) { m[t][i] = -INFINITY; l[t][i] = 0.f; }
#pragma unroll
    for (int x = 0; x < kHalves; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[x][y][t][i] = 0.f;
  }
  // the warp's next unit at or after u: its offset in the pool and first key
  const auto next_unit = [&](int& u, long long& at, int& key0) {
    for (; u < units; u += kWalkers) {
      const int2 e = list[u >> unit_shift];
      const int sub = u & ((1 << unit_shift) - 1);
      key0 = e.y + sub * 16;
      if (e.x >= 0 && key0 < end) {
        at = (((static_cast<long long>(e.x) * p.hkv + h) << p.page_shift) + sub * 16) * D;
        return true;
      }
    }
    return false;
  };
  uint4 ka[2][kK];
  const auto load_k = [&](long long at) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kK; ++c) ka[i][c] = pk_load(p.k + at + (g + 8 * i) * D + c * 32 + kq * 8);
  };
  int u = walker, key0 = 0;
  long long at = 0;
  bool on = next_unit(u, at, key0);
  if (on) load_k(at);
  while (on) {
    uint4 vv[kHalves][4];                                        // keys 2 kq, 2 kq + 1, 2 kq + 8, 2 kq + 9
#pragma unroll
    for (int x = 0; x < kHalves; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) vv[x][i] = pk_load(p.v + at + (2 * kq + (i & 1) + (i >> 1) * 8) * D + x * 64 + g * 8);
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int c = 0; c < kK; ++c) {
        const uint4 b = *reinterpret_cast<const uint4*>(mine_q + (t * 8 + g) * L::kQPitch + c * 64 + kq * 16);
        pk_mma(s[t], ka[0][c].x, ka[1][c].x, ka[0][c].y, ka[1][c].y, b.x, b.y);
        pk_mma(s[t], ka[0][c].z, ka[1][c].z, ka[0][c].w, ka[1][c].w, b.z, b.w);
      }
    }
    const int key = key0;
    u += kWalkers;
    on = next_unit(u, at, key0);
    if (on) load_k(at);
    const bool masked = key + 16 > free_keys;
    uint32_t pb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p.cap_out > 0.f) {
          const float x = s[t][i] * p.cap_in, e = pk_exp2(x > 126.f ? 126.f : x);       // (NaN stays)
          s[t][i] = p.cap_out - __fdividef(2.f * p.cap_out, e + 1.f);
        } else {
          s[t][i] *= p.scale_log2;
        }
        if (masked && key + g + (i >> 1) * 8 >= lim[t][i & 1]) s[t][i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(s[t][i], s[t][2 + i]);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float to = fmaxf(m[t][i], mx), sub = to == -INFINITY ? 0.f : to, alpha = pk_exp2(m[t][i] - sub);
        m[t][i] = to;
        s[t][i] = pk_exp2(s[t][i] - sub);
        s[t][2 + i] = pk_exp2(s[t][2 + i] - sub);
        l[t][i] = l[t][i] * alpha + s[t][i] + s[t][2 + i];       // of this lane's keys
#pragma unroll
        for (int x = 0; x < kHalves; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            o[x][y][t][i] *= alpha;
            o[x][y][t][2 + i] *= alpha;
          }
      }
      pb[t][0] = pk_turn(pack_bf16x2(s[t][0], s[t][1]));
      pb[t][1] = pk_turn(pack_bf16x2(s[t][2], s[t][3]));
    }
    bool odd = false;
    if (masked) {
      // what lies behind the last key may be anything; a value that some columns do not see must be finite, or their zero times it is not
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at_key = key + 2 * kq + (i & 1) + (i >> 1) * 8;
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          uint4& w = vv[x][i];
          if (at_key >= end) w = make_uint4(0u, 0u, 0u, 0u);
          odd |= at_key >= free_keys && (pk_not_finite(w.x) || pk_not_finite(w.y) || pk_not_finite(w.z) || pk_not_finite(w.w));
        }
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
#pragma unroll
      for (int x = 0; x < kHalves; ++x) {
        const uint32_t *w0 = &vv[x][0].x, *w1 = &vv[x][1].x, *w2 = &vv[x][2].x, *w3 = &vv[x][3].x;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t a0 = __byte_perm(w0[y], w1[y], 0x5410), a1 = __byte_perm(w0[y], w1[y], 0x7632);
          const uint32_t a2 = __byte_perm(w2[y], w3[y], 0x5410), a3 = __byte_perm(w2[y], w3[y], 0x7632);
#pragma unroll
          for (int t = 0; t < NT; ++t) pk_mma(o[x][y][t], a0, a1, a2, a3, pb[t][0], pb[t][1]);
        }
      }
    } else {
      // one column at a time, over the values that it sees
#pragma unroll 1
      for (int c = 0; c < L::kCols; ++c) {
        const int seen = mine_limits[c];
        if (mate * L::kCols + c >= cols) break;
        uint32_t keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = key + 2 * kq + (i & 1) + (i >> 1) * 8 < seen ? 0xffffffffu : 0u;
#pragma unroll
        for (int x = 0; x < kHalves; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t w0 = (&vv[x][0].x)[y] & keep[0], w1 = (&vv[x][1].x)[y] & keep[1], w2 = (&vv[x][2].x)[y] & keep[2], w3 = (&vv[x][3].x)[y] & keep[3];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float one[4] = {0.f, 0.f, 0.f, 0.f};
              pk_mma(one, __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410), __byte_perm(w2, w3, 0x7632), pb[t][0], pb[t][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (t * 8 + 2 * kq + (i & 1) == c) o[x][y][t][i] += one[i];
            }
          }
      }
    }
  }

  // ---- the warps' results meet
  __syncthreads();                                               // Q is no longer read
  float* const wo = reinterpret_cast<float*>(work);              // [warps][columns][D + 4]
  float* const wm = wo + kPkWarps * L::kWarpO;                   // [warps][columns] maxima, then sums
  float* const wl = wm + kPkWarps * L::kCols;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[t][i];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      const int c = t * 8 + 2 * kq + i;
      if (g == 0) { wm[wid * L::kCols + c] = m[t][i]; wl[wid * L::kCols + c] = sum; }
      float* dst = wo + wid * L::kWarpO + c * L::kOPitch + g * 8;
#pragma unroll
      for (int x = 0; x < kHalves; ++x) {
        *reinterpret_cast<float4*>(dst + x * 64) = make_float4(o[x][0][t][i], o[x][0][t][2 + i], o[x][1][t][i], o[x][1][t][2 + i]);
        *reinterpret_cast<float4*>(dst + x * 64 + 4) = make_float4(o[x][2][t][i], o[x][2][t][2 + i], o[x][3][t][i], o[x][3][t][2 + i]);
      }
    }
  __syncthreads();
  // a thread owns neighbouring pairs of values of a column
  constexpr int kPairs = L::kAll * D / 2, kEach = (kPairs + kPkThreads - 1) / kPkThreads;
  float2 sums[kEach];
  float tops[kEach], totals[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kPkThreads + threadIdx.x, all = min(i / (D / 2), L::kAll - 1), x = i % (D / 2) * 2, c = all % L::kCols, first = all / L::kCols;
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWalkers; ++w) top = fmaxf(top, wm[(w * CG + first) * L::kCols + c]);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWalkers; ++w) {
      const int at = (w * CG + first) * L::kCols + c;
      const float mw = wm[at], lw = wl[at];
      if (mw == -INFINITY && lw == 0.f) continue;                // (NaN scores have no maximum, but a sum)
      const float f = pk_exp2(mw - (top == -INFINITY ? 0.f : top));
      const float2 y = *reinterpret_cast<const float2*>(wo + (w * CG + first) * L::kWarpO + c * L::kOPitch + x);
      sum.x += f * y.x;
      sum.y += f * y.y;
      total += f * lw;
    }
    sums[e] = sum;
    tops[e] = top;
    totals[e] = total;
  }
  const auto store = [&](int c, int x, float2 sum, float total) {
    if (c >= cols) return;
    const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;       // nothing seen: zeros; NaN stays
    *reinterpret_cast<uint32_t*>(p.out + (static_cast<long long>(r.q_off + c / group) * p.hq + h * group + c % group) * D + x) =
        pack_bf16x2(sum.x * inv, sum.y * inv);
  };
  if (p.parts == 1) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kPkThreads + threadIdx.x;
      if (i < kPairs) store(i / (D / 2), i % (D / 2) * 2, sums[e], totals[e]);
    }
    return;
  }
  // ---- and those of the blocks: each joins a share of the columns' values
  __syncthreads();
  float* const bm = wo + L::kAll * L::kOPitch;                   // [columns] maxima, then sums, behind the columns' values
  float* const bl = bm + L::kAll;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kPkThreads + threadIdx.x;
    if (i >= kPairs) continue;
    const int c = i / (D / 2), x = i % (D / 2) * 2;
    *reinterpret_cast<float2*>(wo + c * L::kOPitch + x) = sums[e];
    if (x == 0) { bm[c] = tops[e]; bl[c] = totals[e]; }
  }
  cluster_sync_all();
  for (int i = rank * kPkThreads + threadIdx.x; i < kPairs; i += p.parts * kPkThreads) {
    const int c = i / (D / 2), x = i % (D / 2) * 2;
    float top = -INFINITY, total = 0.f, ms[8];
    float2 sum = make_float2(0.f, 0.f);
    for (int k = 0; k < p.parts; ++k) {
      ms[k] = pk_peer(bm + c, k);
      top = fmaxf(top, ms[k]);
    }
    for (int k = 0; k < p.parts; ++k) {
      const float lk = pk_peer(bl + c, k);
      if (ms[k] == -INFINITY && lk == 0.f) continue;
      const float f = pk_exp2(ms[k] - (top == -INFINITY ? 0.f : top));
      sum.x += f * pk_peer(wo + c * L::kOPitch + x, k);
      sum.y += f * pk_peer(wo + c * L::kOPitch + x + 1, k);
      total += f * lk;
    }
    store(c, x, sum, total);
  }
  cluster_sync_all();                       // nobody leaves while a peer may still read its words
}

template <int D, int NT, int CG>
static int launch_picked(PickedParams p, int rows, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (configured.first_time() && cudaFuncSetAttribute(attn_picked_kernel<D, NT, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return -200;
  const long long blocks = static_cast<long long>(rows) * p.hkv, units = static_cast<long long>(p.width) << (p.page_shift - 4);
  // blocks of a row: as long as all fit the processors at once (two each where the registers allow it) and every warp has a unit of its own
  p.parts = 1;
  while (p.parts < 8 && blocks * p.parts * 2 <= (NT == 1 ? 2 : 1) * num_sms() && units > p.parts * (kPkWarps / CG)) p.parts *= 2;
  p.cap = (p.width + p.parts - 1) / p.parts;
  const int smem = PkLayout<D, NT, CG>::bytes(p.cap);
  if (smem > 232448) return -6;
  if (static_cast<long long>(rows) * p.parts >= (1ll << 31)) return -3;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * p.parts, p.hkv);
  cfg.blockDim = dim3(kPkThreads);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_picked_kernel<D, NT, CG>, p);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}

// Columns of a warp in eights, as few as hold the row's with one, two or four warps side by side.
template <int D>
static int launch_columns(const PickedParams& p, int rows, cudaStream_t stream) {
  const int eights = (p.run * (p.hq / p.hkv) + 7) / 8;
  if (eights <= 1) return launch_picked<D, 1, 1>(p, rows, stream);
  if (eights <= 2) return launch_picked<D, 2, 1>(p, rows, stream);
  if (eights <= 3) return launch_picked<D, 3, 1>(p, rows, stream);
  if (eights <= 4) return launch_picked<D, 2, 2>(p, rows, stream);
  if (eights <= 6) return launch_picked<D, 3, 2>(p, rows, stream);
  if (eights <= 8) return launch_picked<D, 2, 4>(p, rows, stream);
  if (eights <= 12) return launch_picked<D, 3, 4>(p, rows, stream);
  return launch_picked<D, 4, 4>(p, rows, stream);
}

}  // namespace b200

using namespace b200;

constexpr int kPickedWidth = 4096;

// Whether rows of `cols` columns (queries times heads of a group) go through the tensor-core tiles of attn_picked_tc.cu (1) or b200_attn_picked (0). A tile takes
// 128 rows whatever the columns, 40 us for 2112 keys with a processor to itself and 53 with another beside it (heads of 64: 34 and 42); here a block takes 10 us
// and 9 for every eight columns (7 and 5.3), and few rows are shared by several blocks. us, here / tiles, rows x key heads in front: heads of 128, 24 columns: 144 36 / 56,
// 192 65 / 57, 400 99 / 112; 40 columns: 32 39 / 41, 64 60 / 45, 144 63 / 57, 288 122 / 68; 64 columns: 16 33 / 41, 32 56 / 41, 400 283 / 116; 128 columns: 8 37 / 40,
// 16 53 / 41; heads of 64, 35 columns: 24 26 / 35, 48 39 / 35; 112 columns: 16 33 / 35, 24 54 / 35. Up to 16 columns there is little between the two from 200 rows on.
// (Sequences of one run, which leave every other row of the grid without one.) One query of each sequence, whose heads are the columns and whose rows all have a run:
// heads of 128, 24 columns: 144 34 / 48, 192 64 / 55; 64 columns: 16 43 / 39, 32 32 / 39, 148 97 / 50, 400 282 / 109; 128 columns: 8 35 / 39, 16 69 / 39, 300 420 / 104;
// heads of 64, 112 columns: 8 22 / 33, 24 32 / 33, 200 184 / 45.
B200_API int b200_attn_picked_form(int rows, int cols, int hkv, int d, int page, int width, long long pages, float scale, float softcap) {
  if (cols <= 16 || width > 1024 || !(scale > 0.f) || softcap > 0.f || pages * hkv * page >= (1ll << 31)) return 0;
  const double r = static_cast<double>(rows) * hkv, sms = num_sms(), keys = width * static_cast<double>(page) / 2112.;
  const int eights = (cols + 7) / 8, held = eights <= 4 ? eights : eights <= 6 ? 6 : eights <= 8 ? 8 : eights <= 12 ? 12 : 16;
  const double block = d == 128 ? 10. + 9. * held : 7. + 5.3 * held;
  const double here = 5. + keys * block * fmin(1., fmax(0.3, r * 3. / sms)) * ceil(r / sms);
  const double one = d == 128 ? 32. : 26., two = d == 128 ? 49. : 40.;
  const double tiles = 8. + keys * (r <= sms ? one + (two - one) * r / sms : two * ceil(r / (2. * sms)));
  return tiles < here;
}

// q, out [tokens][hq][d], k, v [pages][hkv][page][d] bf16; picked int32 [rows][hkv][width] (see picked.cuh), rows = (tokens + seqs (run - 1)) / run.
// Causal; entries below 0 or behind the run's last query are no pages. A page named twice counts twice.
B200_API int b200_attn_picked(const void* q, const void* k, const void* v, void* out, const int* picked, const int* block_table, const int* kv_lens,
                              const int* cu_q, int seqs, int rows, int tokens, int hq, int hkv, int d, int page, int max_pages, long long pages, int run,
                              int width, float scale, float softcap, void* status, cudaStream_t stream) {
  if (rows <= 0 || seqs <= 0 || tokens <= 0) return 0;
  PickedParams p{};
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
  if (p.page_shift < 0 || hkv < 1 || hkv > 65535 || hq < 1 || hq % hkv || pages < 1 || max_pages < 1 || (d != 64 && d != 128)) return -2;
  if (run < 1 || static_cast<long long>(run) * (hq / hkv) > 128 || (!cu_q && (run != 1 || rows != seqs || tokens != seqs))) return -3;
  if (width < 1 || width > kPickedWidth) return -5;
  uintptr_t all = 0;
  for (const void* x : {q, k, v, static_cast<const void*>(out)}) all |= reinterpret_cast<uintptr_t>(x);
  if (all & 15) return -4;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.picked = picked; p.block_table = block_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
  p.pages = pages;
  p.seqs = seqs; p.tokens = tokens; p.hq = hq; p.hkv = hkv; p.run = run; p.max_pages = max_pages; p.width = width;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cap_out = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
  p.cap_in = softcap > 0.f ? 2.f * scale / softcap * 1.4426950408889634f : 0.f;
  p.status = static_cast<DeviceStatus*>(status);
  return d == 128 ? launch_columns<128>(p, rows, stream) : launch_columns<64>(p, rows, stream);
}
