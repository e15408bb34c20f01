// Attention over chosen pages (picked.cuh) for runs of a prompt, and for single queries with many heads on a key head, on the 5th-generation tensor cores.
//
// One CTA owns one row of pages: the queries of a run times the heads of a group, up to 128 rows of Q, walk the keys of the pages that they chose
// together in tiles of 64. Rows have pages of their own, so two of them share nothing; two CTAs lie on a processor instead, and one's products
// run during the other's softmax.
//   warp 0       TMA producer: the Q tile (tokens x heads of the group, one box a half head), then per key tile one box per
//                page and half head of K and of V, read in place; what is no page starts past the end of the pool and arrives as zeros
//   warp 1       one thread issues every tcgen05.mma: S(j + 1) into one of two halves of TMEM ahead of O += P(j) V(j); P is written over S and
//                read from TMEM, V is consumed as it lies in the pages (an MN-major operand)
//   warp 2       in tiles with keys that not all rows see: clears the rows of V behind the last key (what a page held before may not be
//                finite, and its probability is zero), and rows with values that are not finite, which the rows that see them add by themselves
//   warps 4..7   softmax, one row per thread, lazy rescale: the running maximum is raised only when it grows by more than 2^8; sums in 32 bits, of unrounded
//                probabilities, which are rounded to bf16 once: the second product takes them in the type of V
//
// 2048 queries of 64 heads on 8, runs of 16, 2144 keys each behind 30720: 197 us (711 TFLOP/s; 1134 by mma.sync). Bound by the two CTAs' products and the softmax
// about equally: a product of 16 channels takes as long for 64 keys as for 128, since Q is read from shared memory for each. Tiles of 128 keys with one set of
// scores were slower all the same (244 us: neither hides the other within a CTA).
#include "picked.cuh"

namespace b200 {

int make_kmajor_map(CUtensorMap* out, const void* base, int elem_bytes, long long rows, long long k, long long ld, int box_rows);
int make_heads_map(CUtensorMap* out, const void* base, long long tokens, int heads, int d, int box_tokens, int box_heads);

constexpr int kTpThreads = 256;
constexpr int kTpTile = 64;               // keys
constexpr int kTpStages = 2;
constexpr int kTpRegisters = 128;         // of a thread at launch; the first four warps give 64 of them to the softmax warps
constexpr int kTpWidth = 1024;            // pages of a row that the list in shared memory holds
constexpr int kTpFar = 0x40000000;        // first key of what is no page
constexpr float kTpRescaleGap = 8.f;

struct TpBarriers {
  uint64_t q_full, k_full[kTpStages], k_empty[kTpStages], v_full[kTpStages], v_empty[kTpStages];
  uint64_t v_ask, v_clean;                // the V tile at hand has landed; its rows are cleared
  uint64_t s_full[2], p_ready[2], o_done, o_last;      // (o_done: of all products but the last)
  uint64_t drain;                         // all products have been carried out
  uint32_t tmem_base, abort_flag;
  int entries, free_entries, odd;         // pages up to the last real one; those in front of the first that not all rows see; whether there are keys that rows add by themselves
};

struct TpParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;          // [tokens][hq][D]
  const int* picked;           // [rows][hkv][width]
  const int *block_table, *kv_lens, *cu_q;
  long long pages;
  int seqs, tokens, hq, hkv, run, page_shift, box_shift, max_pages, width, pool_rows;
  float scale_log2;
  DeviceStatus* status;
};

__device__ __forceinline__ float tp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether one of two bf16 is not finite.
__device__ __forceinline__ bool tp_not_finite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

template <int D>
__global__ void __launch_bounds__(kTpThreads, 2)
attn_picked_tc_kernel(const TpParams p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v) {
  constexpr int kHalves = D / 64;
  constexpr int kQBytes = 128 * D * 2, kTileBytes = kTpTile * D * 2, kHalfBytes = kTpTile * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                                   // [half head][128 rows][128 bytes]
  uint8_t* sk = sq + kQBytes;
  uint8_t* sv = sk + kTpStages * kTileBytes;
  int2* list = reinterpret_cast<int2*>(sv + kTpStages * kTileBytes);      // row of the pool, first key
  TpBarriers* bars = reinterpret_cast<TpBarriers*>(list + p.width);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.hq / p.hkv;
  const int row_id = blockIdx.x, h = blockIdx.y;
  pdl_wait();
  const RunOfRow r = run_of_row(p.cu_q, p.kv_lens, p.seqs, p.run, row_id, static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x3fffffffll)), p.tokens);
  if (r.tokens <= 0) return;
  const int end = r.begin + r.tokens, real_rows = r.tokens * group;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->v_ask, 1);
    mbar_init(&bars->v_clean, 1);
    mbar_init(&bars->o_done, 1);
    mbar_init(&bars->o_last, 1);
    mbar_init(&bars->drain, 1);
    for (int i = 0; i < kTpStages; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->v_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_ready[t], 4);
    }
    bars->abort_flag = 0;
    bars->entries = 0;
    bars->free_entries = p.width;
    bars->odd = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 256);
    tmem_relinquish();
  }
  __syncthreads();
  {
    const int* mine = p.picked + (static_cast<long long>(row_id) * p.hkv + h) * p.width;
    int last = 0, partly = p.width;
    for (int i = threadIdx.x; i < p.width; i += kTpThreads) {
      const int at = mine[i];
      int2 e = make_int2(p.pool_rows, kTpFar);
      if (at >= 0 && at < p.max_pages && at <= (end - 1) >> p.page_shift) {
        const int id = p.block_table[static_cast<long long>(r.seq) * p.max_pages + at];
        if (id >= 0 && id < p.pages) {
          e = make_int2((id * p.hkv + h) << p.page_shift, at << p.page_shift);
          last = i + 1;
        } else {
          report_status(p.status, kBadArgument, kKernelPicked, 4, static_cast<uint32_t>(r.seq));
        }
      }
      list[i] = e;
      if (e.y + (1 << p.page_shift) > r.begin + 1) partly = min(partly, i);
    }
    last = __reduce_max_sync(0xffffffffu, last);
    partly = __reduce_min_sync(0xffffffffu, partly);
    if (lane == 0) {
      atomicMax(&bars->entries, last);
      atomicMin(&bars->free_entries, partly);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_trigger();                                        // (not before this block has its TMEM: a kernel that starts early may take what it waits for, and wait for this grid)
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int box = 1 << p.box_shift, per_page = p.page_shift - p.box_shift;      // boxes of a page, as a shift
  const int pieces = bars->entries << per_page, per_tile_shift = 6 - p.box_shift;
  const int n_tiles = (pieces + (1 << per_tile_shift) - 1) >> per_tile_shift;
  // place i in the list of all boxes: row of the pool and first key
  const auto piece = [&](int i) {
    if (i >= pieces) return make_int2(p.pool_rows, kTpFar);
    int2 e = list[i >> per_page];
    const int sub = (i & ((1 << per_page) - 1)) << p.box_shift;
    if (e.y != kTpFar) { e.x += sub; e.y += sub; }
    return e;
  };
  const int free_keys = r.begin + 1;                    // keys that every row sees
  // whether a tile has keys that some row does not see
  const int free_tiles = min(bars->free_entries << per_page, pieces) >> per_tile_shift;
  const auto masked = [&](int j) {
    if (j < free_tiles) return false;
    bool some = false;
    for (int i = 0; i < 1 << per_tile_shift; ++i) some |= piece((j << per_tile_shift) + i).y + box > free_keys;
    return some;
  };

  // launch: 128 registers a thread; the softmax group takes what the first group gives back
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
      // ----------------------------------------------------------------------- TMA producer
      bool ok = true;
      int k_sent = 0, v_sent = 0;
      if (lane == 0 && n_tiles > 0) {
        mbar_arrive_expect_tx(&bars->q_full, kHalves * p.run * group * 128);
        for (int a = 0; a < kHalves; ++a) tma_load_3d(sq + a * (kQBytes / kHalves), &tm_q, &bars->q_full, a * 64, h * group, r.q_off);
      }
      const int boxes = kHalves << per_tile_shift, i = lane / kHalves, half = lane % kHalves;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j % kTpStages;
        const uint32_t ph = static_cast<uint32_t>((j / kTpStages) & 1);
        const int2 e = lane < boxes ? piece((j << per_tile_shift) + i) : make_int2(0, 0);
        uint8_t* const at = sk + s * kTileBytes + half * kHalfBytes + (i << p.box_shift) * 128;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty[s], ph ^ 1, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->k_full[s], kTileBytes);
        __syncwarp();
        if (lane < boxes) tma_load_2d(at, &tm_k, &bars->k_full[s], half * 64, e.x);
        ++k_sent;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_empty[s], ph ^ 1, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->v_full[s], kTileBytes);
        __syncwarp();
        if (lane < boxes) tma_load_2d(at + (sv - sk), &tm_v, &bars->v_full[s], half * 64, e.x);
        ++v_sent;
      }
      for (int j = max(0, n_tiles - kTpStages); j < n_tiles && ok; ++j) {      // until the last tiles have been read, or somebody gives up
        const uint32_t ph = static_cast<uint32_t>((j / kTpStages) & 1);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty[j % kTpStages], ph, abort_flag) && mbar_wait(&bars->v_empty[j % kTpStages], ph, abort_flag));
      }
      if (!ok) {
        if (lane == 0) report_status(p.status, kWaitTimeout, kKernelPicked, 41, blockIdx.x);
        // copies on their way land before the shared memory is given back
        uint32_t none = 0;
        mbar_wait(&bars->q_full, 0, &none);
        for (int b = 0; b < kTpStages; ++b) {
          const int k_last = (k_sent - 1 - b) >= 0 ? k_sent - 1 - b : -1, v_last = (v_sent - 1 - b) >= 0 ? v_sent - 1 - b : -1;
          if (k_last >= 0) mbar_wait(&bars->k_full[k_last % kTpStages], static_cast<uint32_t>((k_last / kTpStages) & 1), &none);
          if (v_last >= 0) mbar_wait(&bars->v_full[v_last % kTpStages], static_cast<uint32_t>((v_last / kTpStages) & 1), &none);
        }
      }
    } else if (warp == 1) {
      // ----------------------------------------------------------------------- MMA issuer
      if (lane == 0 && n_tiles > 0) {
        constexpr uint32_t kIdescS = make_idesc(128, kTpTile, kFmtBf16, kFmtBf16);
        constexpr uint32_t kIdescPV = make_idesc(128, D, kFmtBf16, kFmtBf16) | kIdescBMn;
        bool ok = mbar_wait(&bars->q_full, 0, abort_flag);
        uint32_t asked = 0;
        // S(j) = Q K_j^T into TMEM columns [(j & 1) * 64, .. + 64)
        auto issue_s = [&](int j) {
          const int s = j % kTpStages;
          if (!mbar_wait(&bars->k_full[s], static_cast<uint32_t>((j / kTpStages) & 1), abort_flag)) return false;
          tc_fence_after_sync();
#pragma unroll
          for (int a = 0; a < kHalves; ++a) {
            const uint64_t ad = make_desc_sw128(smem_u32(sq + a * (kQBytes / kHalves)));
            const uint64_t bd = make_desc_sw128(smem_u32(sk + s * kTileBytes + a * kHalfBytes));
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_bf16_ss(tmem_base + (j & 1) * 64, ad + 2 * k, bd + 2 * k, kIdescS, (a | k) != 0);
          }
          tc_commit(&bars->s_full[j & 1]);
          tc_commit(&bars->k_empty[s]);
          return true;
        };
        if (ok) ok = issue_s(0);
        for (int j = 0; j < n_tiles && ok; ++j) {
          // S(j + 1) takes the columns of P(j - 1), whose product was issued before: products run in order
          if (j + 1 < n_tiles && !(ok = issue_s(j + 1))) break;
          const int s = j % kTpStages;
          if (!mbar_wait(&bars->v_full[s], static_cast<uint32_t>((j / kTpStages) & 1), abort_flag)) { ok = false; break; }
          if (masked(j)) {
            mbar_arrive(&bars->v_ask);
            if (!mbar_wait(&bars->v_clean, asked & 1, abort_flag)) { ok = false; break; }
            ++asked;
          }
          if (!mbar_wait(&bars->p_ready[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag)) { ok = false; break; }
          tc_fence_after_sync();
          // O += P(j) V_j: A = P in TMEM (16 keys are 8 columns of bf16 pairs), B = 16 rows of the V tile
          const uint64_t bd = make_desc_sw128_mn(smem_u32(sv + s * kTileBytes), kHalfBytes);
#pragma unroll
          for (int k = 0; k < kTpTile / 16; ++k)
            mma_bf16_ts(tmem_base + 128, tmem_base + (j & 1) * 64 + k * 8, bd + k * (2048 >> 4), kIdescPV, (j | k) != 0);
          tc_commit(j + 1 < n_tiles ? &bars->o_done : &bars->o_last);
          tc_commit(&bars->v_empty[s]);
        }
        if (!ok) report_status(p.status, kWaitTimeout, kKernelPicked, 42, blockIdx.x);
        // no product reads shared memory or writes TMEM when they are given back, whoever gave up
        uint32_t none = 0;
        tc_commit(&bars->drain);
        mbar_wait(&bars->drain, 0, &none);
      }
    } else if (warp == 2) {
      // ----------------------------------------------------------------------- rows of V that not all rows of P may touch
      // (told by the MMA thread: a waiter that has not seen every phase of v_full cannot tell which one it is in)
      uint32_t asked = 0;
      for (int j = 0; j < n_tiles; ++j) {
        if (!masked(j)) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->v_ask, asked & 1, abort_flag))) break;
        ++asked;
        uint8_t* tile = sv + (j % kTpStages) * kTileBytes;
        for (int i = 0; i < 1 << per_tile_shift; ++i) {
          const int2 e = piece((j << per_tile_shift) + i);
          if (e.y == kTpFar || e.y + box <= free_keys) continue;
          for (int c = max(0, free_keys - e.y); c < box; ++c) {
            // whole 128-byte rows, so the swizzle inside a row does not matter; eight lanes a half
            uint4* const at = reinterpret_cast<uint4*>(tile + (lane >> 3) * kHalfBytes + ((i << p.box_shift) + c) * 128) + (lane & 7);
            bool odd = false;
            if (lane < 8 * kHalves) {
              const uint4 w = *at;
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int u = 0; u < 4; ++u) odd |= tp_not_finite(x[u]);
            }
            odd = __any_sync(0xffffffffu, odd);
            if (e.y + c >= end || odd) {
              if (lane < 8 * kHalves) *at = make_uint4(0u, 0u, 0u, 0u);
              if (e.y + c < end && lane == 0) bars->odd = 1;
              __syncwarp();
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->v_clean);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------------------- softmax warps
    const int quarter = warp & 3;                         // TMEM lane quarter this warp may touch
    const int row = quarter * 32 + lane;                  // row of Q = TMEM lane
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t o_col = lane_base + 128;
    const int lim = row < real_rows ? r.begin + row / group + 1 : 0;        // keys this row sees
    float m_run = -INFINITY, l_run = 0.f;
    const float c = p.scale_log2;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const uint32_t s_col = lane_base + (j & 1) * 64;
      if (!__all_sync(0xffffffffu, mbar_wait(&bars->s_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag))) { ok = false; break; }
      tc_fence_after_sync();
      uint32_t x[64];
      tmem_ld_32x32(s_col, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
      tmem_ld_32x32(s_col + 32, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
      tmem_ld_wait();
      if (masked(j)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int place = (j << 6) + u * 16;            // of 16 keys of one page
          const int2 e = piece(place >> p.box_shift);
          const int valid = lim - e.y - (place & (box - 1));
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i >= valid) x[u * 16 + i] = 0xff800000u;
        }
      }
      float mf[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) mf[u] = __uint_as_float(x[u]);
#pragma unroll
      for (int i = 8; i < 64; ++i) mf[i & 7] = fmaxf(mf[i & 7], __uint_as_float(x[i]));
      const float mx = fmaxf(fmaxf(fmaxf(mf[0], mf[1]), fmaxf(mf[2], mf[3])), fmaxf(fmaxf(mf[4], mf[5]), fmaxf(mf[6], mf[7]))) * c;
      // raise the running maximum only when it would grow by more than the gap (or on the first tile);
      // a warp decides together because the O rescale below is a warp-wide TMEM access
      if (__any_sync(0xffffffffu, mx > m_run + kTpRescaleGap && row < real_rows)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_run == -INFINITY ? 0.f : tp_exp2(m_run - m_new);
        if (j > 0) {
          if (!__all_sync(0xffffffffu, mbar_wait(&bars->o_done, (j - 1) & 1, abort_flag))) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            tmem_ld_32x32(o_col + cc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32(o_col + cc * 32, o);
          }
          tmem_st_wait();
        }
        l_run *= alpha;
        m_run = m_new;
      }
      const float sub = m_run == -INFINITY ? 0.f : m_run;
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t packed[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float a = tp_exp2(fmaf(__uint_as_float(x[2 * i]), c, -sub));
        const float b = tp_exp2(fmaf(__uint_as_float(x[2 * i + 1]), c, -sub));
        sums[i & 3] += a + b;
        packed[i] = pack_bf16x2(a, b);
      }
      tmem_st_32x32(s_col, packed);                      // P: columns [0, 32) of S
      tmem_st_wait();
      l_run += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_ready[j & 1]);
    }
    // The last product has a barrier of its own, with a single phase: the last scores told of all products but two, and a warp that comes late
    // to o_done's last two phases finds both gone by, which looks like the first of them still to come.
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_last, 0, abort_flag));
    if (!ok) {
      if (lane == 0) report_status(p.status, kWaitTimeout, kKernelPicked, 43, blockIdx.x);
    } else {
      tc_fence_after_sync();
      const float inv = l_run > 0.f ? 1.f / l_run : l_run == 0.f ? 0.f : l_run;       // nothing seen: zeros; NaN stays
      const bool odd = *reinterpret_cast<volatile int*>(&bars->odd) != 0;
      // The Q tile is no longer read: 32 rows of 128 bytes per warp turn the rows that the lanes hold into
      // 128-byte runs. 16-byte pieces are placed by (piece xor row), which keeps the banks apart.
      uint8_t* strip = sq + quarter * 32 * 128;
#pragma unroll
      for (int hc = 0; hc < kHalves; ++hc) {
        uint32_t o[64];
        tmem_ld_32x32(o_col + hc * 64, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
        tmem_ld_32x32(o_col + hc * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
        tmem_ld_wait();
        // keys whose values are not all finite: this row's probability of them, once more (all that were cleared are looked for again, however
        // often their page is named)
        for (int n = odd ? free_tiles << per_tile_shift : pieces; n < pieces; ++n) {
          const int2 e = piece(n);
          if (e.y == kTpFar) continue;
          for (int sub = max(0, free_keys - e.y); sub < box && e.y + sub < lim; ++sub) {
            const __nv_bfloat16* vr = p.v + static_cast<long long>(e.x + sub) * D;
            bool some = false;
            for (int i = 0; i < D / 2; ++i) some |= tp_not_finite(reinterpret_cast<const uint32_t*>(vr)[i]);
            if (!some) continue;
            const __nv_bfloat16* qr = p.q + (static_cast<long long>(r.q_off + row / group) * p.hq + h * group + row % group) * D;
            const __nv_bfloat16* kr = p.k + static_cast<long long>(e.x + sub) * D;
            float s = 0.f;
            for (int i = 0; i < D; ++i) s += __bfloat162float(qr[i]) * __bfloat162float(kr[i]);
            const float w = tp_exp2(fmaf(s, c, -(m_run == -INFINITY ? 0.f : m_run)));
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + w * __bfloat162float(vr[hc * 64 + i]));
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            w[u] = n_tiles > 0 ? pack_bf16x2(__uint_as_float(o[i * 8 + 2 * u]) * inv, __uint_as_float(o[i * 8 + 2 * u + 1]) * inv) : 0u;
          *reinterpret_cast<uint4*>(strip + lane * 128 + ((i ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = i * 4 + (lane >> 3), at = lane & 7, mine = quarter * 32 + rr;
          const uint4 w = *reinterpret_cast<const uint4*>(strip + rr * 128 + ((at ^ (rr & 7)) * 16));
          if (mine < real_rows)
            *reinterpret_cast<uint4*>(p.out + (static_cast<long long>(r.q_off + mine / group) * p.hq + h * group + mine % group) * D + hc * 64 + at * 8) = w;
        }
        __syncwarp();
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 256);
  }
}

template <int D>
static int launch_picked_tc(const TpParams& p, int rows, int tokens, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  int rc = make_heads_map(&tq, p.q, tokens, p.hq, D, p.run, p.hq / p.hkv);
  if (rc == 0) rc = make_kmajor_map(&tk, p.k, 2, p.pool_rows, D, D, 1 << p.box_shift);
  if (rc == 0) rc = make_kmajor_map(&tv, p.v, 2, p.pool_rows, D, D, 1 << p.box_shift);
  if (rc) return rc;
  const int smem = 1024 + 128 * D * 2 + 2 * kTpStages * kTpTile * D * 2 + p.width * 8 + static_cast<int>(sizeof(TpBarriers));
  static PerDeviceOnce configured;
  if (configured.first_time() && cudaFuncSetAttribute(attn_picked_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 115712) != cudaSuccess) return -200;
  if (smem > 115712) return -6;
  static int registers;                   // of the kernel as it was built
  if (registers == 0) {
    cudaFuncAttributes has{};
    if (cudaFuncGetAttributes(&has, attn_picked_tc_kernel<D>) != cudaSuccess) return -200;
    registers = has.numRegs;
  }
  if (registers != kTpRegisters) return -8;      // the softmax warps would wait for registers that nobody gives back
  const cudaError_t e = launch_pdl(attn_picked_tc_kernel<D>, dim3(rows, p.hkv), dim3(kTpThreads), smem, stream, p, tq, tk, tv);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}

}  // namespace b200

using namespace b200;

// As b200_attn_picked (attn_picked.cu), for scale > 0 without a cap and up to 1024 pages a row; tokens: rows of q.
B200_API int b200_attn_picked_tc(const void* q, const void* k, const void* v, void* out, const int* picked, const int* block_table, const int* kv_lens,
                                 const int* cu_q, int seqs, int rows, int tokens, int hq, int hkv, int d, int page, int max_pages, long long pages, int run,
                                 int width, float scale, void* status, cudaStream_t stream) {
  if (rows <= 0 || seqs <= 0 || tokens <= 0) return 0;
  TpParams p{};
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
  if (p.page_shift < 0 || hkv < 1 || hkv > 65535 || hq < 1 || hq % hkv || pages < 1 || max_pages < 1 || (d != 64 && d != 128)) return -2;
  if (run < 1 || static_cast<long long>(run) * (hq / hkv) > 128 || (!cu_q && (run != 1 || rows != seqs || tokens != seqs))) return -3;
  if (width < 1 || width > kTpWidth || !(scale > 0.f)) return -5;
  const long long pool_rows = pages * hkv * page;
  if (pool_rows >= (1ll << 31)) return -7;
  uintptr_t all = 0;
  for (const void* x : {q, k, v, static_cast<const void*>(out)}) all |= reinterpret_cast<uintptr_t>(x);
  if (all & 15) return -4;
  p.box_shift = p.page_shift < 6 ? p.page_shift : 6;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.picked = picked; p.block_table = block_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
  p.pages = pages;
  p.seqs = seqs; p.tokens = tokens; p.hq = hq; p.hkv = hkv; p.run = run; p.max_pages = max_pages; p.width = width;
  p.pool_rows = static_cast<int>(pool_rows);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = static_cast<DeviceStatus*>(status);
  return d == 128 ? launch_picked_tc<128>(p, rows, tokens, stream) : launch_picked_tc<64>(p, rows, tokens, stream);
}
