// Attention of prompt chunks over a K/V cache held in 4 bits (format: kv4.cuh) on the 5th-generation tensor cores.
//
// The query heads of a group read the same keys, so rows are (query, head of the group) pairs of one sequence and one kv head, heads fastest: row
// r is query r / G, head r % G. A block owns two tiles of 128 rows and walks the keys that they see in tiles of 128:
//   warps 0, 1    a thread each issues the tcgen05.mma of a row tile; TMEM holds S0 | S1 | O0 | O1 (128 columns each, of which heads of 64
//                 use half in O0 and O1). S is made in halves of 64 keys, two ahead of the softmax, P is written over S
//                 (in bf16; the sums that the result is divided by are of unrounded ones) and read from there
//   warps 4..11   softmax of tile 0 and 1, one row per thread, 64 keys a step: the maximum is raised only where it grows by more than 2^8;
//                 steps that the diagonal, a window or the last key crosses are masked before it. Before the first they bring the rows of Q
//   warps 12..15  a thread per key: its row of codes and scales (68 bytes for a head of 128; the next tile's are in flight) becomes bf16 values of
//                 keys, then of values, exactly, in the swizzled rows that the products read: keys along K, values along N, as they lie
//
// Packed rows mean that a tile is converted once for 256 rows whatever the group, and that the diagonal crosses few tiles: 256 rows of a
// group of 8 are 32 queries. Bound by the tensor core and by what a processor issues, about equally: a chunk of 2048 queries behind 6144
// keys takes 282 us for 32 heads over 8 (145 at the rate of the products alone; the kernel over a bf16 cache takes 245), four prompts of 2048
// tokens 410 us for 64 heads over 8 (165). What counts is how long a row tile waits for its next scores: S of 128 keys at once, made after P V of
// the ones before, takes 316 and 488; halves with one thread that issues for both row tiles 452 and 571, since it waits for each in turn.
// A grid that stays and takes blocks from a counter was slower (400): the issuing thread's state then no longer fits its registers.
#include "kv4.cuh"

namespace b200 {

int num_sms();      // of the current device, see gemm_tcgen05.cu

constexpr int kPf4Tile = 128;
constexpr int kPf4Sub = 64;               // keys of a product S: two of them are half a tile's
constexpr int kPf4Threads = 512;
constexpr int kPf4Stages = 2;
constexpr int kPf4Registers = 128;        // of a thread at launch: 65536 / kPf4Threads
constexpr int kPf4Half = kPf4Tile * 128;    // bytes of a tile's 64 values of a row: 128 bytes a row, swizzled
constexpr float kPf4Gap = 8.f;            // raise the running maximum only beyond this many powers of two
constexpr float kPf4Log2e = 1.4426950408889634f;

struct Pf4Barriers {
  uint64_t q_full;
  uint64_t k_full[kPf4Stages], k_empty[kPf4Stages];
  uint64_t v_full[kPf4Stages], v_empty[kPf4Stages];
  uint64_t s_full[2][2], p_ready[2][2], o_done[2][2];      // [row tile][half of a key tile]
  uint32_t tmem_base;
  uint32_t abort_flag;
};

struct Pf4Params {
  const __nv_bfloat16* q;      // [tokens][hq][d]
  __nv_bfloat16* out;
  const int* kv_lens;          // [sequences]
  const int* cu_q;             // [sequences + 1]
  Kv4Pool pool;
  int hq, group, causal, window;
  float scale_log2;            // softmax scale * log2(e)
  float cap_in, cap_out;       // capped: cap_out * tanh(score * scale / softcap) in log2 units
};

__device__ __forceinline__ float pf4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 columns of this warp's 32 lanes: half of the helpers' of common.cuh, for where 128 scores are in registers already.
__device__ __forceinline__ void pf4_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pf4_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

template <int D, bool kCap>
__global__ void __launch_bounds__(kPf4Threads, 1) attn_prefill_kv4_kernel(const Pf4Params p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kHalves = D / 64, kBytes = kHalves * kPf4Half;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                                   // two Q tiles, each [half head][128 rows][128 bytes]
  uint8_t* sk = sq + 2 * kBytes;
  uint8_t* sv = sk + kPf4Stages * kBytes;
  Pf4Barriers* bars = reinterpret_cast<Pf4Barriers*>(sv + kPf4Stages * kBytes);

  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.z, kvh = blockIdx.y, G = p.group;
  const int q_off = p.cu_q[seq], q_len = p.cu_q[seq + 1] - q_off;
  const int rows = q_len * G;
  const int row0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * 2 * kPf4Tile;     // the longest rows first
  if (row0 >= rows) return;
  const int kv_len = kv4_length(p.pool, p.kv_lens[seq], kKernelKv4);
  const int ctx = kv_len - q_len;                       // keys in front of the first query
  const bool tile1 = row0 + kPf4Tile < rows;
  const int last_query = (min(rows, row0 + 2 * kPf4Tile) - 1) / G;
  const int n_keys = p.causal ? min(kv_len, ctx + last_query + 1) : kv_len;
  const int first_tile = p.window > 0 ? kv4_window_start(ctx + row0 / G + 1, p.window) / kPf4Tile : 0;
  const int n_tiles = n_keys > first_tile * kPf4Tile ? (n_keys + kPf4Tile - 1) / kPf4Tile - first_tile : 0;
  const int n_subs = n_tiles > 0 ? (n_keys + kPf4Sub - 1) / kPf4Sub - 2 * first_tile : 0;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 8);
    for (int i = 0; i < kPf4Stages; ++i) {
      mbar_init(&bars->k_full[i], 4);
      mbar_init(&bars->k_empty[i], tile1 ? 2 : 1);
      mbar_init(&bars->v_full[i], 4);
      mbar_init(&bars->v_empty[i], tile1 ? 2 : 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[t][b], 1);
        mbar_init(&bars->p_ready[t][b], 4);
        mbar_init(&bars->o_done[t][b], 1);
      }
    }
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  constexpr uint32_t kIdescS = make_idesc(128, kPf4Sub, kFmtBf16, kFmtBf16);
  constexpr uint32_t kIdescPV = make_idesc(128, D, kFmtBf16, kFmtBf16) | kIdescBMn;

  // launch: 128 registers a thread, 512 for the four warpgroups' threads of a lane; 96 + 2 * 160 + 96 of them below, which the host makes sure of
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp < (tile1 ? 2 : 1) && lane == 0 && n_tiles > 0) {
      // ----------------------------------------------------------------------- one issuer per row tile
      const int t = warp;
      const uint32_t s_at = tmem_base + t * 128, o_at = tmem_base + 256 + t * 128;
      const uint64_t qd = make_desc_sw128(smem_u32(sq + t * kBytes)), kd = make_desc_sw128(smem_u32(sk)), vd = make_desc_sw128_mn(smem_u32(sv), kPf4Half);
      bool ok = mbar_wait(&bars->q_full, 0, abort_flag);
      // S(u) = Q K_u^T into the columns of half u & 1
      auto issue_s = [&](int u) {
        const int s = (u >> 1) % kPf4Stages, b = u & 1;
#pragma unroll
        for (int a = 0; a < kHalves; ++a) {
          const uint64_t ad = qd + a * (kPf4Half >> 4), bd = kd + ((s * kBytes + a * kPf4Half + b * kPf4Sub * 128) >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_bf16_ss(s_at + b * kPf4Sub, ad + 2 * k, bd + 2 * k, kIdescS, (a | k) != 0);
        }
        tc_commit(&bars->s_full[t][b]);
        if (b) tc_commit(&bars->k_empty[s]);
      };
      if (ok) ok = mbar_wait(&bars->k_full[0], 0, abort_flag);
      if (ok) {
        tc_fence_after_sync();
        for (int u = 0; u < min(2, n_subs); ++u) issue_s(u);
      }
      for (int u = 0; u < n_subs && ok; ++u) {
        const int j = u >> 1, b = u & 1, s = j % kPf4Stages;
        if (!(ok = mbar_wait(&bars->p_ready[t][b], j & 1, abort_flag))) break;
        if (b == 0 && !(ok = mbar_wait(&bars->v_full[s], static_cast<uint32_t>((j / kPf4Stages) & 1), abort_flag))) break;
        tc_fence_after_sync();
        // O += P V_u: A = P in TMEM (16 keys are 8 columns of bf16 pairs), B = 16 rows of the V tile
        const uint64_t bd = vd + ((s * kBytes + b * kPf4Sub * 128) >> 4);
#pragma unroll
        for (int k = 0; k < kPf4Sub / 16; ++k) mma_bf16_ts(o_at, s_at + b * kPf4Sub + k * 8, bd + k * (2048 >> 4), kIdescPV, (u | k) != 0);
        if (b) tc_commit(&bars->v_empty[s]);
        tc_commit(&bars->o_done[t][b]);
        if (u + 2 < n_subs) {
          const int s1 = (j + 1) % kPf4Stages;
          if (b == 0 && !(ok = mbar_wait(&bars->k_full[s1], static_cast<uint32_t>(((j + 1) / kPf4Stages) & 1), abort_flag))) break;
          tc_fence_after_sync();
          issue_s(u + 2);          // executes after the P V_u above: it overwrites the columns P lives in
        }
      }
      if (!ok) report_status(p.pool.status, kWaitTimeout, kKernelKv4, 51, blockIdx.x);
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ------------------------------------------------------------------------- codes to numbers, one key per thread
    const int key = (warp - 12) * 32 + lane;
    const int* table = p.pool.block_table + static_cast<long long>(seq) * p.pool.max_pages;
    const int last = n_keys;
    auto unit_of = [&](int j) -> const uint8_t* {       // the unit of this thread's key of tile j, or none
      const int at = (first_tile + j) * kPf4Tile + key;
      return j < n_tiles && at < last ? kv4_unit<D>(p.pool, table, kvh, at >> 4, kKernelKv4) : nullptr;
    };
    uint32_t kw[D / 8], vw[D / 8], ks = 0, vs = 0;
    auto load = [&](const uint8_t* unit, bool values, uint32_t (&w)[D / 8], uint32_t& scales) {
      if (unit) {
        kv4_load_row<D>(unit + (values ? kv4_plane_bytes(D) : 0), key & 15, values, w, scales);
      } else {
        scales = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = 0x88888888u;      // zeros: their probabilities are, but what lies there need not be a number
      }
    };
    const uint8_t* unit = unit_of(0);
    load(unit, false, kw, ks);
    load(unit, true, vw, vs);
    unit = unit_of(1);
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j % kPf4Stages;
      const uint32_t ph = static_cast<uint32_t>((j / kPf4Stages) & 1) ^ 1;
      auto row_at = [&](uint8_t* tile, int piece) { return tile + (piece >> 3) * kPf4Half + key * 128 + (((piece & 7) ^ (key & 7)) << 4); };
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty[s], ph, abort_flag)))) break;
      kv4_key_row<D>(kw, ks, [&](int piece, uint4 v) { *reinterpret_cast<uint4*>(row_at(sk + s * kBytes, piece)) = v; });
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->k_full[s]);
      load(unit, false, kw, ks);
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_empty[s], ph, abort_flag)))) break;
      kv4_value_row<D>(vw, vs, [&](int piece, uint4 v) { *reinterpret_cast<uint4*>(row_at(sv + s * kBytes, piece)) = v; });
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->v_full[s]);
      load(unit, true, vw, vs);
      unit = unit_of(j + 2);
    }
    if (!ok && lane == 0) report_status(p.pool.status, kWaitTimeout, kKernelKv4, 52, blockIdx.x);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    // ------------------------------------------------------------------------- softmax warps
    const int t = (warp >> 2) - 1;                        // row tile of this warp group
    const int quarter = warp & 3;                         // TMEM lane quarter this warp may touch
    const int local = quarter * 32 + lane;                // row inside the tile = TMEM lane
    const int row_first = row0 + t * kPf4Tile + quarter * 32, row = row_first + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_col = lane_base + t * 128, o_col = lane_base + 256 + t * 128;
    const int query = row / G, head = row - query * G;
    {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + ((static_cast<long long>(q_off) + query) * p.hq + kvh * G + head) * D);
      uint8_t* dst = sq + t * kBytes + local * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<uint4*>(dst + (i >> 3) * kPf4Half + (((i & 7) ^ (local & 7)) << 4)) = row < rows ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full);
    }
    if (t == 0 || tile1) {
      const int pos = ctx + query;
      const int lim = row >= rows ? 0 : p.causal ? min(kv_len, pos + 1) : kv_len;         // keys [start, lim) are this row's
      const int start = p.window > 0 ? kv4_window_start(pos + 1, p.window) : 0;
      // keys that every row of the warp sees
      const int open_from = __reduce_max_sync(0xffffffffu, start), open_to = __reduce_min_sync(0xffffffffu, lim);
      float m_run = -INFINITY, l_run = 0.f;
      const float c = kCap ? 1.f : p.scale_log2;
      bool ok = true;
      for (int u = 0; u < n_subs && ok; ++u) {
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->s_full[t][u & 1], (u >> 1) & 1, abort_flag))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t col = s_col + (u & 1) * kPf4Sub;
        uint32_t r[kPf4Sub];
        float mf[8];
        tmem_ld_32x32(col, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld_32x32(col + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_wait();
        const int key0 = first_tile * kPf4Tile + u * kPf4Sub;
        if (kCap)
#pragma unroll
          for (int i = 0; i < kPf4Sub; ++i)               // cap tanh(x) = cap - 2 cap / (exp(2 x) + 1)
            r[i] = __float_as_uint(p.cap_out - __fdividef(2.f * p.cap_out, pf4_exp2(kv4_cut(__uint_as_float(r[i]) * p.cap_in)) + 1.f));
        if (key0 < open_from || key0 + kPf4Sub > open_to) {
          const int from = start - key0, to = lim - key0;
#pragma unroll
          for (int i = 0; i < kPf4Sub; ++i)
            if (i >= to || i < from) r[i] = 0xff800000u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mf[i] = __uint_as_float(r[i]);
#pragma unroll
        for (int i = 8; i < kPf4Sub; ++i) mf[i & 7] = fmaxf(mf[i & 7], __uint_as_float(r[i]));
        const float mx = fmaxf(fmaxf(fmaxf(mf[0], mf[1]), fmaxf(mf[2], mf[3])), fmaxf(fmaxf(mf[4], mf[5]), fmaxf(mf[6], mf[7]))) * c;
        // raise the running maximum only when it would grow by more than the gap (or on the first tile);
        // a warp decides together because the O rescale below is a warp-wide TMEM access
        if (__any_sync(0xffffffffu, mx > m_run + kPf4Gap)) {
          const float m_new = fmaxf(m_run, mx);
          const float alpha = m_run == -INFINITY ? 0.f : pf4_exp2(m_run - m_new);
          if (u > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(&bars->o_done[t][(u - 1) & 1], ((u - 1) >> 1) & 1, abort_flag))) { ok = false; break; }
            tc_fence_after_sync();
#pragma unroll
            for (int cc = 0; cc < D / 16; ++cc) {
              uint32_t o[16];
              pf4_ld16(o_col + cc * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              pf4_st16(o_col + cc * 16, o);
            }
            tmem_st_wait();
          }
          l_run *= alpha;
          m_run = m_new;
        }
        const float sub = m_run == -INFINITY ? 0.f : m_run;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cc = 0; cc < kPf4Sub / 32; ++cc) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = pf4_exp2(fmaf(__uint_as_float(r[cc * 32 + 2 * i]), c, -sub));
            const float b = pf4_exp2(fmaf(__uint_as_float(r[cc * 32 + 2 * i + 1]), c, -sub));
            sums[i & 3] += a + b;
            packed[i] = pack_bf16x2(a, b);
          }
          pf4_st16(col + cc * 16, packed);               // P_t over the first half of S_t
        }
        tmem_st_wait();
        l_run += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_ready[t][u & 1]);
      }
      // scores are two ahead, so the last two products may both be outstanding
      for (int u = max(0, n_subs - 2); u < n_subs && ok; ++u) ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_done[t][u & 1], (u >> 1) & 1, abort_flag));
      if (!ok) {
        if (lane == 0) report_status(p.pool.status, kWaitTimeout, kKernelKv4, 53, blockIdx.x);
      } else {
        tc_fence_after_sync();
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        // The Q tile is no longer read: 32 rows of 128 bytes per warp turn the rows that the lanes hold into
        // 128-byte runs. 16-byte pieces are placed by (piece xor row), which keeps the banks apart.
        uint8_t* strip = sq + t * kBytes + quarter * 32 * 128;
#pragma unroll
        for (int hc = 0; hc < kHalves; ++hc) {
          uint32_t o[64];
          tmem_ld_32x32(o_col + hc * 64, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
          tmem_ld_32x32(o_col + hc * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              w[u] = n_tiles > 0 && inv != 0.f ? pack_bf16x2(__uint_as_float(o[i * 8 + 2 * u]) * inv, __uint_as_float(o[i * 8 + 2 * u + 1]) * inv) : 0u;
            *reinterpret_cast<uint4*>(strip + lane * 128 + ((i ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = i * 4 + (lane >> 3), piece = lane & 7, out_row = row_first + rr;
            const uint4 v = *reinterpret_cast<const uint4*>(strip + rr * 128 + ((piece ^ (rr & 7)) * 16));
            if (out_row < rows) {
              const int oq = out_row / G;
              *reinterpret_cast<uint4*>(p.out + ((static_cast<long long>(q_off) + oq) * p.hq + kvh * G + (out_row - oq * G)) * D + hc * 64 + piece * 8) = v;
            }
          }
          __syncwarp();
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace b200

using namespace b200;

// Which kernel takes a batch of prompt chunks of these sizes: 0 b200_attn_kv4, 1 b200_attn_prefill_kv4, 2 b200_attn_few_kv4.
B200_API int b200_attn_kv4_choice(int seqs, int max_q_len, int max_kv_len, int hq, int hkv, int d, int causal, int window, float scale) {
  if (seqs < 1 || max_q_len < 1 || hkv < 1 || hq < hkv) return 0;
  // Estimates in us from the times below. Blocks of 64 rows (b200_attn_kv4) start fastest and share a processor; blocks of 256 rows (this file's)
  // come in waves; parts of the key axis (b200_attn_few_kv4) read all units once for every 16 columns.
  // Measured in us, 64 rows / 256 rows / parts, 32 heads over 8: one sequence of 100 queries 7.1 / 11.4 / -, of 512 24 / 19 / -, of 2048
  // 191 / 74 / -; 17 queries behind 1000 keys 30 / 23 / 22, behind 8000 210 / 130 / 36; 100 there 213 / 175 / 99; 8 behind 30000 768 / 458 / 39;
  // 16 sequences of 17 behind 100 keys 9.8 / 10.7 / -, behind 1000 44 / 25 / 57, of 5 behind 3000 81 / 63 / 57. 32 heads over 32: 16 of 17
  // behind 1000 83 / 98 / 76. Heads of 64, 32 over 8: 100 queries 5.3 / 8.5 / -, 512 18 / 15 / -, 2048 behind 6000 623 / 236 / -, 17 behind
  // 8000 145 / 123 / 26, 100 there 147 / 164 / 67.
  const long long rows = static_cast<long long>(max_q_len) * (hq / hkv), lists = static_cast<long long>(seqs) * hkv;
  const long long waves = ((rows + 2 * kPf4Tile - 1) / (2 * kPf4Tile) * lists + num_sms() - 1) / num_sms();
  const double each = static_cast<double>((rows + 63) / 64 * lists) / num_sms();       // blocks of 64 rows a processor
  const double keys = window > 0 && window + static_cast<double>(max_q_len) < max_kv_len ? window + static_cast<double>(max_q_len) : max_kv_len;
  const double units = keys / kKv4Unit * static_cast<double>((rows + 15) / 16 * lists);
  const bool big = d == 128;
  const double small = (big ? 3.3 : 3.) + (each > 1. ? each : 1.) * (big ? 0.026 : 0.0178) * keys;
  const double wide = static_cast<double>(waves) * (big ? 7.5 + 0.0195 * keys : 6. + 0.018 * keys);
  const double parts = big ? 18. + 0.0008 * units : 14. + 0.00051 * units;
  const bool can = scale > 0.f, best = can && wide < small;
  if (causal && keys > 512. && rows < 65536 && seqs <= kKv4MaxSeqs && parts < (best ? wide : small)) return 2;
  return best;
}

// Arguments as of b200_attn_kv4 with cu_q; a scale above 0.
B200_API int b200_attn_prefill_kv4(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, const int* cu_q,
                                   int seqs, int max_q_len, int hq, int hkv, int d, int page, int max_pages, long long pages,
                                   int causal, int window, float scale, float softcap, void* status, cudaStream_t stream) {
  if (seqs <= 0 || max_q_len <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || max_pages < 1 || pages < 1 || !kv4_pool_fits(pool, d, page)) return -2;
  if (seqs > 65535 || hkv > 65535 || static_cast<long long>(max_q_len) * (hq / hkv) >= (1ll << 30)) return -3;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) return -4;
  if (!(scale > 0.f)) return -5;
  Pf4Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.kv_lens = kv_lens;
  p.cu_q = cu_q;
  p.pool = Kv4Pool{static_cast<const uint8_t*>(pool), block_table, pages, hkv, max_pages, kv4_unit_shift(page), static_cast<DeviceStatus*>(status)};
  p.hq = hq; p.group = hq / hkv; p.causal = causal; p.window = window;
  p.scale_log2 = scale * kPf4Log2e;
  if (softcap > 0.f) {
    p.cap_in = 2.f * kPf4Log2e * scale / softcap;
    p.cap_out = softcap * kPf4Log2e;
  }
  const int smem = (2 + 2 * kPf4Stages) * kPf4Half * (d / 64) + static_cast<int>(sizeof(Pf4Barriers)) + 1024;
  static PerDeviceOnce once[4];
  static int registers[4];                             // of the kernels as they were built
  auto go = [&](auto kernel, int which) -> cudaError_t {
    if (registers[which] == 0) {
      cudaFuncAttributes has{};
      const cudaError_t e = cudaFuncGetAttributes(&has, kernel);
      if (e != cudaSuccess) return e;
      registers[which] = has.numRegs;
    }
    if (registers[which] != kPf4Registers) return cudaErrorInvalidConfiguration;   // warps would wait for registers that nobody gives back
    if (once[which].first_time()) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
    }
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(max_q_len) * p.group + 2 * kPf4Tile - 1) / (2 * kPf4Tile)), hkv, seqs);
    return launch_pdl(kernel, grid, dim3(kPf4Threads), smem, stream, p);
  };
  cudaError_t e;
  if (d == 128) e = softcap > 0.f ? go(attn_prefill_kv4_kernel<128, true>, 0) : go(attn_prefill_kv4_kernel<128, false>, 1);
  else e = softcap > 0.f ? go(attn_prefill_kv4_kernel<64, true>, 2) : go(attn_prefill_kv4_kernel<64, false>, 3);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}
