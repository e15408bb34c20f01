// Attention over a K/V cache held in 4 bits (format: kv4.cuh), any number of query tokens per sequence.
//
// The query heads of a group read the same keys, so a block's 64 rows are (query, head of the group) pairs of one sequence and one kv head, heads
// fastest: row r is query r / G, head r % G. A tile of 64 keys is turned into bf16 in shared memory once for all of them: one row of
// keys or values per thread, whose bytes of the next tile are in flight during the products of this one.
//
// Products are mma.sync m16n8k16; softmax is the usual one pass with a running maximum, in 32 bits; probabilities enter
// the second product in bf16, their sum unrounded. Bound by how long a block of four warps
// takes for a key (26 ns with heads of 128, 18 with 64, whatever else runs until a processor has several blocks): a block starts in
// 3 us, so short prompts come here (five prompts of about 97 tokens: 5.9 us; 100 queries 7.1, where the blocks of 256 rows take 11.4).
#include "kv4.cuh"
#include "mma_sync.cuh"

namespace b200 {

constexpr int kKv4Tile = 64;               // keys
constexpr int kKv4Rows = 64;
constexpr float kKv4Log2e = 1.4426950408889634f;

struct AttnKv4Params {
  const __nv_bfloat16* q;      // [tokens][hq][d]
  __nv_bfloat16* out;
  const int* kv_lens;          // [sequences] keys up to the last query of each
  const int* cu_q;             // [sequences + 1]
  Kv4Pool pool;
  int hq, group, causal, window;
  float scale_log2;            // softmax scale * log2(e)
  float cap_in, cap_out;       // softcap: cap_out * tanh(score scale / softcap) in log2 units; cap_out 0: none
};

__device__ __forceinline__ float kv4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Score in log2 units. cap tanh(x) = cap - 2 cap / (exp(2 x) + 1)
__device__ __forceinline__ float kv4_score(const AttnKv4Params& p, float s) {
  if (p.cap_out == 0.f) return s * p.scale_log2;
  const float e = kv4_exp2(kv4_cut(s * p.cap_in));
  return p.cap_out - __fdividef(2.f * p.cap_out, e + 1.f);
}

template <int D>
__device__ __forceinline__ uint32_t kv4_tile_off(int token, int piece) {
  return static_cast<uint32_t>(token * (D * 2) + ((piece ^ (token & 7)) << 4));
}

template <int D>
__global__ void __launch_bounds__(128) attn_kv4_kernel(const AttnKv4Params p) {
  pdl_wait();
  pdl_trigger();
  __shared__ __align__(128) uint8_t smem[2 * kKv4Tile * D * 2];
  const int seq = blockIdx.z, kvh = blockIdx.y, G = p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int q_off = p.cu_q[seq], q_len = p.cu_q[seq + 1] - q_off;
  const long long rows = static_cast<long long>(q_len) * G;
  const long long block_row = static_cast<long long>(blockIdx.x) * kKv4Rows;
  if (block_row >= rows) return;
  const int kv_len = kv4_length(p.pool, p.kv_lens[seq], kKernelKv4);
  const int ctx = kv_len - q_len;
  const uint32_t k_smem = smem_u32(smem), v_smem = k_smem + kKv4Tile * D * 2;

  int lim[2], start[2], query[2], head[2];
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const long long row = block_row + warp * 16 + g + 8 * r;
    const bool on = row < rows;
    query[r] = on ? static_cast<int>(row / G) : -1;
    head[r] = on ? static_cast<int>(row - static_cast<long long>(query[r]) * G) : 0;
    const int pos = ctx + query[r];
    lim[r] = !on ? 0 : p.causal ? min(kv_len, pos + 1) : kv_len;
    start[r] = on && p.window > 0 ? kv4_window_start(pos + 1, p.window) : 0;
    const __nv_bfloat16* src = p.q + ((static_cast<long long>(q_off) + max(query[r], 0)) * p.hq + kvh * G + head[r]) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const int c = kk * 16 + tq * 2;
      qf[kk][r] = on ? *reinterpret_cast<const uint32_t*>(src + c) : 0u;
      qf[kk][2 + r] = on ? *reinterpret_cast<const uint32_t*>(src + c + 8) : 0u;
    }
  }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

  // keys that some row of the block sees
  const int first_query = static_cast<int>(block_row / G);
  const int last_query = static_cast<int>(min(rows, block_row + kKv4Rows) - 1) / G;
  const int keys = p.causal ? min(kv_len, ctx + last_query + 1) : kv_len;
  const int key0 = p.window > 0 ? kv4_window_start(ctx + first_query + 1, p.window) : 0;
  const int tiles = keys > 0 ? (keys + kKv4Tile - 1) / kKv4Tile : 0;
  const int* table = p.pool.block_table + static_cast<long long>(seq) * p.pool.max_pages;
  // this thread's row of a tile: a key (threads 0 .. 63) or a value
  const int my_key = threadIdx.x & 63;
  const bool values = threadIdx.x >= 64;
  uint32_t raw[D / 8], scales = 0;
  auto load = [&](int tile) {
    const int key = tile * kKv4Tile + my_key;
    if (tile < tiles && key < keys) {
      const uint8_t* unit = kv4_unit<D>(p.pool, table, kvh, key >> 4, kKernelKv4);
      kv4_load_row<D>(unit + (values ? kv4_plane_bytes(D) : 0), key & 15, values, raw, scales);
    } else {
      scales = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) raw[i] = 0x88888888u;        // zeros
    }
  };
  load(key0 / kKv4Tile);
  for (int tile = key0 / kKv4Tile; tile < tiles; ++tile) {
    __syncthreads();                                   // the products of the last tile have read it
    auto put = [&](int piece, uint4 v) {
      *reinterpret_cast<uint4*>(smem + (values ? kKv4Tile * D * 2 : 0) + kv4_tile_off<D>(my_key, piece)) = v;
    };
    if (values) kv4_value_row<D>(raw, scales, put);
    else kv4_key_row<D>(raw, scales, put);
    __syncthreads();
    load(tile + 1);
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const int mi = lane >> 3;
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(k_smem + kv4_tile_off<D>(gi * 16 + (lane & 7) + 8 * (mi >> 1), kk * 2 + (mi & 1)), b0, b1, b2, b3);
        mma_bf16_16816(s[gi * 2], qf[kk], b0, b1);
        mma_bf16_16816(s[gi * 2 + 1], qf[kk], b2, b3);
      }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j >> 1, key = tile * kKv4Tile + nt * 8 + tq * 2 + (j & 1);
        const float x = kv4_score(p, s[nt][j]);
        s[nt][j] = key < lim[r] && key >= start[r] ? x : -INFINITY;
        mx[r] = fmaxf(mx[r], s[nt][j]);
      }
    float safe[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float top = fmaxf(m[r], mx[r]);
      safe[r] = top == -INFINITY ? 0.f : top;          // a row that sees nothing yet
      const float alpha = m[r] == -INFINITY ? 0.f : kv4_exp2(m[r] - safe[r]);
      m[r] = top;
      l[r] *= alpha;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][2 * r] *= alpha;
        o[i][2 * r + 1] *= alpha;
      }
    }
    uint32_t pf[4][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = kv4_exp2(s[nt][j] - safe[j >> 1]);
        l[j >> 1] += e[j];
      }
      pf[nt >> 1][(nt & 1) * 2] = pack_bf16x2(e[0], e[1]);
      pf[nt >> 1][(nt & 1) * 2 + 1] = pack_bf16x2(e[2], e[3]);
    }
#pragma unroll
    for (int gi = 0; gi < 4; ++gi)
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const int mi = lane >> 3;
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(v_smem + kv4_tile_off<D>(gi * 16 + (lane & 7) + 8 * (mi & 1), c * 2 + (mi >> 1)), b0, b1, b2, b3);
        mma_bf16_16816(o[c * 2], pf[gi], b0, b1);
        mma_bf16_16816(o[c * 2 + 1], pf[gi], b2, b3);
      }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (query[r] < 0) continue;
    const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
    __nv_bfloat16* dst = p.out + ((static_cast<long long>(q_off) + query[r]) * p.hq + kvh * G + head[r]) * D + tq * 2;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint32_t*>(dst + i * 8) = pack_bf16x2(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
  }
}

}  // namespace b200

using namespace b200;

// q, out [tokens][hq][d] bf16, packed by cu_q. window > 0: every query sees that many last keys.
B200_API int b200_attn_kv4(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, const int* cu_q, int seqs,
                           int max_q_len, int hq, int hkv, int d, int page, int max_pages, long long pages, int causal, int window,
                           float scale, float softcap, void* status, cudaStream_t stream) {
  if (seqs <= 0 || max_q_len <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || max_pages < 1 || pages < 1 || !kv4_pool_fits(pool, d, page)) return -2;
  if (seqs > 65535 || hkv > 65535 || static_cast<long long>(max_q_len) * (hq / hkv) >= (1ll << 30)) return -3;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) return -4;
  if (!cu_q) return -6;
  AttnKv4Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.kv_lens = kv_lens;
  p.cu_q = cu_q;
  p.pool = Kv4Pool{static_cast<const uint8_t*>(pool), block_table, pages, hkv, max_pages, kv4_unit_shift(page), static_cast<DeviceStatus*>(status)};
  p.hq = hq; p.group = hq / hkv; p.causal = causal; p.window = window;
  p.scale_log2 = scale * kKv4Log2e;
  if (softcap > 0.f) {
    p.cap_in = 2.f * kKv4Log2e * scale / softcap;
    p.cap_out = softcap * kKv4Log2e;
  }
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(max_q_len) * p.group + kKv4Rows - 1) / kKv4Rows), hkv, seqs);
  const cudaError_t e = d == 128 ? launch_pdl(attn_kv4_kernel<128>, grid, dim3(128), 0, stream, p) : launch_pdl(attn_kv4_kernel<64>, grid, dim3(128), 0, stream, p);
  return e == cudaSuccess ? 0 : -static_cast<int>(e) - 300;
}
