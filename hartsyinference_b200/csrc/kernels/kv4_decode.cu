// One query token per sequence, or a few, over a K/V cache held in 4 bits (format: kv4.cuh).
//
// Bound by the bytes of the cache only as long as a byte costs few instructions: at 6.5 TB/s a processor gets 24 bytes (45 values) a cycle and issues
// four warp instructions in it. So codes are never unpacked one by one; the tensor core multiplies registers that are masked words of a row:
//
//   S^T (keys x heads) = K Q^T     A = codes of 16 keys, B = queries, both in half precision: masked with 0x000f000f a word is two
//                                  subnormals code * 2^-24, with 0x00f000f0 two of code * 2^-20 (queries of those places are divided by 16; all
//                                  are times a power of two that keeps a bf16's bits). A block of 32 values has one scale per key: its
//                                  partial sums are multiplied by it in 32 bits. The offset 8 of the codes is in what the sums start from
//   O^T (values x heads) = V^T P^T A = codes of 16 values of 16 keys (four bits in the mantissa of a bf16 128) times the keys' scales of that
//                                  block, less 136 of them, in one fused multiply-add for two: exact, since a code times a scale has 7
//                                  bits. B = P^T, rounded to 8 bits; what the sums are divided by sums unrounded ones. In bf16, since
//                                  probabilities have no bound from below: a first token that takes nearly all of the weight and has
//                                  values near zero leaves the rest to probabilities of 2^-24. (With the scales in P^T and the offset as a
//                                  second product P^T would be rounded twice; 64 sequences of 2048 to 2304 tokens 54.8 us for 54.0)
//
// P^T is S^T after the softmax with its 8 x 8 blocks transposed (movmatrix). Rows of the tile are not the keys in order: row 2 i is key i and
// row 2 i + 1 key 7 - i of eight, which lets every shared-memory read of codes touch each bank once.
//
// Work: a unit is 16 tokens of one kv head. All units of all sequences and heads in a row are cut into equal shares, one per resident
// block (or one per unit, where there are fewer of them than blocks), whatever the lengths; a share's first and last sequence may be
// other blocks' too, whose parts the second kernel joins (in the order of the blocks, so results do not depend on timing). Within a
// share every warp takes units side by side and has its own ring of bulk copies, so warps meet only at the end. Short sequences get one
// block each and no second kernel.
#include "kv4.cuh"
#include "mma_sync.cuh"

#include <type_traits>

namespace b200 {

int num_sms();      // of the current device, see gemm_tcgen05.cu

constexpr int kDec4Warps = 8;
constexpr int kDec4Threads = kDec4Warps * 32;
constexpr int kDec4Stages = 2;            // of a warp's ring, two units each
constexpr int kDec4MaxSeqs = kKv4MaxSeqs;
constexpr float kDec4Gap = 8.f;            // the reference of the exponentials is raised once a score passes it by this many powers of two
constexpr float kDec4Log2e = 1.4426950408889634f;

struct DecodeKv4Params {
  const __nv_bfloat16* q;      // [tokens][hq][d]
  __nv_bfloat16* out;
  const int* kv_lens;
  const int* cu_q;             // [sequences + 1]: the last tokens of a sequence ask; null: one token a sequence
  Kv4Pool pool;
  float* parts;                // [blocks][2][heads of a chunk][d + 4]: sums, maximum, denominator
  int* prefix;                 // [sequences + 1] units before a sequence, for the second kernel
  int seqs, hq, group, chunks, chunk_heads;      // columns (query, head of a group), heads fastest, are walked in `chunks` parts
  int window, blocks;
  float scale_log2, cap_in, cap_out;
};

__device__ __forceinline__ uint32_t scaled_bf16x2(uint32_t x, uint32_t s) {
  const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t x, uint32_t s, uint32_t off) {
  const __nv_bfloat162 y = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&s), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&y);
}
// d += A B. Not volatile: products of keys and of values of two units may be interleaved.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A constant that the compiler keeps in a register: as an immediate next to another one it would take an instruction more.
__device__ __forceinline__ uint32_t in_register(uint32_t x) {
  uint32_t y;
  asm volatile("mov.b32 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Four numbers of shared memory, loaded where this stands: two operands that start alike would else be one load and four moves.
__device__ __forceinline__ void load_here(float (&x)[4], const float4* at) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(smem_u32(at)));
}
// (x & mask) | bits in one instruction
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
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

// Tokens of a sequence that ask; few: several of them, else one. Known when compiled except in the joins: decoded tokens would
// otherwise pay for the other case (4.4 us became 5.7 for 16 short sequences).
__device__ __forceinline__ int dec4_queries(const DecodeKv4Params& p, bool few, int s) { return few ? p.cu_q[s + 1] - p.cu_q[s] : 1; }
// Blocks that have a share of `total` units. The host counts blocks from a bound of the lengths, so there may be more of them than units; those
// behind these write nothing, and the join must not read what they would have written.
__device__ __forceinline__ long long dec4_shares(const DecodeKv4Params& p, long long total) { return total < p.blocks ? total : p.blocks; }
// Units of a sequence that its queries see, and the first of them.
__device__ __forceinline__ int dec4_units(const DecodeKv4Params& p, bool few, int s, int& first) {
  const int len = kv4_length(p.pool, p.kv_lens[s], kKernelKv4), queries = dec4_queries(p, few, s);
  first = p.window > 0 ? kv4_window_start(len - queries + 1, p.window) / kKv4Unit : 0;
  return len > 0 && queries > 0 ? (len + kKv4Unit - 1) / kKv4Unit - first : 0;
}
// The columns of part h % chunks of kv head h / chunks: how many there are, and the row of q and of the output of one of them.
struct Dec4Columns {
  int first, n, group, hq;
  long long row0;
  bool few;
  __device__ __forceinline__ Dec4Columns(const DecodeKv4Params& p, bool few, int s, int h) : few(few) {
    const int kv_head = h / p.chunks;
    first = (h - kv_head * p.chunks) * p.chunk_heads;
    n = min(p.chunk_heads, dec4_queries(p, few, s) * p.group - first);
    group = p.group;
    hq = p.hq;
    row0 = static_cast<long long>(few ? p.cu_q[s] : s) * hq + kv_head * group;
  }
  __device__ __forceinline__ int query(int c) const { return static_cast<int>(static_cast<uint32_t>(first + c) / static_cast<uint32_t>(group)); }
  __device__ __forceinline__ long long row(int c) const {
    const int i = few ? query(c) : 0;
    return row0 + static_cast<long long>(i) * hq + first + c - i * group;
  }
};

// Dynamic shared memory: rings, one part of a sequence for every warp, the prefix.
__host__ __device__ constexpr int dec4_ring_bytes(int d) { return kDec4Warps * kDec4Stages * 2 * kv4_unit_bytes(d); }
__host__ __device__ constexpr int dec4_merge_bytes(int d, int nt) { return kDec4Warps * 8 * nt * (d + 4) * 4; }
__host__ __device__ constexpr int dec4_smem_bytes(int d, int nt) { return dec4_ring_bytes(d) + dec4_merge_bytes(d, nt) + (kDec4MaxSeqs + 1) * 4; }

// A part of a sequence that a warp could not finish: slot 0 what began before the warp's units, slot 1 what goes on behind them.
struct Dec4Part {
  int s, h;          // -1: none
  int rel;           // first unit of the sequence (and head) in the order, from the block's first one on
  int n;             // its units
};

template <int D, int NT, bool kShares, bool kFew>
__global__ void __launch_bounds__(kDec4Threads, NT == 1 ? 2 : 1) attn_decode_kv4_kernel(const DecodeKv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr uint32_t kValueBias = ((127 - 15 + kKv4ValueExp) << 7) * 0x10001u;
  constexpr int kUnit = kv4_unit_bytes(D), kPlane = kv4_plane_bytes(D), kBlocks = D / 32, kWords = D / 32, kPitch = D + 4;
  __shared__ uint64_t full[kDec4Warps][kDec4Stages];
  __shared__ Dec4Part parked[kDec4Warps][2];
  __shared__ float4 starts[kDec4Warps][NT][D / 32][4];      // [block][lane quarter]: what the sums of key products start from
  __shared__ int warp_units[kDec4Warps];
  __shared__ uint32_t abort_word;
  float* merge = reinterpret_cast<float*>(smem + dec4_ring_bytes(D));
  int* prefix = reinterpret_cast<int*>(smem + dec4_ring_bytes(D) + dec4_merge_bytes(D, NT));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  uint8_t* ring = smem + warp * kDec4Stages * 2 * kUnit;
  volatile uint32_t* abort_flag = &abort_word;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kDec4Stages; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
    parked[warp][0].s = parked[warp][1].s = -1;
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
      int first, n = s < p.seqs ? dec4_units(p, kFew, s, first) : 0;
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
    const long long total = static_cast<long long>(run) * heads_v, shares = dec4_shares(p, total);
    if (blockIdx.x >= shares) return;
    f0 = total * blockIdx.x / shares;
    f1 = total * (blockIdx.x + 1) / shares;
  } else {
    only_seq = blockIdx.x / heads_v;
    only_units = dec4_units(p, kFew, only_seq, only_first);
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
      h = static_cast<int>(static_cast<uint32_t>(f - seq_at) / static_cast<uint32_t>(n));
      at = seq_at + static_cast<long long>(h) * n;
      first = 0;
      if (p.window > 0) dec4_units(p, kFew, s, first);
    } else {
      s = only_seq; h = blockIdx.x - only_seq * heads_v; at = 0; n = only_units; first = only_first;
    }
  };
  const int share = static_cast<int>(f1 - f0);
  if (!kShares && share == 0) {                      // a sequence without keys
    const Dec4Columns cols(p, kFew, only_seq, blockIdx.x - only_seq * heads_v);
    for (int c = warp; c < cols.n; c += kDec4Warps)
      for (int j = lane; j < D / 2; j += 32) reinterpret_cast<uint32_t*>(p.out + cols.row(c) * D)[j] = 0u;
    return;
  }
  // this warp's part of the share, in pairs of units
  const int w0 = static_cast<int>(static_cast<long long>(share) * warp / kDec4Warps), units = static_cast<int>(static_cast<long long>(share) * (warp + 1) / kDec4Warps) - w0;
  const int mine = (units + 1) >> 1;
  f0 += w0;
  const uint8_t* src = nullptr;                      // lane j: address of unit 32 (i / 16) + j of the warp
  auto addresses = [&](int i0) {
    const int rel = 2 * i0 + lane;
    src = nullptr;
    if (rel >= units) return;
    int s, h, n, first;
    long long at;
    find(f0 + rel, s, h, at, n, first);
    src = kv4_unit<D>(p.pool, p.pool.block_table + static_cast<long long>(s) * p.pool.max_pages, h / p.chunks, first + static_cast<int>(f0 + rel - at), kKernelKv4);
  };
  // pair i into slot `to` of the ring; a unit behind the last is left out
  auto fetch = [&](int i, int to) {
    if (i >= mine) return;
    if ((i & 15) == 0 && i > 0) addresses(i);
    const unsigned long long a = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), 2 * (i & 15)), b = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), 2 * (i & 15) + 1);
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[warp][to], b ? 2 * kUnit : kUnit);
      bulk_load(ring + 2 * to * kUnit, reinterpret_cast<const void*>(a), kUnit, &full[warp][to]);
      if (b) bulk_load(ring + (2 * to + 1) * kUnit, reinterpret_cast<const void*>(b), kUnit, &full[warp][to]);
    }
  };
  const int ka = (g & 1) ? 7 - (g >> 1) : g >> 1;    // keys of rows g and g + 8: ka, ka + 8
  // where a lane reads in a unit: its words of keys ka and of the values of keys tq and 7 - tq, and their scales
  const int k_at = ka * (D / 2) + tq * (D / 8), ks_at = 8 * D + ka * (D / 32);
  const int v_at = kPlane + tq * (D / 2) + (D == 128 ? (g ^ ((tq & 2) << 1)) * 8 : g * 4), vs_at = kPlane + 8 * D + tq * (D / 32);
  const int w_at = kPlane + (7 - tq) * (D / 2) + (D == 128 ? (g ^ (((7 - tq) & 2) << 1)) * 8 : g * 4), ws_at = kPlane + 8 * D + (7 - tq) * (D / 32);
  constexpr int kOther = 8 * (D / 2), kOtherScale = 8 * (D / 32);          // eight keys on
  const uint32_t value_bias = in_register(kValueBias), sixteen = in_register(16u);     // (a shift by four would be in the pipe of the masks)
  const uint32_t offset = in_register(0xc308c308u);   // -136 twice

  bool ok = true;
  int i = 0, slot = 0, phase = 0;                    // pair i of the warp is in `slot`
  for (int done = 0; done < units;) {
    int s, h, n, first, at_rel;                        // at_rel: where the sequence's units start, from the warp's first one on
    {
      long long at;
      find(f0 + done, s, h, at, n, first);
      at_rel = static_cast<int>(at - f0);
    }
    const int stop = min(at_rel + n, units);
    const Dec4Columns cols(p, kFew, s, h);

    // queries of columns 8 t + g in half precision, with a power of two taken out so that the largest is in [2^12, 2^13)
    uint32_t q[NT][D / 16][2];
    float factor[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const bool on = 8 * t + g < cols.n;
      const __nv_bfloat16* qh = p.q + (on ? cols.row(8 * t + g) * D : 0);
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) q[t][m][r] = on ? *reinterpret_cast<const uint32_t*>(qh + m * 16 + r * 8 + tq * 2) : 0u;
    }
    if (done == 0) {                                   // the first copies, while the queries are on their way
      addresses(0);
#pragma unroll
      for (int j = 0; j < kDec4Stages; ++j) fetch(j, j);
    }
    const int len = kv4_length(p.pool, p.kv_lens[s], kKernelKv4);
    // columns of query i see the keys below len - before + i, where `before` queries are in front of the last one
    const int before = dec4_queries(p, kFew, s) - 1;
    const int start = p.window > 0 ? kv4_window_start(len, p.window) : 0;       // of the last query: the others' masks begin before it
    const int stop_key = (first + units - at_rel) * kKv4Unit;          // keys from here on are not this warp's
    const int last = min(len - before, stop_key);
    __syncwarp();                                      // the last sequence's products have read `starts`
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float amax = 0.f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q[t][m][r]));
          amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = amax > 0.f ? min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 12, -100), 85) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        float sum = 0.f;
#pragma unroll
        for (int m = 2 * b; m < 2 * b + 2; ++m)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q[t][m][r]));
            const float sh = r ? down * 0.0625f : down;                 // places 8 .. 15 meet codes times 16
            q[t][m][r] = pack_f16x2(v.x * sh, v.y * sh);
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&q[t][m][r]));
            sum += (x.x + x.y) * (r ? 16.f : 1.f);
          }
        // the offset of the codes: -8 * 2^-24 times the block's queries, for the two heads of a lane's results
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= -4.76837158203125e-7f;
        const float s0 = __shfl_sync(0xffffffffu, sum, 8 * tq), s1 = __shfl_sync(0xffffffffu, sum, 8 * tq + 4);
        if (g == 0) starts[warp][t][b][tq] = make_float4(s0, s1, s0, s1);
      }
      // codes are times 2^24, scales (as fp32 with bits byte << 20 under an exponent of 96) times 2^(16 + key exponent)
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * (p.cap_out == 0.f ? p.scale_log2 : p.cap_in) *
                       __uint_as_float(static_cast<uint32_t>(127 + 24 + 16 + kKv4KeyExp) << 23);
      factor[t][0] = __shfl_sync(0xffffffffu, up, 8 * tq);
      factor[t][1] = __shfl_sync(0xffffffffu, up, 8 * tq + 4);
    }
    __syncwarp();

    float o[NT][D / 16][4], mx[NT][2], line[NT][2], l[NT][2];      // line: what a score has to pass to raise mx
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][m][j] = 0.f;
      mx[t][0] = mx[t][1] = -1e30f;                    // finite: a column may see nothing of a unit
      line[t][0] = line[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
    // scores of two units
    auto key_products = [&](const uint8_t* unit, float (&sc)[2][NT][4]) {
      uint32_t w[2][2][kWords], scale[2][2];           // [unit][key ka or ka + 8]
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* x = unit + u * kUnit + r * kOther + k_at;
          const uint8_t* y = unit + u * kUnit + r * kOtherScale + ks_at;
          if (D == 128) {
            const uint4 z = *reinterpret_cast<const uint4*>(x);
            w[u][r][0] = z.x; w[u][r][1] = z.y; w[u][r][kWords - 2] = z.z; w[u][r][kWords - 1] = z.w;
            scale[u][r] = *reinterpret_cast<const uint32_t*>(y);
          } else {
            const uint2 z = *reinterpret_cast<const uint2*>(x);
            w[u][r][0] = z.x; w[u][r][1] = z.y;
            scale[u][r] = *reinterpret_cast<const uint16_t*>(y);
          }
        }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t xa = w[u][0][b], xb = w[u][1][b], ya = xa >> 8, yb = xb >> 8;
            const uint32_t a0[4] = {xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u};
            const uint32_t a1[4] = {ya & 0x000f000fu, yb & 0x000f000fu, ya & 0x00f000f0u, yb & 0x00f000f0u};
            const uint32_t sa = scale[u][0], sb = scale[u][1];
            const float fa = __uint_as_float(masked_or(b < 3 ? sa << (20 - 8 * b) : sa >> 4, 0x0ff00000u, 0x30000000u));
            const float fb = __uint_as_float(masked_or(b < 3 ? sb << (20 - 8 * b) : sb >> 4, 0x0ff00000u, 0x30000000u));
            float acc[4];
            load_here(acc, &starts[warp][t][b][tq]);
            mma_f16(acc, a0, q[t][2 * b]);
            mma_f16(acc, a1, q[t][2 * b + 1]);
            sc[u][t][0] = b == 0 ? acc[0] * fa : fmaf(acc[0], fa, sc[u][t][0]);
            sc[u][t][1] = b == 0 ? acc[1] * fa : fmaf(acc[1], fa, sc[u][t][1]);
            sc[u][t][2] = b == 0 ? acc[2] * fb : fmaf(acc[2], fb, sc[u][t][2]);
            sc[u][t][3] = b == 0 ? acc[3] * fb : fmaf(acc[3], fb, sc[u][t][3]);
          }
        }
    };
    // P^T of two units from their scores; key0: the first key of the first one
    auto softmax = [&](float (&sc)[2][NT][4], uint32_t (&pt)[2][NT][2], int key0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[u][t][j] *= factor[t][j & 1];
        if (p.cap_out != 0.f)                         // cap tanh(x) = cap - 2 cap / (exp(2 x) + 1)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[u][t][j] = p.cap_out - __fdividef(2.f * p.cap_out, dec4_exp2(kv4_cut(sc[u][t][j])) + 1.f);
      }
      // keys below 0 are a pair's first unit where that is the list's before this one
      if (key0 < start || key0 + 2 * kKv4Unit > last)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + u * kKv4Unit + ka + (j & 2) * 4;
            if (kFew) {
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const int seen = len - before + cols.query(8 * t + 2 * tq + (j & 1));
                if (key < 0 || key >= min(seen, stop_key) || (p.window > 0 && key < kv4_window_start(seen, p.window))) sc[u][t][j] = -INFINITY;
              }
            } else if (key < start || key >= last) {
#pragma unroll
              for (int t = 0; t < NT; ++t) sc[u][t][j] = -INFINITY;
            }
          }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float top0 = fmaxf(fmaxf(sc[0][t][0], sc[0][t][2]), fmaxf(sc[1][t][0], sc[1][t][2]));
        const float top1 = fmaxf(fmaxf(sc[0][t][1], sc[0][t][3]), fmaxf(sc[1][t][1], sc[1][t][3]));
        if (__any_sync(0xffffffffu, top0 > line[t][0] || top1 > line[t][1])) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = j ? top1 : top0;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (top > line[t][j]) {
              const float alpha = dec4_exp2(mx[t][j] - top);
              mx[t][j] = top;
              line[t][j] = top + kDec4Gap;
              l[t][j] *= alpha;
#pragma unroll
              for (int m = 0; m < D / 16; ++m) {
                o[t][m][j] *= alpha;
                o[t][m][2 + j] *= alpha;
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = dec4_exp2(sc[u][t][j] - mx[t][j & 1]);
          l[t][0] += e[0] + e[2];
          l[t][1] += e[1] + e[3];
          pt[u][t][0] = transpose8x8(pack_bf16x2(e[0], e[1]));
          pt[u][t][1] = transpose8x8(pack_bf16x2(e[2], e[3]));
        }
      }
    };
    // values: keys tq, 7 - tq and the same plus 8. What lies behind the last key has probability 0, and every byte is a finite scale
    auto value_products = [&](const uint8_t* unit, const uint32_t (&pt)[NT][2]) {
      uint32_t w[4][D / 64], s4[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint8_t* x = unit + (r & 1 ? w_at : v_at) + (r >> 1) * kOther;
        const uint8_t* y = unit + (r & 1 ? ws_at : vs_at) + (r >> 1) * kOtherScale;
        if (D == 128) {
          const uint2 z = *reinterpret_cast<const uint2*>(x);
          w[r][0] = z.x; w[r][D / 64 - 1] = z.y;
          s4[r] = *reinterpret_cast<const uint32_t*>(y);
        } else {
          w[r][0] = *reinterpret_cast<const uint32_t*>(x);
          s4[r] = *reinterpret_cast<const uint16_t*>(y);
        }
      }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        // scale bytes of a pair of keys, then where a bf16 has them
        const uint32_t sel = 0x0400u + 0x0101u * b;
        const uint32_t s01[2] = {(__byte_perm(s4[0], s4[1], sel) & 0x00ff00ffu) * sixteen + value_bias, (__byte_perm(s4[2], s4[3], sel) & 0x00ff00ffu) * sixteen + value_bias};
        const uint32_t off[2] = {scaled_bf16x2(offset, s01[0]), scaled_bf16x2(offset, s01[1])};
        uint32_t a[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j) {                // byte j of this block's half of the words: values of two products' rows g and g + 8
            const uint32_t x = __byte_perm(w[2 * r][b / 2], w[2 * r + 1][b / 2], (b & 1 ? 0x7632 : 0x5410) + (j ? 0x0101 : 0));
            a[j][2 * r] = fma_bf16x2(masked_or(x, 0x000f000fu, 0x43004300u), s01[r], off[r]);
            a[j][2 * r + 1] = fma_bf16x2(masked_or(x >> 4, 0x000f000fu, 0x43004300u), s01[r], off[r]);
          }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_bf16(o[t][2 * b], a[0], pt[t][0], pt[t][1]);
          mma_bf16(o[t][2 * b + 1], a[1], pt[t][0], pt[t][1]);
        }
      }
    };
    // The pairs that have units of this sequence. One that reaches into the next sequence is kept for it.
    int key0 = (first - at_rel + 2 * i) * kKv4Unit;
    for (int rel = 2 * i; ok && rel < stop; key0 += 2 * kKv4Unit) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][slot], phase, abort_flag)))) break;
      const uint8_t* unit = ring + slot * 2 * kUnit;
      float sc[2][NT][4];
      uint32_t pt[2][NT][2];
      key_products(unit, sc);
      softmax(sc, pt, key0);
      value_products(unit, pt[0]);
      value_products(unit + kUnit, pt[1]);
      rel += 2;
      if (rel > stop && stop < units) break;
      __syncwarp();
      fetch(i + kDec4Stages, slot);
      ++i;
      phase ^= slot;
      slot ^= 1;
    }

#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], d);
    if (at_rel >= 0 && at_rel + n <= units) {
      // all of the sequence: neighbouring lane groups exchange a head each, so that both have pairs of neighbouring values
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float inv0 = l[t][0] == 0.f ? 0.f : 1.f / l[t][0], inv1 = l[t][1] == 0.f ? 0.f : 1.f / l[t][1];
        const int col = 8 * t + 2 * tq + (g & 1);
        __nv_bfloat16* dst = p.out + (col < cols.n ? cols.row(col) * D : 0) + (g & 6);
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float v0 = o[t][m][2 * r] * inv0, v1 = o[t][m][2 * r + 1] * inv1;
            const float got = __shfl_xor_sync(0xffffffffu, g & 1 ? v0 : v1, 4);
            if (col < cols.n) *reinterpret_cast<uint32_t*>(dst + m * 16 + r * 8) = g & 1 ? pack_bf16x2(got, v1) : pack_bf16x2(v0, got);
          }
      }
    } else {
      // a part of it, kept until the end: the first one in memory of its own, the last one in the ring, which has done its work by then
      const int which = at_rel < 0 ? 0 : 1;
      float* park = which ? reinterpret_cast<float*>(ring) : merge + warp * 8 * NT * kPitch;
      __syncwarp();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* row = park + (8 * t + 2 * tq + j) * kPitch;
#pragma unroll
          for (int m = 0; m < D / 16; ++m) {
            row[m * 16 + g] = o[t][m][j];
            row[m * 16 + 8 + g] = o[t][m][2 + j];
          }
          if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(l[t][j] == 0.f ? -INFINITY : mx[t][j], l[t][j]);
        }
      if (lane == 0) parked[warp][which] = Dec4Part{s, h, at_rel + w0, n};
    }
    done = stop;
  }
  if (!ok) {
    // copies in flight end before the block does, whichever warp gave up: the block's flag, which is set by now, would end these waits at once
    for (int j = 0; j < kDec4Stages; ++j) {
      uint32_t alone = 0;
      if (i + j < mine) mbar_wait(&full[warp][slot], phase, &alone, 1 << 22);
      phase ^= slot;
      slot ^= 1;
    }
    if (lane == 0) report_status(p.pool.status, kWaitTimeout, kKernelKv4, 43, blockIdx.x);
  }
  __syncthreads();

  // Parts of the same sequence in a row of warps: owned by the warp where it begins, or by the block (job 0) where that is before it
  for (int job = 0; job <= kDec4Warps; ++job) {
    int from = job - 1, which = 1;
    if (job == 0) {
      for (from = 0; from < kDec4Warps && parked[from][0].s < 0 && parked[from][1].s < 0; ++from) {}       // warps without units
      which = 0;
      if (from == kDec4Warps || parked[from][0].s < 0 || parked[from][0].rel >= 0) continue;
    } else if (parked[from][1].s < 0) {
      continue;
    }
    const Dec4Part seq = parked[from][which];
    bool in[kDec4Warps];                               // warps with parts of it, all but the owner's in slot 0
#pragma unroll
    for (int w = 0; w < kDec4Warps; ++w) in[w] = w == from || (w > from && parked[w][0].s == seq.s && parked[w][0].h == seq.h);
    const Dec4Columns cols(p, kFew, seq.s, seq.h);
    const bool all = seq.rel >= 0 && seq.rel + seq.n <= share;
    float* dst_part = kShares ? p.parts + (static_cast<long long>(blockIdx.x) * 2 + (seq.rel < 0 ? 0 : 1)) * p.chunk_heads * (D + 4) : nullptr;
    for (int col = warp; col < cols.n; col += kDec4Warps) {
      const int c = lane * (D / 32);
      float2 ml[kDec4Warps];
      float top = -INFINITY, den = 0.f, acc[D / 32];
      auto row = [&](int w) { return (w == from && which ? reinterpret_cast<const float*>(smem + w * kDec4Stages * 2 * kUnit) : merge + w * 8 * NT * kPitch) + col * kPitch; };
#pragma unroll
      for (int w = 0; w < kDec4Warps; ++w) {
        ml[w] = in[w] ? *reinterpret_cast<const float2*>(row(w) + D) : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[w].x);
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j) acc[j] = 0.f;
#pragma unroll
      for (int w = 0; w < kDec4Warps; ++w)
        if (in[w]) {
          const float wt = ml[w].x == top ? 1.f : dec4_exp2(ml[w].x - top);
          const float* x = row(w) + c;
          den = fmaf(wt, ml[w].y, den);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) acc[j] = fmaf(wt, x[j], acc[j]);
        }
      if (all) {
        const float inv = den == 0.f ? 0.f : 1.f / den;
        __nv_bfloat16* dst = p.out + cols.row(col) * D + c;
#pragma unroll
        for (int j = 0; j < D / 32; j += 2) *reinterpret_cast<uint32_t*>(dst + j) = pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
      } else {
        float* dst = dst_part + col * (D + 4);
#pragma unroll
        for (int j = 0; j < D / 32; j += 2) *reinterpret_cast<float2*>(dst + c + j) = make_float2(acc[j], acc[j + 1]);
        if (lane == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(top, den);
      }
    }
  }
}

// Joins the parts of sequences that several blocks share; zeros for those without keys. One block per (sequence, part of a kv head's heads)
// with a warp per head, or (kSlices 8, where a sequence has many parts) one block per head whose warps take every eighth part.
template <int D, int kSlices>
__global__ void __launch_bounds__(256) join_decode_kv4_kernel(const DecodeKv4Params p) {
  __shared__ __align__(8) float sums[kSlices > 1 ? 8 : 1][D + 4];
  pdl_wait();
  pdl_trigger();
  const int heads_v = p.pool.hkv * p.chunks, s = blockIdx.x / heads_v, h = blockIdx.x - s * heads_v;
  const long long total = static_cast<long long>(p.prefix[p.seqs]) * heads_v, shares = dec4_shares(p, total);
  const int n = p.prefix[s + 1] - p.prefix[s];
  const long long at = static_cast<long long>(p.prefix[s]) * heads_v + static_cast<long long>(h) * n;
  const Dec4Columns cols(p, p.cu_q != nullptr, s, h);
  // block of unit f: the last whose share starts at or before it
  const auto block_of = [&](long long f) {
    const long long x = (f + 1) * shares - 1;
    return (x | total) >> 32 ? static_cast<int>(x / total) : static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(total));
  };
  const int c0 = n > 0 ? block_of(at) : 0, c1 = n > 0 ? block_of(at + n - 1) : 0;
  if (n > 0 && c0 == c1) return;                     // one block had all of it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kEach = D / 32;                      // values of a lane
  for (int col = kSlices > 1 ? blockIdx.y : warp; col < cols.n; col += kSlices > 1 ? p.chunk_heads : 8) {
    // the first part is the second one of its block: the sequence starts in that share
    auto part = [&](int c) { return p.parts + ((static_cast<long long>(c) * 2 + (c == c0 ? 1 : 0)) * p.chunk_heads + col) * (D + 4); };
    float top = -INFINITY, den = 0.f, acc[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) acc[j] = 0.f;
    // four parts at a time, all of whose loads are on their way at once; the reference rises as it has to
    for (int c = n > 0 ? c0 + (kSlices > 1 ? warp : 0) : c1 + 1; c <= c1; c += 4 * kSlices) {
      float2 ml[4], v[4][kEach / 2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        if (c + u * kSlices <= c1) {
          const float* x = part(c + u * kSlices);
          ml[u] = *reinterpret_cast<const float2*>(x + D);
#pragma unroll
          for (int j = 0; j < kEach / 2; ++j) v[u][j] = *reinterpret_cast<const float2*>(x + lane * kEach + 2 * j);
        }
      }
      const float now = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top);
      const float alpha = top == now ? 1.f : dec4_exp2(top - now);
      top = now;
      den *= alpha;
#pragma unroll
      for (int j = 0; j < kEach; ++j) acc[j] *= alpha;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * kSlices <= c1) {
          const float w = ml[u].x == top ? 1.f : dec4_exp2(ml[u].x - top);
          den = fmaf(w, ml[u].y, den);
#pragma unroll
          for (int j = 0; j < kEach / 2; ++j) {
            acc[2 * j] = fmaf(w, v[u][j].x, acc[2 * j]);
            acc[2 * j + 1] = fmaf(w, v[u][j].y, acc[2 * j + 1]);
          }
        }
    }
    if (kSlices > 1) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) sums[warp][lane * kEach + j] = acc[j];
      if (lane == 0) *reinterpret_cast<float2*>(&sums[warp][D]) = make_float2(top, den);
      __syncthreads();
      if (warp) return;
      float2 ml[8];
      top = -INFINITY;
      den = 0.f;
#pragma unroll
      for (int j = 0; j < kEach; ++j) acc[j] = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        ml[w] = *reinterpret_cast<const float2*>(&sums[kSlices > 1 ? w : 0][D]);
        top = fmaxf(top, ml[w].x);
      }
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float wt = ml[w].x == top ? 1.f : dec4_exp2(ml[w].x - top);
        den = fmaf(wt, ml[w].y, den);
#pragma unroll
        for (int j = 0; j < kEach; ++j) acc[j] = fmaf(wt, sums[kSlices > 1 ? w : 0][lane * kEach + j], acc[j]);
      }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    __nv_bfloat16* out = p.out + cols.row(col) * D;
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
// Sixteen columns at a time take one block of a processor, eight two: a walk of eight costs 0.6 to 0.7 of one of sixteen, so three replace two. 20
// columns behind 16 times 3000 keys 55.5 us (55.0 with two of ten), with heads of 64 36.7 (41.8); 128 sequences of 6000 tokens and 20 heads over
// one 57 (62) with heads of 64 and 90 (86) with 128; 64 of 3000 34 (36); eight of 100 tokens 7.2 (9.0).
static void dec4_chunks(int columns, int& chunks, int& heads) {
  chunks = columns > 16 && columns <= 24 ? 3 : (columns + 15) / 16;
  heads = (columns + chunks - 1) / chunks;
}
static long long dec4_workspace(int seqs, int columns, int hkv, int d, int max_kv_len) {
  int chunks, heads;
  dec4_chunks(columns, chunks, heads);
  const int blocks = dec4_blocks(seqs, hkv * chunks, heads, max_kv_len);
  return blocks == 0 ? 0 : static_cast<long long>(blocks) * 2 * heads * (d + 4) * 4 + (seqs + 1ll) * 4;
}

static int dec4_run(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, const int* cu_q, int seqs, int max_q_len,
                    int hq, int hkv, int d, int page, int max_pages, long long pages, int max_kv_len, int window, float scale,
                    float softcap, void* workspace, long long workspace_bytes, void* status, cudaStream_t stream) {
  if (seqs <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || max_pages < 1 || pages < 1 || !kv4_pool_fits(pool, d, page)) return -2;
  const long long columns = static_cast<long long>(max_q_len) * (hq / hkv), units = static_cast<long long>(max_pages) * (page / kKv4Unit);
  if (columns >= (1ll << 20) || units * seqs >= (1ll << 31)) return -3;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) return -4;
  DecodeKv4Params p{};
  dec4_chunks(static_cast<int>(columns), p.chunks, p.chunk_heads);
  if (units * hkv * p.chunks >= (1ll << 32)) return -3;        // the kernels divide the units of a sequence in 32 bits
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.kv_lens = kv_lens;
  p.cu_q = cu_q;
  p.pool = Kv4Pool{static_cast<const uint8_t*>(pool), block_table, pages, hkv, max_pages, kv4_unit_shift(page), static_cast<DeviceStatus*>(status)};
  p.seqs = seqs; p.hq = hq; p.group = hq / hkv;
  p.window = window;
  p.scale_log2 = scale * kDec4Log2e;
  if (softcap > 0.f) {
    p.cap_in = 2.f * kDec4Log2e * scale / softcap;
    p.cap_out = softcap * kDec4Log2e;
  }
  const long long pairs = static_cast<long long>(seqs) * hkv * p.chunks;
  if (pairs >= (1ll << 31)) return -3;
  const long long seen = window + (max_q_len - 1ll);  // keys that some query of a sequence sees
  if (window > 0 && seen < max_kv_len) max_kv_len = static_cast<int>(min(static_cast<long long>(max_kv_len), seen + kKv4Unit));
  p.blocks = dec4_blocks(seqs, hkv * p.chunks, p.chunk_heads, max_kv_len);
  const bool shares = p.blocks > 0;
  if (cu_q && !shares) return -6;                    // short caches and many sequences are for the other kernels
  if (shares) {
    const long long floats = static_cast<long long>(p.blocks) * 2 * p.chunk_heads * (d + 4);
    if (!workspace || workspace_bytes < floats * 4 + (seqs + 1ll) * 4) return -5;
    p.parts = static_cast<float*>(workspace);
    p.prefix = reinterpret_cast<int*>(p.parts + floats);
  }
  const bool two = p.chunk_heads > 8;
  const int most = dec4_smem_bytes(d, two ? 2 : 1), smem = most - (shares ? kDec4MaxSeqs - seqs : kDec4MaxSeqs + 1) * 4;
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kernel, PerDeviceOnce& o) {
    if (o.first_time()) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) e = launch_pdl(kernel, dim3(static_cast<unsigned>(shares ? p.blocks : pairs)), dim3(kDec4Threads), smem, stream, p);
  };
  auto pick = [&](auto dim, auto tiles, auto few) {
    static PerDeviceOnce once[2];
    if constexpr (few()) go(attn_decode_kv4_kernel<dim(), tiles(), true, true>, once[0]);
    else if (shares) go(attn_decode_kv4_kernel<dim(), tiles(), true, false>, once[0]);
    else go(attn_decode_kv4_kernel<dim(), tiles(), false, false>, once[1]);
  };
  auto pick_few = [&](auto dim, auto tiles) {
    if (cu_q) pick(dim, tiles, std::true_type{}); else pick(dim, tiles, std::false_type{});
  };
  using std::integral_constant;
  if (d == 128) {
    if (two) pick_few(integral_constant<int, 128>{}, integral_constant<int, 2>{}); else pick_few(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  } else {
    if (two) pick_few(integral_constant<int, 64>{}, integral_constant<int, 2>{}); else pick_few(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  }
  if (e != cudaSuccess) return -static_cast<int>(e) - 300;
  if (!shares) return 1;
  // a warp takes 0.3 us a part: with a dozen of them a block per head is faster, with a few the blocks' own start is what counts
  const bool many = p.blocks >= 8 * pairs;
  const dim3 grid(static_cast<unsigned>(pairs), many ? p.chunk_heads : 1);
  if (d == 128) e = many ? launch_pdl(join_decode_kv4_kernel<128, 8>, grid, dim3(256), 0, stream, p) : launch_pdl(join_decode_kv4_kernel<128, 1>, grid, dim3(256), 0, stream, p);
  else e = many ? launch_pdl(join_decode_kv4_kernel<64, 8>, grid, dim3(256), 0, stream, p) : launch_pdl(join_decode_kv4_kernel<64, 1>, grid, dim3(256), 0, stream, p);
  return e == cudaSuccess ? 2 : -static_cast<int>(e) - 400;
}

}  // namespace b200

using namespace b200;

// Bytes of workspace for these sizes (0: none is used).
B200_API long long b200_attn_decode_kv4_workspace(int seqs, int hq, int hkv, int d, int max_kv_len) {
  return seqs <= 0 || hkv < 1 || hq < hkv || hq % hkv ? 0 : dec4_workspace(seqs, hq / hkv, hkv, d, max_kv_len);
}

// q, out [sequences][hq][d] bf16. window > 0: the last `window` keys. max_kv_len chooses how the work is cut, nothing else; the workspace
// (16-byte aligned) is of the size that b200_attn_decode_kv4_workspace gives for the same sizes. Returns the number of launches.
B200_API int b200_attn_decode_kv4(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, int seqs, int hq,
                                  int hkv, int d, int page, int max_pages, long long pages, int max_kv_len, int window, float scale,
                                  float softcap, void* workspace, long long workspace_bytes, void* status, cudaStream_t stream) {
  return dec4_run(q, pool, out, block_table, kv_lens, nullptr, seqs, 1, hq, hkv, d, page, max_pages, pages, max_kv_len, window, scale, softcap,
                  workspace, workspace_bytes, status, stream);
}

// A few queries per sequence behind a long cache: q, out [tokens][hq][d] packed by cu_q [sequences + 1], causal. Columns of the products are
// (query, head) pairs, 16 at a time, each time over all units. For more than 512 keys and at most 256 sequences. The workspace is of the size that b200_attn_few_kv4_workspace gives.
B200_API long long b200_attn_few_kv4_workspace(int seqs, int max_q_len, int hq, int hkv, int d, int max_kv_len) {
  if (seqs <= 0 || max_q_len < 1 || hkv < 1 || hq < hkv || hq % hkv || static_cast<long long>(max_q_len) * (hq / hkv) >= (1ll << 20)) return 0;
  return dec4_workspace(seqs, max_q_len * (hq / hkv), hkv, d, max_kv_len);
}
B200_API int b200_attn_few_kv4(const void* q, const void* pool, void* out, const int* block_table, const int* kv_lens, const int* cu_q, int seqs,
                               int max_q_len, int hq, int hkv, int d, int page, int max_pages, long long pages, int max_kv_len, int window,
                               float scale, float softcap, void* workspace, long long workspace_bytes, void* status, cudaStream_t stream) {
  if (max_q_len < 1) return 0;
  if (!cu_q) return -2;
  return dec4_run(q, pool, out, block_table, kv_lens, cu_q, seqs, max_q_len, hq, hkv, d, page, max_pages, pages, max_kv_len, window, scale, softcap,
                  workspace, workspace_bytes, status, stream);
}
