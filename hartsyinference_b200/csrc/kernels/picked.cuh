// Pages that queries choose: what the kernels of the bounds, the choice and the attention over it share.
//
// Queries choose in runs of `run` neighbouring tokens of a sequence. Rows of runs are packed: run r of sequence s is row
// (cu_q[s] + s (run - 1)) / run + r, which leaves a row unused at most between two sequences. A row holds, for every key head, page numbers
// of the sequence in order, then -1.
//
// Bounds of the keys of a page and key head, 2 D + 16 bytes: D codes of the largest value of every channel, D of the smallest, then
// e + 64 and zeros. e is the smallest exponent from -50 to 50 with max |value| <= 127 * 2^e; codes are rounded away from the page's values.
#pragma once
#include "common.cuh"

namespace b200 {

int num_sms();      // of the current device, see gemm_tcgen05.cu

constexpr int kBoundsTail = 16;
constexpr int kBoundsBias = 64;

// Smallest e in [-50, 50] with top <= 127 * 2^e (top >= 0, not NaN).
__device__ __forceinline__ int bounds_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int x = static_cast<int>(bits >> 23) - 127;              // top = (1 + m / 2^23) 2^x, and 127 = 1.984375 * 2^6
  const int e = x - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return min(50, max(-50, e));
}
__device__ __forceinline__ float bounds_pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Sequence of a row of runs: the last one whose rows begin at or before it (all lanes of a warp take part).
__device__ __forceinline__ int row_sequence(const int* __restrict__ cu_q, int seqs, int run, int row) {
  if (cu_q == nullptr) return row;
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = seqs;                            // sequence lo begins there, hi does not
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const bool before = at < hi && (cu_q[at] + static_cast<long long>(at) * (run - 1)) / run <= row;
    const int n = __popc(__ballot_sync(0xffffffffu, before));
    const int top = lo + (n + 1) * step;
    lo += n * step;
    hi = min(hi, top);
  }
  return lo;
}

struct RunOfRow {
  int seq, q_off;     // first query of the run
  int tokens;         // <= 0: the row belongs to no run
  int begin, kv_len;  // position of its first query (may be negative: such queries see nothing), keys of the sequence
};

// (tokens: rows of q, behind which no run reaches whatever cu_q holds)
__device__ __forceinline__ RunOfRow run_of_row(const int* __restrict__ cu_q, const int* __restrict__ kv_lens, int seqs, int run, int row, int most_keys, int tokens) {
  RunOfRow r;
  r.seq = row_sequence(cu_q, seqs, run, row);
  const int off = cu_q ? cu_q[r.seq] : r.seq, len = cu_q ? cu_q[r.seq + 1] - off : 1;
  const int first = static_cast<int>((off + static_cast<long long>(r.seq) * (run - 1)) / run);
  const int skip = (row - first) * run;            // queries of the sequence in front of the run
  r.q_off = off + skip;
  r.tokens = skip < 0 || off < 0 ? 0 : min(min(run, len - skip), tokens - r.q_off);
  r.kv_len = min(kv_lens[r.seq], most_keys);
  r.begin = r.kv_len - len + skip;
  return r;
}

}  // namespace b200
