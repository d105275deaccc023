// What the kernels of windowed paged decode attention share: their parameters, the chunks of keys that a sequence
// sees, and the line of all chunks that a grid's blocks share out (decode_window.cu, decode_window_wide.cu).
#pragma once

#include "common.cuh"

namespace vlc {
namespace decode_window {

constexpr int HD = 128;
constexpr int MIN_BLOCK = 32;            // a page's tokens are a multiple of it
constexpr int MAX_ROWS = 128;           // tokens x query heads of a KV head
constexpr float SLACK = 8.f;            // log2 that the maximum may grow by before O is rescaled
constexpr float NO_MAX = -3e38f;        // the maximum of no key (finite: differences of two are numbers)

struct Params {
  // decode_window.cu: {64 dims, Hk, slots, 2 halves of a row, caches}, box {64, 1, 16, 2, caches}.  Joined, the caches are
  // the two, whose stride is their distance (v_first: V lies before K); else kv[0] is K and kv[1] V.
  // decode_window_wide.cu: K and V, {64 dims, Hk, slots, 2 halves}, box {64, 1, WIDE_BOX, 1}.
  CUtensorMap kv[2];
  bool joined, v_first;
  const __nv_bfloat16* q;
  int64_t q_token_stride;
  const int32_t* block_tables;
  int64_t table_stride;
  int table_width, block_size, num_pages;
  const int32_t* context_lens;
  int num_seqs, max_len, tokens, window, sinks;
  int group, num_kv_heads, rows;  // rows = tokens * group
  uint32_t group_inverse;         // 2^16 / group, rounded up: exact for rows below 128
  __device__ __forceinline__ int token_of(int row) const { return (int)((uint32_t)row * group_inverse >> 16); }
  int cluster;                    // blocks of a pair's cluster (0: the line)
  float scale_log2;               // |softmax scale| * log2(e), above 0: a hidden key's score stays -infinity
  uint32_t q_flip;                // the signs of a pair of q's elements where the scale is negative
  __nv_bfloat16* out;
  int64_t out_token_stride;
  int num_blocks;
  // Workspace: a block's first pair and its last leave parts when they are not whole.
  float* parts;     // [num_blocks][2][rows][HD] sums of P V
  float2* part_ml;  // [num_blocks][2][rows] (maximum, sum of P)
  int2* places;     // [num_seqs][num_kv_heads] of each pair with keys: (slot of its first part, parts)
};

// The chunks of a sequence that any of its rows sees: chunk v is v for v < first (of the sinks), and
// v + jump from there on.
template <int CK>  // keys of a chunk
struct Span {
  int len;          // cut to the host's bound
  int low;          // first key of the window of the sequence's first row
  int first, jump;
  int count;
  // Chunks whose keys every row sees: [0, all0) of the sinks and [all1, all2): they end by the first row's
  // position and begin in the last row's window.
  __device__ __forceinline__ int all0(const Params& p) const { return min(first, p.sinks / CK); }
  __device__ __forceinline__ int all1(const Params& p) const {
    return p.window > 0 ? max(first, (max(0, len - p.window) + CK - 1) / CK - jump) : 0;
  }
  __device__ __forceinline__ int all2(const Params& p) const { return (len - p.tokens + 1) / CK - jump; }
};
template <int CK>
__device__ __forceinline__ Span<CK> span_of(const Params& p, int len) {
  Span<CK> s;
  s.len = min(max(len, 0), p.max_len);
  s.low = p.window > 0 ? max(0, s.len - p.tokens - p.window + 1) : 0;
  const int wc = s.low / CK;
  s.first = min(wc, (p.sinks + CK - 1) / CK);
  s.jump = wc - s.first;
  s.count = (s.len + CK - 1) / CK - s.jump;
  return s;
}

// How the line of `total` chunks is shared: every block takes each() of them and the first extra()
// one more.
struct Shares {
  int64_t each, extra;
  __device__ __forceinline__ Shares(int64_t total, int blocks) : each(total / blocks), extra(total % blocks) {}
  __device__ __forceinline__ int64_t first(int64_t block) const { return block * each + min(block, extra); }
  __device__ __forceinline__ int64_t count(int64_t block) const { return each + (block < extra ? 1 : 0); }
  __device__ __forceinline__ int64_t block_of(int64_t chunk) const {
    const int64_t big = extra * (each + 1);
    return chunk < big ? chunk / (each + 1) : extra + (chunk - big) / each;
  }
};


// A block's run of the line: `count` chunks from chunk c0 on, which is chunk j0 of the pair (seq, head).
template <int CK>
struct Run {
  int seq = 0, head = 0, j0 = 0, count = 0;
  int64_t c0 = 0;
  Span<CK> span;  // of seq
  // On to the pair behind the current one.  Call it only where the run goes on: so does a sequence with keys.
  __device__ __forceinline__ void next_pair(const Params& p) {
    j0 = 0;
    if (++head < p.num_kv_heads) return;
    head = 0;
    do {
      span = span_of<CK>(p, __ldg(p.context_lens + ++seq));
    } while (span.count <= 0);
  }
};
// Each warp finds the block's run for itself.
template <int CK>
__device__ __forceinline__ Shares run_of(const Params& p, Run<CK>& run, int warp, int lane) {
  int64_t total = 0;
  for (int i = lane; i < p.num_seqs; i += 32) {
    const int len = __ldg(p.context_lens + i);
    if (blockIdx.x == 0 && warp == 0 && len > p.max_len) record_error(VLC_DEV_ERR_LENGTH);
    total += span_of<CK>(p, len).count;
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  const Shares all(total * p.num_kv_heads, p.num_blocks);
  run.c0 = all.first(blockIdx.x);
  run.count = (int)all.count(blockIdx.x);
  int64_t at = run.c0;  // c0's place among the chunks from the sequence's first on
  for (int base = 0; run.count > 0 && base < p.num_seqs; base += 32) {
    const int64_t n = base + lane < p.num_seqs
                          ? (int64_t)span_of<CK>(p, __ldg(p.context_lens + base + lane)).count * p.num_kv_heads
                          : 0;
    int64_t upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, upto > at);
    if (past) {
      const int first = __ffs(past) - 1;
      run.seq = base + first;
      at -= __shfl_sync(0xffffffffu, upto - n, first);
      break;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
  }
  run.span = span_of<CK>(p, __ldg(p.context_lens + run.seq));
  if (run.count > 0) {
    run.head = (int)(at / run.span.count);
    run.j0 = (int)(at - (int64_t)run.head * run.span.count);
  }
  return all;
}

// decode_window_wide.cu: chunks of WIDE_CHUNK keys, a block an SM.
constexpr int WIDE_CHUNK = 128;
constexpr int WIDE_BOX = 32;  // keys of a copy; a box of keys that no row sees is not read
int launch_wide(const Params& p, cudaStream_t st);

}  // namespace decode_window
}  // namespace vlc
