// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i is accepted iff u_i q_i(d_i) < p_i(d_i) (q_i(d_i) = 1 for drafts without probabilities); the
// first refusal ends the run.  Then one token is sampled: from max(p_i - q_i, 0) at a refused draft (p_i
// without d_i for drafts without probabilities), from the row after the last accepted draft else.
//
// Which token that is must not depend on the order of a sum.  So a probability x counts as the whole
// number floor(clamp(x, 0, 1) 2^42) (x = fp32(p - q)), sums are exact in 64 bits (2^18 values of 1 fill
// 60), and the token is the first whose running sum passes floor(floor(u 2^24) total / 2^24).  The
// product u q of two fp32 numbers is exact in 64-bit floating point, so acceptance is exact too.
//
// The floor is one row of p, and one of q where a draft is refused.  A cluster takes a request: every
// warp sums a run of the row, the warps' sums are pushed to all blocks of the cluster, and the block
// whose warp's run holds the token reads that run again (from L2), a thread a few values.
#include <algorithm>

#include "common.cuh"
#include "runtime.h"

namespace vlc {
namespace verify {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCKS = 8;
constexpr int MAX_DRAFTS = 32;
constexpr int MAX_VOCAB = 1 << 18;
constexpr float COUNT = 4398046511104.f;  // 2^42

struct Params {
  const int64_t* drafts;
  int64_t draft_stride;
  const void* p;
  const void* q;  // null: drafts without probabilities
  int64_t p_seq, p_row, q_seq, q_row;  // strides
  const float* u;
  int64_t u_stride;
  const float* u_last;
  int64_t* tokens;   // [num_seqs][num_drafts + 1]
  int32_t* emitted;
  int num_drafts, vocab;
  int run;           // values of a warp, a multiple of THREADS
};

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  return (float)x;
}
__device__ __forceinline__ uint64_t count_of(float x) {
  // (NaN counts as 0)
  return (uint64_t)__float2ull_rz(fminf(fmaxf(x, 0.f), 1.f) * COUNT);
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// The row that the token is sampled from.
template <typename T>
struct Row {
  const T* p;
  const T* q;   // null: none to take off
  int without;  // value that counts as 0 (-1: none)
  __device__ __forceinline__ uint64_t count(int v) const {
    float x = (float)__ldg(p + v);
    if (q) x = __fsub_rn(x, (float)__ldg(q + v));
    return v == without ? 0 : count_of(x);
  }
};

// The sum of a warp's run [v0, v1).
template <typename T>
__device__ __forceinline__ uint64_t sum_of(const Row<T>& row, int v0, int v1, int lane) {
  uint64_t sum = 0;
#pragma unroll 8
  for (int v = v0 + lane; v < v1; v += 32) sum += row.count(v);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) verify_kernel(const Params a) {
  __shared__ uint64_t sums[MAX_BLOCKS * WARPS];  // of all warps of the cluster
  __shared__ uint64_t upto[WARPS];
  __shared__ int s_taken, s_refused;
  const int rank = (int)cluster_ctarank(), blocks = gridDim.x, warps = blocks * WARPS;
  const int seq = blockIdx.y, warp = warp_id(), lane = lane_id();
  const int64_t* const drafts = a.drafts + seq * a.draft_stride;
  const T* const p0 = (const T*)a.p + seq * a.p_seq;
  const T* const q0 = (const T*)a.q + seq * a.q_seq;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for before the first push)

  // ---- acceptance, in every block
  if (warp == 0) {
    bool live = false, taken = false;
    if (lane < a.num_drafts) {
      const int64_t d = drafts[lane];
      live = d >= 0 && d < a.vocab;
      if (d >= a.vocab && rank == 0) record_error(VLC_DEV_ERR_TOKEN);
      if (live) {
        const float there = (float)__ldg(p0 + lane * a.p_row + d);
        const float draft = a.q ? (float)__ldg(q0 + lane * a.q_row + d) : 1.f;
        taken = (double)a.u[seq * a.u_stride + lane] * (double)draft < (double)there;
      }
    }
    const uint32_t yes = __ballot_sync(0xffffffffu, taken), have = __ballot_sync(0xffffffffu, live);
    const int n = __ffs(~yes) == 0 ? 32 : __ffs(~yes) - 1;
    if (lane == 0) {
      s_taken = n;
      s_refused = n < a.num_drafts && (have >> n & 1);
    }
  }
  __syncthreads();
  const int taken = s_taken;
  const bool refused = s_refused != 0;
  Row<T> row;
  row.p = p0 + taken * a.p_row;
  row.q = refused && a.q ? q0 + taken * a.q_row : nullptr;
  row.without = refused && !a.q ? (int)drafts[taken] : -1;

  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // The second round, over p alone, is for a difference that has no positive value.
  for (int round = 0;; ++round) {
    const int me = rank * WARPS + warp;
    const int v0 = min(a.vocab, me * a.run), v1 = min(a.vocab, v0 + a.run);
    const uint64_t sum = sum_of(row, v0, v1, lane);
    if (lane < blocks) st_cluster_u64(mapa_shared(smem_u32(sums + me), lane), sum);
    cluster_sync();
    // ---- where the token is: every warp of the cluster finds it for itself
    uint64_t total = 0, mine[(MAX_BLOCKS * WARPS + 31) / 32], before = 0;
#pragma unroll
    for (int x = 0; x < (MAX_BLOCKS * WARPS + 31) / 32; ++x) {
      uint64_t v = x * 32 + lane < warps ? sums[x * 32 + lane] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += y;
      }
      mine[x] = total + v;
      total += __shfl_sync(0xffffffffu, v, 31);
    }
    int64_t token = -1;
    bool writer = false;
    if (total > 0) {
      const float u = fminf(fmaxf(a.u_last[seq], 0.f), 1.f - 0x1p-24f);
      const uint64_t goal = __umul64hi((uint64_t)(u * 0x1p24f) << 40, total);
      int where = 0;
#pragma unroll
      for (int x = 0; x < (MAX_BLOCKS * WARPS + 31) / 32; ++x) {
        const uint32_t past = __ballot_sync(0xffffffffu, mine[x] > goal);
        const uint32_t low = ~past;  // sums not past the goal come first
        where += __popc(low);
        const uint64_t last = past == 0xffffffffu ? 0 : __shfl_sync(0xffffffffu, mine[x], 31 - __clz(low | 1));
        if (low != 0) before = last;
      }
      if (where / WARPS != rank) return;
      // ---- the token in that run: a thread takes run / THREADS values
      const int each = a.run / THREADS, w0 = where * a.run + threadIdx.x * each;
      uint64_t own = 0;
      for (int v = w0; v < min(a.vocab, w0 + each); ++v) own += row.count(v);
      uint64_t end = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, end, d);
        if (lane >= d) end += y;
      }
      if (lane == 31) upto[warp] = end;
      __syncthreads();
      for (int w = 0; w < warp; ++w) before += upto[w];
      end += before;
      writer = end > goal && end - own <= goal;
      if (writer) {
        uint64_t at = end - own;
        int v = w0;
        while ((at += row.count(v)) <= goal) ++v;
        token = v;
      }
    } else if (round == 0 && refused) {
      row.q = nullptr;
      row.without = -1;
      cluster_sync();  // every block has read its sums
      continue;
    } else {
      writer = rank == 0 && threadIdx.x == 0;  // no value is positive: no token
    }
    if (writer) {
      int64_t* const out = a.tokens + (int64_t)seq * (a.num_drafts + 1);
      for (int i = 0; i <= a.num_drafts; ++i) out[i] = i < taken ? drafts[i] : i == taken ? token : -1;
      a.emitted[seq] = taken + 1;
    }
    return;
  }
}

template <typename T>
static int launch(const Params& a, int num_seqs, int blocks, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, num_seqs);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, verify_kernel<T>, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}

}  // namespace verify
}  // namespace vlc

using namespace vlc;
using namespace vlc::verify;

extern "C" int vlc_verify_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                                 const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                                 const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride, int vocab,
                                 int dtype, const float* u, int64_t u_stride, const float* u_last, int64_t* tokens,
                                 int32_t* emitted, void* stream) {
  if (num_seqs < 0 || num_seqs > 65535 || num_drafts < 0 || vocab <= 0) return VLC_ERR_SHAPE;
  if (num_drafts > MAX_DRAFTS - 1 || vocab > MAX_VOCAB || dtype < 0 || dtype > 2) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0) return VLC_OK;
  if (!target_probs || !u_last || !tokens || !emitted || (num_drafts > 0 && (!drafts || !u))) return VLC_ERR_NULL;
  Params a;
  a.drafts = drafts;
  a.draft_stride = draft_stride;
  a.p = target_probs;
  a.q = num_drafts > 0 ? draft_probs : nullptr;
  a.p_seq = target_seq_stride;
  a.p_row = target_row_stride;
  a.q_seq = draft_seq_stride;
  a.q_row = draft_row_stride;
  a.u = u;
  a.u_stride = u_stride;
  a.u_last = u_last;
  a.tokens = tokens;
  a.emitted = emitted;
  a.num_drafts = num_drafts;
  a.vocab = vocab;
  const int blocks = MAX_BLOCKS;
  a.run = ((vocab + blocks * WARPS - 1) / (blocks * WARPS) + THREADS - 1) / THREADS * THREADS;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == 0 ? launch<float>(a, num_seqs, blocks, st)
         : dtype == 1 ? launch<__nv_bfloat16>(a, num_seqs, blocks, st)
                      : launch<__half>(a, num_seqs, blocks, st);
}
