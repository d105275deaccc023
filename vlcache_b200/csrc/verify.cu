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
// warp sums a run of the row, tile by tile, the next tile's loads in flight; the warps' sums are pushed to all
// blocks of the cluster, and the block whose warp's run holds the token finds the tile by its kept sum and
// reads that again (from L2), a thread a few values.  As many blocks a request as are resident at once: a
// second wave would wait for its acceptance again.  One request of 151,936 tokens takes 7.8 us (a chain of drafts,
// their probabilities, the row, the cluster's sums and the tile), 64 with four drafts 16.2 (floor 10.0), 256
// without draft probabilities, in bf16, 24 (floor 11.9: one block a request, 256 on 148 SMs).  With conversions to
// whole numbers instead of the additions in 64-bit floating point 16.9 and 39; four blocks an SM (spilling) 18.0
// and 25.4.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace vlc {
namespace verify {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCKS = 8;
constexpr int BLOCKS_PER_SM = 3;
constexpr int MAX_TILES = 33;   // of a warp's run
constexpr int MAX_DRAFTS = 32;
constexpr int MAX_VOCAB = 1 << 18;
constexpr float COUNT = 4398046511104.f;  // 2^42

struct Params {
  const int64_t* drafts;
  int64_t draft_stride;
  const void* p;
  const void* q;
  bool sampled;  // else drafts without probabilities: q is p
  int64_t p_seq, p_row, q_seq, q_row;  // strides
  const float* u;
  int64_t u_stride;
  const float* u_last;
  int64_t* tokens;   // [num_seqs][num_drafts + 1]
  int32_t* emitted;
  int32_t* context_lens;  // null, or moved on by emitted (idle places, below 0, stay)
  const int32_t* block_tables;  // of the step's rows, with block_size; block_size 0: every row is in the cache
  int64_t table_stride;
  int table_width, block_size;
  int num_drafts, vocab;
  int tiles;         // of a warp
};

__device__ __forceinline__ uint64_t count_of(float x) {  // (NaN counts as 0)
  return (uint64_t)__float2ull_rz(__saturatef(x) * COUNT);
}

// A running sum of counts in 64-bit floating point: between 2^10 and 2^11 its last place stands for 2^-42, so
// that adding x rounded down adds floor(x 2^42) places, and its 52 bits are the count.  Up to 1023 values.
struct Counter {
  double at = 1024.0;
  template <bool SHORT>  // x is a 16-bit number
  __device__ __forceinline__ void add(float x) {
    const uint32_t b = __float_as_uint(__saturatef(x));  // (NaN counts as 0, -0.0 saturates to 0.0: tested)
    // the same number in 64 bits, but 2^-127 for 0 and less than 2^-126 for smaller ones
    at = __dadd_rd(at, __hiloint2double((int)((b >> 3) + 0x38000000u), SHORT ? 0 : (int)(b << 29)));
  }
  __device__ __forceinline__ uint64_t count() const {
    return (uint64_t)__double_as_longlong(at) & ((1ull << 52) - 1);
  }
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

template <typename T>
constexpr int kVector = 16 / (int)sizeof(T);  // values of a 16-byte load

// Places of a tile: eight loads a lane.
template <typename T>
constexpr int kTile = 8 * 32 * kVector<T>;

// Value i of a 16-byte load.
__device__ __forceinline__ float value(const uint4& u, int i, const float*) {
  return __uint_as_float(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w);
}
__device__ __forceinline__ float value(const uint4& u, int i, const __nv_bfloat16*) {
  const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
  return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ float value(const uint4& u, int i, const __half*) {
  const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return i & 1 ? __high2float(h) : __low2float(h);
}

// The row that the token is sampled from.  Its values are numbered from the 16-byte boundary before the
// first: value v is at place v + lead, so that runs of places are read in whole vectors.  Every load is of
// a place inside the row: one outside counts 0, and its load is of the nearest inside.
template <typename T>
struct Row {
  const T* p;
  const T* q;         // p where none is to be taken off
  bool both;
  int without;        // value that counts as 0 (-1: none)
  int vocab, lead;
  int first, last;    // places of the first whole vector and the last
  bool vectors;       // p and q lie alike to 16 bytes, and there are whole vectors
  __device__ __forceinline__ void settle() {
    constexpr int N = kVector<T>;
    const int at = (int)(reinterpret_cast<uintptr_t>(p) % 16), other = (int)(reinterpret_cast<uintptr_t>(q) % 16);
    lead = at / (int)sizeof(T);
    first = lead ? N : 0;
    last = (vocab + lead) / N * N - N;
    vectors = at == other && last >= first;
  }
  __device__ __forceinline__ float at(int v) const {
    const float x = (float)__ldg(p + v), y = both ? (float)__ldg(q + v) : 0.f;
    return __fsub_rn(x, y);
  }
  __device__ __forceinline__ uint64_t count(int place) const {
    const int v = place - lead, near = min(max(v, 0), vocab - 1);
    const uint64_t n = count_of(at(near));
    return v != near || v == without ? 0 : n;
  }
  // Sums of the `tiles` tiles from place `begin` on to kept[], by a warp; returns a lane's part of their sum.
  __device__ __forceinline__ uint64_t sum(int begin, int tiles, uint64_t* kept, int lane) const {
    if (!vectors) {
      uint64_t total = 0;
      for (int x = 0; x < tiles; ++x) {
        uint64_t part = 0;
#pragma unroll 8
        for (int y = lane; y < kTile<T>; y += 32) part += count(begin + x * kTile<T> + y);
        total += part;
        keep(part, kept + x, lane);
      }
      return total;
    }
    return both ? sum_vectors<true>(begin, tiles, kept, lane) : sum_vectors<false>(begin, tiles, kept, lane);
  }
  static __device__ __forceinline__ void keep(uint64_t part, uint64_t* kept, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
    if (lane == 0) *kept = part;
  }
  // 64 bytes a thread at a time, and as many on their way.
  template <bool BOTH>
  struct Loaded {
    static constexpr int U = BOTH ? 2 : 4;
    uint4 a[U], b[BOTH ? U : 1];
  };
  template <bool BOTH>
  __device__ __forceinline__ void load(Loaded<BOTH>& l, int x) const {
#pragma unroll
    for (int u = 0; u < l.U; ++u) {
      const int v = min(max(x + u * 32 * kVector<T>, first), last) - lead;
      l.a[u] = __ldg(reinterpret_cast<const uint4*>(p + v));
      if (BOTH) l.b[u] = __ldg(reinterpret_cast<const uint4*>(q + v));
    }
  }
  template <bool BOTH>
  __device__ __forceinline__ uint64_t count(const Loaded<BOTH>& l, int x) const {
    constexpr int N = kVector<T>;
    Counter sum;
    uint64_t rest = 0;
#pragma unroll
    for (int u = 0; u < l.U; ++u) {
      const int place = x + u * 32 * N;
      if (place >= first && place <= last) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = value(l.a[u], i, p);
          if constexpr (BOTH) sum.template add<false>(__fsub_rn(y, value(l.b[u], i, q)));
          else sum.template add<sizeof(T) == 2>(y);
        }
        if ((uint32_t)(without + lead - place) < (uint32_t)N) rest -= count_of(at(max(without, 0)));
      } else if (place + N > lead && place < vocab + lead) {  // the row's first or last values
        for (int i = 0; i < N; ++i) rest += count(place + i);
      }
    }
    return sum.count() + rest;
  }
  template <bool BOTH>
  __device__ __forceinline__ uint64_t sum_vectors(int begin, int tiles, uint64_t* kept, int lane) const {
    constexpr int STEP = Loaded<BOTH>::U * 32 * kVector<T>, STEPS = kTile<T> / STEP;
    static_assert(STEPS % 2 == 0, "two steps at a time");
    const int x0 = begin + lane * kVector<T>, end = x0 + tiles * kTile<T>;
    uint64_t total = 0;
    Loaded<BOTH> even, odd;
    load(even, x0);
    for (int x = x0, tile = 0; x < end; ++tile) {
      uint64_t part = 0;
#pragma unroll
      for (int y = 0; y < STEPS; y += 2, x += 2 * STEP) {
        load(odd, x + STEP);
        part += count(even, x);
        if (x + 2 * STEP < end) load(even, x + 2 * STEP);
        part += count(odd, x + STEP);
      }
      total += part;
      keep(part, kept + tile, lane);
    }
    return total;
  }
};

// PAGED: rows of the step without a page are left out.
template <typename T, bool PAGED>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM) verify_kernel(const Params a) {
  __shared__ uint64_t sums[MAX_BLOCKS * WARPS];  // of all warps of the cluster
  __shared__ uint64_t kept[WARPS][MAX_TILES];    // of the tiles of this block's warps
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
    int stored = 32;
    if constexpr (PAGED) {
      // Row r of the step (its last token, then the drafts) is in the cache iff the table has a page for it; what is
      // behind the first that is not, was computed without its key.
      const int len = a.context_lens[seq];
      if (len >= 0) {  // (idle places have no rows)
        const uint32_t t = (uint32_t)len + lane, page = t / (uint32_t)a.block_size;
        const int number = page < (uint32_t)a.table_width ? __ldg(a.block_tables + seq * a.table_stride + page) : -1;
        const bool there = number >= 0 && (int64_t)number * a.block_size + t % (uint32_t)a.block_size <= INT_MAX;
        const uint32_t none = ~__ballot_sync(0xffffffffu, there);
        stored = none ? __ffs(none) - 1 : 32;
      }
    }
    if (lane < a.num_drafts) {
      const int64_t d = !PAGED || lane + 1 < stored ? drafts[lane] : -1;
      live = d >= 0 && d < a.vocab;
      if (d >= a.vocab && rank == 0) record_error(VLC_DEV_ERR_TOKEN);
      const int64_t v = live ? d : 0;
      const float there = (float)__ldg(p0 + lane * a.p_row + v);
      const float draft = a.sampled ? (float)__ldg(q0 + lane * a.q_row + v) : 1.f;
      taken = live && (double)a.u[seq * a.u_stride + lane] * (double)draft < (double)there;
    }
    const uint32_t yes = __ballot_sync(0xffffffffu, taken), have = __ballot_sync(0xffffffffu, live);
    const int n = __ffs(~yes) == 0 ? 32 : __ffs(~yes) - 1;
    if (lane == 0) {
      s_taken = !PAGED || stored > 0 ? n : -1;
      s_refused = n < a.num_drafts && (have >> n & 1);
    }
  }
  __syncthreads();
  const int taken = s_taken;
  if (PAGED && taken < 0) {  // the sequence's own token is not in the cache: it waits for a page
    if (rank == 0 && threadIdx.x <= a.num_drafts) a.tokens[(int64_t)seq * (a.num_drafts + 1) + threadIdx.x] = -1;
    if (rank == 0 && threadIdx.x == 0) a.emitted[seq] = 0;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  const bool refused = s_refused != 0;
  Row<T> row;
  row.p = p0 + taken * a.p_row;
  row.both = refused && a.sampled;
  row.q = row.both ? q0 + taken * a.q_row : row.p;
  row.without = refused && !a.sampled ? (int)drafts[taken] : -1;
  row.vocab = a.vocab;
  row.settle();

  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // The second round, over p alone, is for a difference that has no positive value.
  for (int round = 0;; ++round) {
    const int me = rank * WARPS + warp;
    uint64_t sum = row.sum(me * a.tiles * kTile<T>, a.tiles, kept[warp], lane);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
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
      // ---- the tile in that run (every warp finds it), and the token in the tile: a thread takes a few values
      const uint64_t* const of = kept[where % WARPS];
      int tile = 0;
      for (int x0 = 0; x0 < a.tiles; x0 += 32) {
        uint64_t v = x0 + lane < a.tiles ? of[x0 + lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint64_t y = __shfl_up_sync(0xffffffffu, v, d);
          if (lane >= d) v += y;
        }
        const uint32_t low = ~__ballot_sync(0xffffffffu, before + v > goal);  // tiles that end at or before the goal
        const uint64_t last = __shfl_sync(0xffffffffu, v, 31 - __clz(low | 1));
        tile += __popc(low);
        if (low != 0) before += last;
        if (low != 0xffffffffu) break;
      }
      constexpr int each = kTile<T> / THREADS;
      const int w0 = (where * a.tiles + tile) * kTile<T> + threadIdx.x * each;
      uint64_t own = 0;
#pragma unroll
      for (int x = w0; x < w0 + each; ++x) own += row.count(x);
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
        int x = w0;
        while ((at += row.count(x)) <= goal && x + 1 < w0 + each) ++x;
        token = x - row.lead;
      }
    } else if (round == 0 && refused) {
      row.both = false;
      row.q = row.p;
      row.without = -1;
      row.settle();
      cluster_sync();  // every block has read its sums
      continue;
    } else {
      writer = rank == 0 && threadIdx.x == 0;  // no value is positive: no token
    }
    if (writer) {
      int64_t* const out = a.tokens + (int64_t)seq * (a.num_drafts + 1);
      for (int i = 0; i <= a.num_drafts; ++i) out[i] = i < taken ? drafts[i] : i == taken ? token : -1;
      a.emitted[seq] = taken + 1;
      if (a.context_lens && a.context_lens[seq] >= 0) a.context_lens[seq] += taken + 1;
    }
    return;
  }
}

template <typename T>
static int launch(const Params& a, int num_seqs, int blocks, cudaStream_t st) {
  const auto kernel = a.block_size > 0 ? verify_kernel<T, true> : verify_kernel<T, false>;
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
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}

}  // namespace verify
}  // namespace vlc

using namespace vlc;
using namespace vlc::verify;

// block_size 0: without block tables.
static int verify_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                         const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                         const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride, int vocab, int dtype,
                         const float* u, int64_t u_stride, const float* u_last, int64_t* tokens, int32_t* emitted,
                         int32_t* context_lens, const int32_t* block_tables, int64_t block_table_stride,
                         int block_table_width, int block_size, void* stream) {
  if (num_seqs < 0 || num_seqs > 65535 || num_drafts < 0 || vocab <= 0) return VLC_ERR_SHAPE;
  if (num_drafts > MAX_DRAFTS - 1 || vocab > MAX_VOCAB || dtype < 0 || dtype > 2) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0) return VLC_OK;
  if (!target_probs || !u_last || !tokens || !emitted || (num_drafts > 0 && (!drafts || !u))) return VLC_ERR_NULL;
  Params a;
  a.drafts = drafts;
  a.draft_stride = draft_stride;
  a.p = target_probs;
  a.sampled = num_drafts > 0 && draft_probs;
  a.q = a.sampled ? draft_probs : target_probs;
  a.p_seq = target_seq_stride;
  a.p_row = target_row_stride;
  a.q_seq = a.sampled ? draft_seq_stride : target_seq_stride;
  a.q_row = a.sampled ? draft_row_stride : target_row_stride;
  a.u = u;
  a.u_stride = u_stride;
  a.u_last = u_last;
  a.tokens = tokens;
  a.emitted = emitted;
  a.context_lens = context_lens;
  a.block_tables = block_tables;
  a.table_stride = block_table_stride;
  a.table_width = block_table_width;
  a.block_size = block_size;
  a.num_drafts = num_drafts;
  a.vocab = vocab;
  const int tile = dtype == 0 ? kTile<float> : kTile<__half>;
  static_assert(kTile<float> % THREADS == 0 && kTile<__half> == kTile<__nv_bfloat16>, "tiles are read again by a block");
  static_assert(MAX_TILES * WARPS * kTile<float> >= MAX_VOCAB + kVector<__half>, "one block can take a row");
  const int blocks = std::max(1, std::min(MAX_BLOCKS, vlc_num_sms() * BLOCKS_PER_SM / num_seqs));
  const int places = vocab + kVector<__half> - 1;  // and the lead
  a.tiles = (places + blocks * WARPS * tile - 1) / (blocks * WARPS * tile);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == 0 ? launch<float>(a, num_seqs, blocks, st)
         : dtype == 1 ? launch<__nv_bfloat16>(a, num_seqs, blocks, st)
                      : launch<__half>(a, num_seqs, blocks, st);
}

extern "C" int vlc_verify_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                                 const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                                 const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride, int vocab,
                                 int dtype, const float* u, int64_t u_stride, const float* u_last, int64_t* tokens,
                                 int32_t* emitted, int32_t* context_lens, void* stream) {
  return verify_drafts(drafts, draft_stride, num_seqs, num_drafts, target_probs, target_seq_stride, target_row_stride,
                       draft_probs, draft_seq_stride, draft_row_stride, vocab, dtype, u, u_stride, u_last, tokens, emitted,
                       context_lens, nullptr, 0, 0, 0, stream);
}

extern "C" int vlc_verify_stored_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                                        const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                                        const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride,
                                        int vocab, int dtype, const float* u, int64_t u_stride, const float* u_last,
                                        int64_t* tokens, int32_t* emitted, int32_t* context_lens,
                                        const int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                                        int block_size, void* stream) {
  if (block_table_width < 0 || block_size <= 0) return VLC_ERR_SHAPE;
  if (num_seqs > 0 && (!context_lens || (block_table_width > 0 && !block_tables))) return VLC_ERR_NULL;
  if (num_seqs > 1 && block_table_stride < block_table_width) return VLC_ERR_STRIDE;
  return verify_drafts(drafts, draft_stride, num_seqs, num_drafts, target_probs, target_seq_stride, target_row_stride,
                       draft_probs, draft_seq_stride, draft_row_stride, vocab, dtype, u, u_stride, u_last, tokens, emitted,
                       context_lens, block_tables, block_table_stride, block_table_width, block_size, stream);
}
