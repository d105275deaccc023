// Block tables and slot maps of a step, built on the device from the sequences' lengths.
//
// Sequence i holds L_i tokens and takes n_i new ones at positions L_i .. L_i + n_i - 1.
//   * A table entry below 0 where one of them falls is filled from the end of the free list: the k-th
//     missing page of the batch (sequences in order, pages ascending) is free_pages[num_free - 1 - k].
//   * Pages that no later row sees under the window, p >= ceil(sinks / block) and
//     (p + 1) block <= L_i - window + 1, go back to the end of the list in the same order.
//   * Every new row gets its position and its slot, table[t / block] * block + t % block.
// The work is a few integer operations a row; what counts is latency.  So it is one launch: a cluster of
// blocks shares the sequences, counts, joins the counts through its blocks' shared memory, fills the
// tables and then writes the rows, with cluster barriers in between (pages are taken before any is
// given back into the same places).
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "runtime.h"

namespace vlc {
namespace step_meta {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCKS = 8;
constexpr int MAX_LEN = 1 << 30;

struct Params {
  const int32_t* context_lens;
  const int32_t* new_lens;
  int num_seqs;
  int32_t* block_tables;
  int64_t table_stride;
  int width, block_size, window, sinks;
  int32_t* free_pages;
  int free_capacity;
  int32_t* num_free;
  int64_t* positions;
  int32_t* slots;
  int total_rows;
  int32_t* cu_q;
  int32_t* cu_k;
  int32_t* new_context_lens;
};

// What a sequence's step is made of: its tokens, the pages of the new ones, and the pages behind the
// window (as ranges of table entries).
struct Seq {
  int len, fresh;
  int first, last;    // pages of the new rows, cut to the table
  int gone0, gone1;   // pages behind the window
};
__device__ __forceinline__ Seq seq_of(const Params& p, int i) {
  Seq s;
  s.len = __ldg(p.context_lens + i);
  s.fresh = max(0, __ldg(p.new_lens + i));
  if (s.len < 0) s.len = s.fresh = 0;  // an idle place of the batch
  if (s.len > MAX_LEN || s.fresh > MAX_LEN) {
    record_error(VLC_DEV_ERR_LENGTH);
    s.len = s.fresh = 0;
  }
  s.first = s.len / p.block_size;
  s.last = s.fresh > 0 ? min(p.width, (s.len + s.fresh - 1) / p.block_size + 1) : s.first;
  s.gone0 = (p.sinks + p.block_size - 1) / p.block_size;
  s.gone1 = p.window > 0 && s.len >= p.window ? min(p.width, (s.len - p.window + 1) / p.block_size) : 0;
  return s;
}

__device__ __forceinline__ int ld_cluster_i32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

enum : int { kNeed = 0, kGone = 1, kRows = 2, kKeys = 3, kCounts = 4 };

// Dynamic shared memory: [kCounts][per_block] counts of the block's sequences, then their exclusive sums.
__global__ void __launch_bounds__(THREADS) step_metadata_kernel(const Params p, int per_block) {
  extern __shared__ int counts[];
  __shared__ int totals[kCounts];
  const int rank = (int)cluster_ctarank(), blocks = gridDim.x;
  const int warp = warp_id(), lane = lane_id();
  const int seq0 = rank * per_block, mine = max(0, min(per_block, p.num_seqs - seq0));
  const int num_free = min(max(0, __ldg(p.num_free)), p.free_capacity);  // (written behind the last barrier)

  // ---- counts of each sequence, a warp each
  for (int i = warp; i < mine; i += WARPS) {
    const Seq s = seq_of(p, seq0 + i);
    const int32_t* table = p.block_tables + (seq0 + i) * p.table_stride;
    int need = 0, gone = 0;
    for (int x = s.first + lane; x < s.last; x += 32) need += table[x] < 0;
    for (int x = s.gone0 + lane; x < s.gone1; x += 32) gone += table[x] >= 0;
    need = __reduce_add_sync(0xffffffffu, need);
    gone = __reduce_add_sync(0xffffffffu, gone);
    if (lane == 0) {
      counts[kNeed * per_block + i] = need;
      counts[kGone * per_block + i] = gone;
      counts[kRows * per_block + i] = s.fresh;
      counts[kKeys * per_block + i] = s.len + s.fresh;
    }
  }
  __syncthreads();
  // ---- their sums, a warp each kind
  if (warp < kCounts) {
    int* const c = counts + warp * per_block;
    int before = 0;
    for (int base = 0; base < mine; base += 32) {
      const int v = base + lane < mine ? c[base + lane] : 0;
      int upto = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      if (base + lane < mine) c[base + lane] = before + upto - v;
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) totals[warp] = before;
  }
  cluster_sync();
  int base[kCounts] = {0, 0, 0, 0}, total[kCounts] = {0, 0, 0, 0};
  for (int b = 0; b < blocks; ++b) {
    const uint32_t at = mapa_shared(smem_u32(totals), b);
#pragma unroll
    for (int k = 0; k < kCounts; ++k) {
      const int v = ld_cluster_i32(at + 4 * k);
      if (b < rank) base[k] += v;
      total[k] += v;
    }
  }
  const int taken = min(total[kNeed], num_free);

  // ---- missing pages, lengths and their running sums
  for (int i = warp; i < mine; i += WARPS) {
    const Seq s = seq_of(p, seq0 + i);
    int32_t* table = p.block_tables + (seq0 + i) * p.table_stride;
    int nth = base[kNeed] + counts[kNeed * per_block + i];
    for (int x0 = s.first; x0 < s.last; x0 += 32) {
      const int x = x0 + lane;
      const bool missing = x < s.last && table[x] < 0;
      const uint32_t who = __ballot_sync(0xffffffffu, missing);
      if (missing) {
        const int k = nth + __popc(who & ((1u << lane) - 1));
        if (k < num_free) table[x] = p.free_pages[num_free - 1 - k];
      }
      nth += __popc(who);
    }
    if (lane == 0) {
      const int q = base[kRows] + counts[kRows * per_block + i], k = base[kKeys] + counts[kKeys * per_block + i];
      p.cu_q[seq0 + i] = q;
      p.cu_k[seq0 + i] = k;
      p.new_context_lens[seq0 + i] = s.len + s.fresh;
      if (s.fresh > 0 && (s.len + s.fresh - 1) / p.block_size >= p.width) record_error(VLC_DEV_ERR_BLOCK_RANGE);
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.cu_q[p.num_seqs] = total[kRows];
    p.cu_k[p.num_seqs] = total[kKeys];
    if (total[kNeed] > num_free || num_free - taken + total[kGone] > p.free_capacity) record_error(VLC_DEV_ERR_PAGES);
    if (total[kRows] > p.total_rows) record_error(VLC_DEV_ERR_LENGTH);
  }
  cluster_sync();  // every page is taken, every table filled

  // ---- pages behind the window
  if (p.window > 0) {
    for (int i = warp; i < mine; i += WARPS) {
      const Seq s = seq_of(p, seq0 + i);
      int32_t* table = p.block_tables + (seq0 + i) * p.table_stride;
      int nth = num_free - taken + base[kGone] + counts[kGone * per_block + i];
      for (int x0 = s.gone0; x0 < s.gone1; x0 += 32) {
        const int x = x0 + lane;
        const int page = x < s.gone1 ? table[x] : -1;
        const uint32_t who = __ballot_sync(0xffffffffu, page >= 0);
        if (page >= 0) {
          const int k = nth + __popc(who & ((1u << lane) - 1));
          if (k < p.free_capacity) p.free_pages[k] = page;
          table[x] = -1;
        }
        nth += __popc(who);
      }
    }
  }
  if (rank == 0 && threadIdx.x == 0) *p.num_free = min(num_free - taken + total[kGone], p.free_capacity);

  // ---- rows: a warp takes a run of them
  const int rows = min(total[kRows], p.total_rows);
  const int warps = blocks * WARPS;
  const int run = ((p.total_rows + warps - 1) / warps + 31) / 32 * 32;
  const int64_t r0 = (int64_t)(rank * WARPS + warp) * run;
  int seq = 0, begin = 0, end = 0, len = 0;
  if (r0 < rows) {  // the last sequence that begins at or before the lane's first row
    const int row = min((int)r0 + lane, rows - 1);
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu_q[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    seq = lo;
    begin = p.cu_q[seq];
    end = p.cu_q[seq + 1];
    len = p.new_context_lens[seq] - (end - begin);
  }
  for (int64_t r = r0 + lane; r < r0 + run && r < p.total_rows; r += 32) {
    int64_t position = 0;
    int32_t slot = -1;
    if (r < rows) {
      while (r >= end && seq + 1 < p.num_seqs) {
        begin = end;
        end = p.cu_q[++seq + 1];
        len = p.new_context_lens[seq] - (end - begin);
      }
      const int t = len + (int)(r - begin);
      const int page = t / p.block_size;
      position = t;
      const int number = (uint32_t)page < (uint32_t)p.width ? p.block_tables[seq * p.table_stride + page] : -1;
      const int64_t at = (int64_t)number * p.block_size + (t - page * p.block_size);
      if (number >= 0 && at <= INT_MAX) slot = (int32_t)at;
      else if (number >= 0) record_error(VLC_DEV_ERR_SLOT_RANGE);
    }
    p.positions[r] = position;
    p.slots[r] = slot;
  }
}

}  // namespace step_meta
}  // namespace vlc

using namespace vlc;
using namespace vlc::step_meta;

extern "C" int vlc_step_metadata(const int32_t* context_lens, const int32_t* new_lens, int num_seqs,
                                 int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                                 int block_size, int window, int sinks, int32_t* free_pages, int free_capacity,
                                 int32_t* num_free, int64_t* positions, int32_t* slot_mapping, int total_rows,
                                 int32_t* cu_seqlens_q, int32_t* cu_seqlens_k, int32_t* new_context_lens,
                                 void* stream) {
  if (num_seqs < 0 || num_seqs > 65535 || block_table_width < 0 || block_size <= 0 || window < 0 || sinks < 0 ||
      window > MAX_LEN || sinks > MAX_LEN || free_capacity < 0 || total_rows < 0 || total_rows > MAX_LEN)
    return VLC_ERR_SHAPE;
  if (!num_free || !cu_seqlens_q || !cu_seqlens_k) return VLC_ERR_NULL;
  if (num_seqs > 0 && (!context_lens || !new_lens || !new_context_lens)) return VLC_ERR_NULL;
  if (num_seqs > 0 && block_table_width > 0 && !block_tables) return VLC_ERR_NULL;
  if ((free_capacity > 0 && !free_pages) || (total_rows > 0 && (!positions || !slot_mapping))) return VLC_ERR_NULL;
  if ((int64_t)num_seqs * block_table_width > INT_MAX) return VLC_ERR_SHAPE;  // (pages are counted in 32 bits)
  if (num_seqs > 1 && block_table_stride < block_table_width) return VLC_ERR_STRIDE;
  Params p;
  p.context_lens = context_lens;
  p.new_lens = new_lens;
  p.num_seqs = num_seqs;
  p.block_tables = block_tables;
  p.table_stride = block_table_stride;
  p.width = block_table_width;
  p.block_size = block_size;
  p.window = window;
  p.sinks = sinks;
  p.free_pages = free_pages;
  p.free_capacity = free_capacity;
  p.num_free = num_free;
  p.positions = positions;
  p.slots = slot_mapping;
  p.total_rows = total_rows;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.new_context_lens = new_context_lens;
  // A block a sequence for each of its warps, or for as many rows as its threads write at once.
  int blocks = 1;
  while (blocks < MAX_BLOCKS && (num_seqs > blocks * WARPS || total_rows > blocks * THREADS)) blocks *= 2;
  const int per_block = (num_seqs + blocks - 1) / blocks;
  const int bytes = kCounts * per_block * (int)sizeof(int);
  static std::atomic<uint64_t> smem{0};
  if (ensure_dynamic_smem((const void*)step_metadata_kernel, kCounts * ((65535 + MAX_BLOCKS - 1) / MAX_BLOCKS) * 4,
                          smem) != VLC_OK)
    return VLC_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, step_metadata_kernel, (const Params)p, per_block) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}
