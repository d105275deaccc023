// Block tables and slot maps of a step, built on the device from the sequences' lengths.
//
// Sequence i holds L_i tokens and takes n_i new ones at positions L_i .. L_i + n_i - 1.
//   * A table entry below 0 where one of them falls is filled from the end of the free list: the k-th
//     missing page of the batch (sequences in order, pages ascending) is free_pages[num_free - 1 - k].
//   * Pages that no later row sees under the window, p >= ceil(sinks / block) and
//     (p + 1) block <= L_i - window + 1, go back to the end of the list in the same order.
//   * Every new row gets its position and its slot, table[t / block] * block + t % block.
// The work is a few integer operations a row; what counts is latency.  So it is one launch: a cluster of
// blocks shares the sequences, counts, joins the counts through its blocks' shared memory and fills the
// tables, with a cluster barrier before pages go back (into the places that pages are taken from).  Rows of
// a few tokens a sequence are written by the warp that has just filled its table; where a sequence takes
// more, all warps share all rows behind a barrier, four a lane.  Many rows (whole prompts) are written by
// a second launch over all SMs, a programmatic dependent: 64 prompts of up to 10,617 tokens (295,000 rows) in
// 8.5 us, by the cluster alone in 24.  What bounds it is the chain of dependent loads and barriers (lengths, table
// entries, sums, pages, slots): 4.9 us for 8 sequences, 9.6 for 256 of five tokens under a window.
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
constexpr int MANY_ROWS = 16384;  // of a step, for the second launch
constexpr int FEW_ROWS = 64;  // of a sequence, that its warp writes by itself

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
  bool rows_apart;  // rows are written by the second launch
};

// What a sequence's step is made of: its tokens, the pages of the new ones, and the pages behind the
// window (as ranges of table entries).
struct Seq {
  int len, fresh;     // tokens it has, and that it takes
  int rows;           // of the step: also an idle place's
  int first, last;    // pages of the new rows, cut to the table
  int gone0, gone1;   // pages behind the window
};
__device__ __forceinline__ Seq seq_of(const Params& p, int2 lens) {  // context and new lengths
  Seq s;
  s.len = lens.x;
  s.rows = s.fresh = max(0, lens.y);
  if (s.len > MAX_LEN || s.fresh > MAX_LEN) {
    record_error(VLC_DEV_ERR_LENGTH);
    s.len = s.rows = s.fresh = 0;
  }
  if (s.len < 0) s.len = s.fresh = 0;  // an idle place of the batch
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

enum : int { kNeed = 0, kGone = 1, kRows = 2, kKeys = 3, kMany = 4, kCounts = 5 };  // kMany: sequences of many rows

// Slot of position t, -1 where the table has no page there.
__device__ __forceinline__ int32_t slot_at(const Params& p, int number, int t, int page) {
  const int64_t at = (int64_t)number * p.block_size + (t - page * p.block_size);
  if (number >= 0 && at > INT_MAX) record_error(VLC_DEV_ERR_SLOT_RANGE);
  return number >= 0 && at <= INT_MAX ? (int32_t)at : -1;
}

// Positions and slots of rows, from the sums and the tables that are in memory.
struct Rows {
  const Params& p;
  const int rows;  // of all sequences
  int seq = -1, begin = 0, end = 0, len = 0;
  const bool aligned;
  __device__ __forceinline__ Rows(const Params& p, int rows)
      : p(p), rows(rows),
        aligned((reinterpret_cast<uintptr_t>(p.positions) % 32 | reinterpret_cast<uintptr_t>(p.slots) % 16) == 0) {}
  __device__ __forceinline__ void take(int s) {
    seq = s;
    begin = p.cu_q[s];
    end = p.cu_q[s + 1];
    len = p.new_context_lens[s] - (end - begin);
  }
  // Rows r .. r + n - 1 (n up to 4; r a multiple of 4, and not below that of the call before).
  __device__ __forceinline__ void write(int64_t r, int n) {
    if (r < rows && seq < 0) {  // the last sequence that begins at or before the first row
      int lo = 0, hi = p.num_seqs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu_q[mid] <= r) lo = mid;
        else hi = mid - 1;
      }
      take(lo);
    }
    int page = -1, first = 0, number = -1;  // of the row before, and the page's first position
    int32_t position[4] = {0, 0, 0, 0}, slot[4] = {-1, -1, -1, -1};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (r + x >= rows) continue;
      if (r + x >= end) {
        while (r + x >= end && seq + 1 < p.num_seqs) take(seq + 1);
        page = -1;
      }
      const int t = len + (int)(r + x - begin);
      if (t < 0) continue;  // an idle place's
      if (page < 0 || t - first >= p.block_size) {
        page = t / p.block_size;
        first = page * p.block_size;
        number = (uint32_t)page < (uint32_t)p.width ? p.block_tables[seq * p.table_stride + page] : -1;
      }
      position[x] = t;
      slot[x] = slot_at(p, number, t, page);
    }
    if (n == 4 && aligned) {
      const uint32_t wide[8] = {(uint32_t)position[0], 0, (uint32_t)position[1], 0,
                                (uint32_t)position[2], 0, (uint32_t)position[3], 0};
      st_global_v8(p.positions + r, wide);
      *reinterpret_cast<int4*>(p.slots + r) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (x >= n) continue;
        p.positions[r + x] = position[x];
        p.slots[r + x] = slot[x];
      }
    }
  }
};

// Dynamic shared memory: the block's sequences' lengths, [kCounts][per_block] counts of them, then their exclusive sums.
__global__ void __launch_bounds__(THREADS) step_metadata_kernel(const Params p, int per_block) {
  extern __shared__ int2 lens[];
  int* const counts = reinterpret_cast<int*>(lens + per_block);
  __shared__ int totals[kCounts];
  if (p.rows_apart) pdl_launch_dependents();
  const int rank = (int)cluster_ctarank(), blocks = gridDim.x;
  const int warp = warp_id(), lane = lane_id();
  const int seq0 = rank * per_block, mine = max(0, min(per_block, p.num_seqs - seq0));
  const int num_free = min(max(0, __ldg(p.num_free)), p.free_capacity);  // (written behind the last barrier)

  for (int i = threadIdx.x; i < mine; i += THREADS)
    lens[i] = make_int2(__ldg(p.context_lens + seq0 + i), __ldg(p.new_lens + seq0 + i));
  __syncthreads();
  // ---- counts of each sequence, a warp each
  for (int i = warp; i < mine; i += WARPS) {
    const Seq s = seq_of(p, lens[i]);
    const int32_t* table = p.block_tables + (seq0 + i) * p.table_stride;
    int need = 0, gone = 0;
    for (int x = s.first + lane; x < s.last; x += 32) need += table[x] < 0;
    for (int x = s.gone0 + lane; x < s.gone1; x += 32) gone += table[x] >= 0;
    need = __reduce_add_sync(0xffffffffu, need);
    gone = __reduce_add_sync(0xffffffffu, gone);
    if (lane == 0) {
      counts[kNeed * per_block + i] = need;
      counts[kGone * per_block + i] = gone;
      counts[kRows * per_block + i] = s.rows;
      counts[kKeys * per_block + i] = s.len + s.fresh;
      counts[kMany * per_block + i] = s.rows > FEW_ROWS;
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
  int base[kCounts], total[kCounts];
  {  // lane b: block b's
    const uint32_t at = mapa_shared(smem_u32(totals), min(lane, blocks - 1));
    int v[kCounts];
#pragma unroll
    for (int k = 0; k < kCounts; ++k) v[k] = ld_cluster_i32(at + 4 * k);
#pragma unroll
    for (int k = 0; k < kCounts; ++k) {
      total[k] = (int)__reduce_add_sync(0xffffffffu, (unsigned)(lane < blocks ? v[k] : 0));
      base[k] = (int)__reduce_add_sync(0xffffffffu, (unsigned)(lane < rank ? v[k] : 0));
    }
  }
  const int taken = min(total[kNeed], num_free);
  const bool shared_rows = p.rows_apart || total[kMany] > 0;

  // ---- missing pages, lengths and their running sums
  for (int i = warp; i < mine; i += WARPS) {
    const Seq s = seq_of(p, lens[i]);
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
    const int q = base[kRows] + counts[kRows * per_block + i];
    if (!shared_rows) {
      __syncwarp();  // (the lanes' entries are there)
      for (int r = lane; r < s.rows; r += 32) {
        const int t = s.len + r, page = t / p.block_size;
        const bool idle = s.fresh == 0;
        if (q + r < p.total_rows) {
          p.positions[q + r] = idle ? 0 : t;
          p.slots[q + r] = slot_at(p, !idle && page < p.width ? table[page] : -1, t, page);
        }
      }
    }
    if (lane == 0) {
      const int k = base[kKeys] + counts[kKeys * per_block + i];
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
  // Every page is taken, every table filled; and the sums of this block have been read.
  cluster_sync();

  // ---- pages behind the window
  if (p.window > 0) {
    for (int i = warp; i < mine; i += WARPS) {
      const Seq s = seq_of(p, lens[i]);
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

  // ---- rows behind the last, and all rows where a sequence has many: a warp takes a run of them, a lane four at once
  if (p.rows_apart) return;
  const int rows = min(max(total[kRows], 0), p.total_rows);
  const int from = shared_rows ? 0 : rows / 4 * 4, warps = blocks * WARPS;
  const int run = ((p.total_rows - from + warps - 1) / warps + 127) / 128 * 128;
  const int64_t r0 = from + (int64_t)(rank * WARPS + warp) * run, r1 = min(r0 + run, (int64_t)p.total_rows);
  Rows at(p, rows);
  for (int64_t r = r0 + lane * 4; r < r1; r += 128) at.write(r, (int)min(r1 - r, (int64_t)4));
}

// Many rows: a thread four of them.
__global__ void __launch_bounds__(THREADS) step_rows_kernel(const Params p) {
  pdl_wait();  // the tables and sums are the launch before's
  const int64_t r = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 4;
  if (r >= p.total_rows) return;
  Rows at(p, min(max(p.cu_q[p.num_seqs], 0), p.total_rows));
  at.write(r, (int)min(p.total_rows - r, (int64_t)4));
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
  p.rows_apart = total_rows > MANY_ROWS;
  // A block a sequence for each of its warps, or for as many rows as its threads write at once.
  int blocks = 1;
  while (blocks < MAX_BLOCKS && (num_seqs > blocks * WARPS || (!p.rows_apart && total_rows > blocks * THREADS))) blocks *= 2;
  const int per_block = (num_seqs + blocks - 1) / blocks;
  const int bytes = (kCounts + 2) * per_block * (int)sizeof(int);
  static std::atomic<uint64_t> smem{0};
  if (ensure_dynamic_smem((const void*)step_metadata_kernel, (kCounts + 2) * ((65535 + MAX_BLOCKS - 1) / MAX_BLOCKS) * 4,
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
  if (!p.rows_apart) return VLC_OK;
  cfg.gridDim = dim3((unsigned)(((int64_t)total_rows + 4 * THREADS - 1) / (4 * THREADS)));
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  if (cudaLaunchKernelEx(&cfg, step_rows_kernel, (const Params)p) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}
