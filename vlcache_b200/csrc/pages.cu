// Copies of whole cache pages in every layer, and the rewriting of block tables that goes with
// them: a request's pages are copied when it forks, moved when the pool is compacted.
#include <algorithm>

#include "common.cuh"
#include "runtime.h"

namespace vlc {
namespace pages {

// A plane is one layer's K or V: num_pages pages of page_bytes.  Grid (piece of a page, pair,
// plane), a block taking further pairs where there are more than a grid has room for; 16 KB a piece:
// four 16-byte loads a thread in flight, then the stores.  Bound by HBM: each byte is read once and
// written once.
constexpr int kThreads = 256;
constexpr int kLoads = 4;
constexpr int kPiece = kThreads * kLoads * 16;
constexpr int kMaxGridY = 65535;

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(uint8_t* __restrict__ base, int64_t plane_stride,
                                                              int64_t page_bytes, int64_t num_pages,
                                                              const int32_t* __restrict__ src_pages,
                                                              const int32_t* __restrict__ dst_pages, int num_pairs) {
  uint8_t* const plane = base + (int64_t)blockIdx.z * plane_stride;
  const int64_t first = (int64_t)blockIdx.x * kPiece + threadIdx.x * 16;
  for (int64_t pair = blockIdx.y; pair < num_pairs; pair += gridDim.y) {
    const int src = __ldg(src_pages + pair), dst = __ldg(dst_pages + pair);
    if (src == -1 && dst == -1) continue;  // padding of a fixed-size list
    if (src < 0 || dst < 0 || src >= num_pages || dst >= num_pages) {
      if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0) record_error(VLC_DEV_ERR_BLOCK_RANGE);
      continue;
    }
    if (src == dst) continue;
    const uint4* from = reinterpret_cast<const uint4*>(plane + src * page_bytes + first);
    uint4* to = reinterpret_cast<uint4*>(plane + dst * page_bytes + first);
    uint4 v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (first + (int64_t)i * kThreads * 16 < page_bytes) v[i] = from[i * kThreads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (first + (int64_t)i * kThreads * 16 < page_bytes) to[i * kThreads] = v[i];
  }
}

__global__ void __launch_bounds__(256) remap_tables_kernel(int32_t* tables, int64_t row_stride, int width,
                                                           int64_t entries, const int32_t* __restrict__ page_map,
                                                           int num_pages) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= entries) return;
  int32_t* at = tables + (i / width) * row_stride + i % width;
  const int page = *at;
  if (page == -1) return;
  if (page < 0 || page >= num_pages) {
    record_error(VLC_DEV_ERR_BLOCK_RANGE);
    return;
  }
  *at = __ldg(page_map + page);
}

}  // namespace pages
}  // namespace vlc

using namespace vlc;

extern "C" int vlc_copy_pages(void* base, int64_t plane_stride, int num_planes, int64_t page_bytes,
                              int64_t num_pages, const int32_t* src_pages, const int32_t* dst_pages, int num_pairs,
                              void* stream) {
  if (num_planes < 0 || num_pairs < 0 || page_bytes <= 0 || num_pages <= 0 || num_pages > 0x7fffffff)
    return VLC_ERR_SHAPE;
  if (num_planes == 0 || num_pairs == 0) return VLC_OK;
  if (!base || !src_pages || !dst_pages) return VLC_ERR_NULL;
  if (num_planes > 65535) return VLC_ERR_SHAPE;
  if (page_bytes % 16 || plane_stride % 16) return VLC_ERR_STRIDE;
  if (num_planes > 1 && plane_stride < page_bytes * num_pages) return VLC_ERR_STRIDE;
  if (!aligned16(base)) return VLC_ERR_ALIGN;
  const int64_t pieces = (page_bytes + pages::kPiece - 1) / pages::kPiece;
  if (pieces > 0x7fffffff) return VLC_ERR_SHAPE;
  const dim3 grid((unsigned)pieces, std::min(num_pairs, pages::kMaxGridY), num_planes);
  pages::copy_pages_kernel<<<grid, pages::kThreads, 0, (cudaStream_t)stream>>>(
      (uint8_t*)base, plane_stride, page_bytes, num_pages, src_pages, dst_pages, num_pairs);
  return launch_status();
}

extern "C" int vlc_remap_block_tables(int32_t* block_tables, int64_t row_stride, int num_rows, int width,
                                      const int32_t* page_map, int num_pages, void* stream) {
  if (num_rows < 0 || width < 0 || num_pages <= 0) return VLC_ERR_SHAPE;
  const int64_t entries = (int64_t)num_rows * width;
  if (entries == 0) return VLC_OK;
  if (!block_tables || !page_map) return VLC_ERR_NULL;
  if (row_stride < width) return VLC_ERR_STRIDE;
  const int64_t grid = (entries + 255) / 256;
  if (grid > 0x7fffffff) return VLC_ERR_SHAPE;
  pages::remap_tables_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(block_tables, row_stride, width,
                                                                            entries, page_map, num_pages);
  return launch_status();
}
