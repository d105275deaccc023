// The dense read-back of the 4-bit KV cache, and the move of reused image rows inside it.
#include <cmath>

#include "fp4.cuh"
#include "runtime.h"

namespace vlc {
namespace kv_fp4 {

using fp4::HD;
constexpr int TILE = 64;  // rows per block: divides every block size, so a tile lies in one page

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight values of a group (codes of four bytes, its scale in both halves) as packed fp32 pairs; exact.
__device__ __forceinline__ void values8(uint32_t codes, uint32_t scale2, uint64_t (&v)[4]) {
  uint32_t h[4];
  fp4::decode8(codes, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = hmul2(h[i], scale2);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    v[i] = f2_pack(f.x, f.y);
  }
}
__device__ __forceinline__ uint32_t both_halves(uint32_t scale_byte) {
  return fp4::scales2_f16((scale_byte & 0xff) * 0x0101u);
}

// ---------------------------------------------------------------------------
// Read-back: row cu_seqlens_k[b] + j of the output is key j of sequence b, for every head, in
// bf16 (exact: value = g * s * code).  Bound by the bf16 rows written (256 of the 328 bytes a row
// and head moves).  A block takes 64 rows of one head, K and V, of one layer: eight lanes a row, a
// scale's group of 16 dims a lane, so a warp reads four rows' 256 bytes of codes and a lane writes
// 32 bytes at once; all of a lane's loads (two rows of K and of V) are issued before the first use.
// Block x is given sequence b and tile i with x = cu[b] / 64 + b + i: those starts leave every
// sequence room for its ceil(len / 64) tiles, and a block past the last of them has nothing to do.
// 2556 rows of 2 heads in 36 layers (121 MB): 18 us.
// ---------------------------------------------------------------------------
struct GatherParams {
  const uint8_t* cache[2];
  int64_t layer_stride;
  const int32_t* block_tables;
  int64_t table_stride;
  int table_width;
  const int32_t* cu_seqlens_k;
  int num_seqs;
  int64_t total_k;
  int num_pages;
  int block_size;
  int num_kv_heads;
  float scale[2];
  __nv_bfloat16* out[2];
  int64_t out_row_stride, out_layer_stride;
  bool wide;  // outputs 32-byte aligned
};

__global__ void __launch_bounds__(256) gather_fp4_kernel(const __grid_constant__ GatherParams p) {
  pdl_launch_dependents();  // the attention that follows may start its prologue
  int lo = 0, hi = p.num_seqs - 1;  // largest b whose first block is <= blockIdx.x
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(p.cu_seqlens_k + mid) / TILE + mid <= (int)blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const int64_t begin = __ldg(p.cu_seqlens_k + lo);
  const int len = __ldg(p.cu_seqlens_k + lo + 1) - (int)begin;
  const int64_t j0 = ((int64_t)blockIdx.x - (begin / TILE + lo)) * TILE;
  if (j0 < 0 || j0 >= len) return;
  const int head = blockIdx.y, layer = blockIdx.z;
  const int table_index = (int)j0 / p.block_size;
  const int page = table_index < p.table_width ? __ldg(p.block_tables + lo * p.table_stride + table_index) : -1;
  const bool bad = page < 0 || page >= p.num_pages;
  if (bad && threadIdx.x == 0) record_error(VLC_DEV_ERR_BLOCK_RANGE);
  if ((begin < 0 || begin + len > p.total_k) && threadIdx.x == 0) record_error(VLC_DEV_ERR_LENGTH);
  const int64_t src = layer * p.layer_stride + fp4::head_offset(bad ? 0 : page, p.num_kv_heads, head, p.block_size);
  const int row0 = (int)j0 - table_index * p.block_size;
  const int c = threadIdx.x & 7;
  uint2 codes[2][2];
  uint32_t scales[2][2];
  bool live[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 32 + (threadIdx.x >> 3);
    live[i] = j0 + r < len && begin >= 0 && begin + j0 + r < p.total_k;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      codes[i][w] = make_uint2(0, 0);
      scales[i][w] = 0;
      if (live[i] && !bad) {
        codes[i][w] = __ldg(reinterpret_cast<const uint2*>(p.cache[w] + src + fp4::code_offset(row0 + r)) + c);
        scales[i][w] = __ldg(p.cache[w] + src + fp4::scale_offset(row0 + r, p.block_size) + c);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!live[i]) continue;
    const int64_t at = layer * p.out_layer_stride + (begin + j0 + i * 32 + (threadIdx.x >> 3)) * p.out_row_stride +
                       head * HD + 16 * c;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t s = both_halves(scales[i][w]);
      const uint64_t g = f2_pack(p.scale[w], p.scale[w]);
      uint64_t v[2][4];
      values8(codes[i][w].x, s, v[0]);
      values8(codes[i][w].y, s, v[1]);
      uint32_t u[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        float a, b;
        f2_unpack(f2_mul(v[x >> 2][x & 3], g), a, b);
        u[x] = pack_bf16x2(a, b);
      }
      if (p.wide) {
        st_global_v8(p.out[w] + at, u);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(p.out[w] + at);
        dst[0] = make_uint4(u[0], u[1], u[2], u[3]);
        dst[1] = make_uint4(u[4], u[5], u[6], u[7]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Move of reused rows: K row src_slots[i] rotated by the position delta (as the bf16 shift: pair j
// by inv_freq[j] * delta of its section's axis, cos/sin from the host) to row dst_slots[i], V row
// copied.  K is dequantised (exact), rotated in fp32 with every product and sum rounded by itself,
// rounded to bf16 as a bf16 cache would hold it, and quantised again.  A group of 16 pairs that
// the delta does not turn keeps its codes and scales: quantising again would move it.
// 288 bytes are read and written per row and head; at the copy rate that leaves an SM some 25
// instructions a byte-row lane, so the arithmetic counts as much: packed products, no division
// (fp4.cuh), a row's pages found once for all of a lane's heads.  Lanes: eight a row, eight pairs a
// lane (dims 8c.. and 64 + 8c..), four consecutive rows a warp, kHeads heads a lane, all loads
// first; rows of an image lie next to each other in their pages, so a warp's loads are runs of
// 256 bytes.  2556 rows of 2 heads in 36 layers (53 MB): 22 us, 8 us at the copy rate.
// ---------------------------------------------------------------------------
struct ShiftParams {
  uint8_t* k_cache;
  uint8_t* v_cache;
  int64_t layer_stride;
  int num_pages, block_size, num_kv_heads;
  const int32_t* src_slots;
  const int32_t* dst_slots;
  int num_rows;
  int block_shift;  // log2 of a block size that is a power of two, else -1
  uint32_t turned;  // bit m: group m of 16 pairs turns
  float cos[HD / 2], sin[HD / 2];
};

constexpr int kHeads = 2;

__global__ void __launch_bounds__(256, 4) shift_fp4_kernel(const __grid_constant__ ShiftParams p) {
  __shared__ __align__(8) float s_cos[HD / 2], s_sin[HD / 2];
  if (threadIdx.x < HD / 2) {
    s_cos[threadIdx.x] = p.cos[threadIdx.x];
    s_sin[threadIdx.x] = p.sin[threadIdx.x];
  }
  __syncthreads();
  const int head0 = blockIdx.y * kHeads, layer = blockIdx.z;
  const int c = threadIdx.x & 7;
  uint8_t* const k = p.k_cache + layer * p.layer_stride;
  uint8_t* const v = p.v_cache ? p.v_cache + layer * p.layer_stride : nullptr;
  const int r = blockIdx.x * 32 + (threadIdx.x >> 3);
  bool live = r < p.num_rows;
  int src = 0, dst = 0;
  if (live) {
    src = __ldg(p.src_slots + r);
    dst = p.dst_slots ? __ldg(p.dst_slots + r) : src;
    const uint32_t num_slots = (uint32_t)p.num_pages * (uint32_t)p.block_size;
    if ((uint32_t)src >= num_slots || (uint32_t)dst >= num_slots) {
      if (c == 0 && head0 == 0 && layer == 0) record_error(VLC_DEV_ERR_SLOT_RANGE);
      live = false;
    }
  }
  const int head_bytes = p.block_size * fp4::ROW_BYTES;
  const int src_page = p.block_shift >= 0 ? src >> p.block_shift : src / p.block_size;
  const int dst_page = p.block_shift >= 0 ? dst >> p.block_shift : dst / p.block_size;
  const int src_row = src - src_page * p.block_size, dst_row = dst - dst_page * p.block_size;
  const int64_t from = ((int64_t)src_page * p.num_kv_heads + head0) * head_bytes;
  const int64_t to = ((int64_t)dst_page * p.num_kv_heads + head0) * head_bytes;
  const int from_codes = fp4::code_offset(src_row), from_scales = fp4::scale_offset(src_row, p.block_size);
  const int to_codes = fp4::code_offset(dst_row), to_scales = fp4::scale_offset(dst_row, p.block_size);
  uint32_t lo[kHeads], hi[kHeads], s_lo[kHeads], s_hi[kHeads];
  uint2 vc[kHeads];
  uint8_t vs[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    lo[i] = hi[i] = s_lo[i] = s_hi[i] = 0;
    if (!live || head0 + i >= p.num_kv_heads) continue;
    const uint8_t* kf = k + from + i * head_bytes;
    lo[i] = reinterpret_cast<const uint32_t*>(kf + from_codes)[c];
    hi[i] = reinterpret_cast<const uint32_t*>(kf + from_codes)[8 + c];
    s_lo[i] = kf[from_scales + (c >> 1)];
    s_hi[i] = kf[from_scales + 4 + (c >> 1)];
    if (v) {
      const uint8_t* vf = v + from + i * head_bytes;
      vc[i] = reinterpret_cast<const uint2*>(vf + from_codes)[c];
      vs[i] = vf[from_scales + c];
    }
  }
  uint64_t cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = *reinterpret_cast<const uint64_t*>(s_cos + 8 * c + 2 * i);
    sn[i] = *reinterpret_cast<const uint64_t*>(s_sin + 8 * c + 2 * i);
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    uint64_t x1[4], x2[4];
    values8(lo[i], both_halves(s_lo[i]), x1);
    values8(hi[i], both_halves(s_hi[i]), x2);
    fp4::rotate8(x1, x2, cs, sn);
    const uint4 y1 = fp4::pack8(x1), y2 = fp4::pack8(x2);
    uint32_t m1 = fp4::absmax8(y1), m2 = fp4::absmax8(y2);
    m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
    m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
    if (!live || head0 + i >= p.num_kv_heads) continue;
    if ((p.turned >> (c >> 1)) & 1) {
      s_lo[i] = fp4::encode_scale(m1, 1.f);
      s_hi[i] = fp4::encode_scale(m2, 1.f);
      lo[i] = fp4::quantise8(y1, fp4::inverse_scale(s_lo[i], 1.f));
      hi[i] = fp4::quantise8(y2, fp4::inverse_scale(s_hi[i], 1.f));
    }
    uint8_t* kt = k + to + i * head_bytes;
    reinterpret_cast<uint32_t*>(kt + to_codes)[c] = lo[i];
    reinterpret_cast<uint32_t*>(kt + to_codes)[8 + c] = hi[i];
    if ((c & 1) == 0) kt[to_scales + (c >> 1)] = (uint8_t)s_lo[i];
    else kt[to_scales + 4 + (c >> 1)] = (uint8_t)s_hi[i];
    if (v) {
      uint8_t* vt = v + to + i * head_bytes;
      reinterpret_cast<uint2*>(vt + to_codes)[c] = vc[i];
      vt[to_scales + c] = vs[i];
    }
  }
}

// inv_freq[j] in fp32 as the rotary table's builder has it: 1 / (theta ** (float(2j) / float(128))).
static float inv_freq_f32(float theta, int j) { return 1.0f / powf(theta, (float)(2 * j) / (float)HD); }

}  // namespace kv_fp4
}  // namespace vlc

using namespace vlc;
using namespace vlc::kv_fp4;

extern "C" int vlc_gather_kvcache_fp4(const void* k_cache, const void* v_cache, int64_t layer_stride, int num_layers,
                                      int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                                      const int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                                      const int32_t* cu_seqlens_k, int num_seqs, int64_t total_k, float k_scale,
                                      float v_scale, void* k_out, void* v_out, int64_t out_row_stride,
                                      int64_t out_layer_stride, void* stream) {
  if (num_seqs < 0 || total_k < 0 || num_layers < 0 || block_table_width < 0 || num_kv_heads <= 0)
    return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % TILE != 0 || block_size > fp4::MAX_BLOCK) return VLC_ERR_UNSUPPORTED;
  if (!fp4::power_of_two(k_scale) || !fp4::power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0 || total_k == 0 || num_layers == 0) return VLC_OK;
  if (!k_cache || !v_cache || !block_tables || !cu_seqlens_k || !k_out || !v_out) return VLC_ERR_NULL;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size || num_kv_heads > 65535 || num_layers > 32767)
    return VLC_ERR_SHAPE;
  if (total_k > 0x7fffffff - (int64_t)TILE * ((int64_t)num_seqs + 1)) return VLC_ERR_SHAPE;
  const int64_t page_bytes = fp4::head_offset(1, num_kv_heads, 0, block_size);
  if (num_layers > 1 && (layer_stride < num_pages * page_bytes || layer_stride % 16)) return VLC_ERR_STRIDE;
  if (block_table_stride < block_table_width) return VLC_ERR_STRIDE;
  if (out_row_stride < (int64_t)num_kv_heads * HD || out_row_stride % 8) return VLC_ERR_STRIDE;
  if (num_layers > 1 && (out_layer_stride < total_k * out_row_stride || out_layer_stride % 8)) return VLC_ERR_STRIDE;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out)) return VLC_ERR_ALIGN;
  GatherParams p;
  p.cache[0] = (const uint8_t*)k_cache;
  p.cache[1] = (const uint8_t*)v_cache;
  p.layer_stride = layer_stride;
  p.block_tables = block_tables;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.cu_seqlens_k = cu_seqlens_k;
  p.num_seqs = num_seqs;
  p.total_k = total_k;
  p.num_pages = (int)num_pages;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.out[0] = (__nv_bfloat16*)k_out;
  p.out[1] = (__nv_bfloat16*)v_out;
  p.out_row_stride = out_row_stride;
  p.out_layer_stride = out_layer_stride;
  p.wide = reinterpret_cast<uintptr_t>(k_out) % 32 == 0 && reinterpret_cast<uintptr_t>(v_out) % 32 == 0 &&
           out_row_stride % 16 == 0 && out_layer_stride % 16 == 0;
  const dim3 grid((unsigned)(total_k / TILE + num_seqs), num_kv_heads, num_layers);
  gather_fp4_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  return launch_status();
}

extern "C" int vlc_mrope_shift_fp4(void* k_cache, void* v_cache, int64_t layer_stride, int num_layers,
                                   int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                                   const int32_t* src_slots, const int32_t* dst_slots, int num_rows,
                                   const int32_t* delta_thw, const int32_t* mrope_section, float rope_theta,
                                   void* stream) {
  if (num_rows < 0 || num_layers < 0 || num_kv_heads <= 0) return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % TILE != 0 || block_size > fp4::MAX_BLOCK) return VLC_ERR_UNSUPPORTED;
  if (num_rows == 0 || num_layers == 0) return VLC_OK;
  if (!k_cache || !src_slots || !delta_thw || !mrope_section) return VLC_ERR_NULL;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size || num_kv_heads > 65535 || num_layers > 65535)
    return VLC_ERR_SHAPE;
  if (mrope_section[0] < 0 || mrope_section[1] < 0 || mrope_section[2] < 0 ||
      (int64_t)mrope_section[0] + mrope_section[1] + mrope_section[2] != HD / 2)
    return VLC_ERR_SHAPE;
  const int64_t page_bytes = fp4::head_offset(1, num_kv_heads, 0, block_size);
  if (num_layers > 1 && (layer_stride < num_pages * page_bytes || layer_stride % 16)) return VLC_ERR_STRIDE;
  if (!aligned16(k_cache) || (v_cache && !aligned16(v_cache))) return VLC_ERR_ALIGN;
  ShiftParams p;
  p.k_cache = (uint8_t*)k_cache;
  p.v_cache = dst_slots ? (uint8_t*)v_cache : nullptr;  // in place: V rows stay
  p.layer_stride = layer_stride;
  p.num_pages = (int)num_pages;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.src_slots = src_slots;
  p.dst_slots = dst_slots;
  p.num_rows = num_rows;
  p.block_shift = -1;
  for (int s = 6; s < 31; ++s)
    if (block_size == 1 << s) p.block_shift = s;
  p.turned = 0;
  for (int j = 0; j < HD / 2; ++j) {
    const int axis = j < mrope_section[0] ? 0 : (j < mrope_section[0] + mrope_section[1] ? 1 : 2);
    const double a = (double)inv_freq_f32(rope_theta, j) * (double)delta_thw[axis];
    p.cos[j] = (float)cos(a);
    p.sin[j] = (float)sin(a);
    if (delta_thw[axis] != 0) p.turned |= 1u << (j / fp4::GROUP);
  }
  const dim3 grid((num_rows + 31) / 32, (num_kv_heads + kHeads - 1) / kHeads, num_layers);
  shift_fp4_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  return launch_status();
}
