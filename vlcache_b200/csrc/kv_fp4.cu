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

// Eight values of a group (codes of four bytes, one scale) as floats; exact.
__device__ __forceinline__ void values8(uint32_t codes, uint32_t scale_byte, float (&v)[8]) {
  uint32_t h[4];
  fp4::decode8(codes, h);
  const uint32_t s = fp4::scales2_f16((scale_byte & 0xff) * 0x0101u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = hmul2(h[i], s);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// ---------------------------------------------------------------------------
// Read-back: row cu_seqlens_k[b] + j of the output is key j of sequence b, for every head, in
// bf16 (exact: value = g * s * code).  Bound by the bf16 rows written (256 of the 328 bytes a row
// and head moves).  A block takes 64 rows of one head, K or V, of one layer: sixteen lanes a row,
// eight dims a lane, so a warp reads two rows' 128 bytes of codes and writes two rows' 256-byte
// pieces; a lane has its four rows' loads in flight at once.
// Block x is given sequence b and tile i with x = cu[b] / 64 + b + i: those starts leave every
// sequence room for its ceil(len / 64) tiles, and a block past the last of them has nothing to do.
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
  const int head = blockIdx.y;
  const int layer = blockIdx.z >> 1, which = blockIdx.z & 1;
  const int table_index = (int)(j0 / p.block_size);
  const int page = table_index < p.table_width ? __ldg(p.block_tables + lo * p.table_stride + table_index) : -1;
  const bool bad = page < 0 || page >= p.num_pages;
  if (bad && threadIdx.x == 0) record_error(VLC_DEV_ERR_BLOCK_RANGE);
  if ((begin < 0 || begin + len > p.total_k) && threadIdx.x == 0) record_error(VLC_DEV_ERR_LENGTH);
  const uint8_t* src = p.cache[which] + layer * p.layer_stride +
                       fp4::head_offset(bad ? 0 : page, p.num_kv_heads, head, p.block_size);
  const int row0 = (int)(j0 % p.block_size);
  const int c = threadIdx.x & 15;
  constexpr int N = TILE / 16;
  uint32_t codes[N], scales[N];
  bool live[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = i * 16 + (threadIdx.x >> 4);
    live[i] = j0 + r < len && begin >= 0 && begin + j0 + r < p.total_k;
    codes[i] = scales[i] = 0;
    if (live[i] && !bad) {
      codes[i] = __ldg(reinterpret_cast<const uint32_t*>(src + fp4::code_offset(row0 + r)) + c);
      scales[i] = __ldg(src + fp4::scale_offset(row0 + r, p.block_size) + (c >> 1));
    }
  }
  const float g = p.scale[which];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!live[i]) continue;
    const int r = i * 16 + (threadIdx.x >> 4);
    float v[8];
    values8(codes[i], scales[i], v);
    uint4 u;
    u.x = pack_bf16x2(v[0] * g, v[1] * g);
    u.y = pack_bf16x2(v[2] * g, v[3] * g);
    u.z = pack_bf16x2(v[4] * g, v[5] * g);
    u.w = pack_bf16x2(v[6] * g, v[7] * g);
    __nv_bfloat16* dst = p.out[which] + layer * p.out_layer_stride + (begin + j0 + r) * p.out_row_stride + head * HD;
    *reinterpret_cast<uint4*>(dst + 8 * c) = u;
  }
}

// ---------------------------------------------------------------------------
// Move of reused rows: K row src_slots[i] rotated by the position delta (as the bf16 shift: pair j
// by inv_freq[j] * delta of its section's axis, cos/sin from the host) to row dst_slots[i], V row
// copied.  K is dequantised (exact), rotated in fp32 with every product and sum rounded by itself,
// rounded to bf16 as a bf16 cache would hold it, and quantised again.  A group of 16 pairs that
// the delta does not turn keeps its codes and scales: quantising again would move it.
// Bound by HBM (288 bytes read and written per row and head).  Lanes: eight a row, eight pairs a
// lane (dims 8c.. and 64 + 8c..), four consecutive rows a warp, kRows such rows a lane, all loads
// first; rows of an image lie next to each other in their pages, so a warp's loads are runs of
// 256 bytes.
// ---------------------------------------------------------------------------
struct ShiftParams {
  uint8_t* k_cache;
  uint8_t* v_cache;
  int64_t layer_stride;
  int num_pages, block_size, num_kv_heads;
  const int32_t* src_slots;
  const int32_t* dst_slots;
  int num_rows;
  uint32_t turned;  // bit m: group m of 16 pairs turns
  float cos[HD / 2], sin[HD / 2];
};

constexpr int kRows = 2;

__global__ void __launch_bounds__(256) shift_fp4_kernel(const __grid_constant__ ShiftParams p) {
  __shared__ float s_cos[HD / 2], s_sin[HD / 2];
  if (threadIdx.x < HD / 2) {
    s_cos[threadIdx.x] = p.cos[threadIdx.x];
    s_sin[threadIdx.x] = p.sin[threadIdx.x];
  }
  __syncthreads();
  const int head = blockIdx.y, layer = blockIdx.z;
  const int c = threadIdx.x & 7;
  uint8_t* const k = p.k_cache + layer * p.layer_stride;
  uint8_t* const v = p.v_cache ? p.v_cache + layer * p.layer_stride : nullptr;
  const int64_t num_slots = (int64_t)p.num_pages * p.block_size;
  int64_t from[kRows], to[kRows];  // the head's piece of the page
  int from_row[kRows], to_row[kRows];
  bool live[kRows];
  uint32_t lo[kRows], hi[kRows], s_lo[kRows], s_hi[kRows];
  uint2 vc[kRows];
  uint8_t vs[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = (blockIdx.x * kRows + i) * 32 + (threadIdx.x >> 3);
    live[i] = r < p.num_rows;
    if (!live[i]) continue;
    const int src = __ldg(p.src_slots + r);
    const int dst = p.dst_slots ? __ldg(p.dst_slots + r) : src;
    if (src < 0 || dst < 0 || src >= num_slots || dst >= num_slots) {
      if (c == 0 && head == 0 && layer == 0) record_error(VLC_DEV_ERR_SLOT_RANGE);
      live[i] = false;
      continue;
    }
    from_row[i] = src % p.block_size;
    to_row[i] = dst % p.block_size;
    from[i] = fp4::head_offset(src / p.block_size, p.num_kv_heads, head, p.block_size);
    to[i] = fp4::head_offset(dst / p.block_size, p.num_kv_heads, head, p.block_size);
    const uint8_t* kc = k + from[i] + fp4::code_offset(from_row[i]);
    lo[i] = reinterpret_cast<const uint32_t*>(kc)[c];
    hi[i] = reinterpret_cast<const uint32_t*>(kc)[8 + c];
    const uint8_t* ks = k + from[i] + fp4::scale_offset(from_row[i], p.block_size);
    s_lo[i] = ks[c >> 1];
    s_hi[i] = ks[4 + (c >> 1)];
    if (v) {
      vc[i] = reinterpret_cast<const uint2*>(v + from[i] + fp4::code_offset(from_row[i]))[c];
      vs[i] = v[from[i] + fp4::scale_offset(from_row[i], p.block_size) + c];
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float x1[8], x2[8];
    if (live[i]) {
      values8(lo[i], s_lo[i], x1);
      values8(hi[i], s_hi[i], x2);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x1[e] = x2[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float cs = s_cos[8 * c + e], sn = s_sin[8 * c + e];
      const float y1 = __fsub_rn(__fmul_rn(x1[e], cs), __fmul_rn(x2[e], sn));
      const float y2 = __fadd_rn(__fmul_rn(x2[e], cs), __fmul_rn(x1[e], sn));
      x1[e] = __bfloat162float(__float2bfloat16_rn(y1));
      x2[e] = __bfloat162float(__float2bfloat16_rn(y2));
    }
    uint32_t m1 = fp4::absmax8_bits(x1), m2 = fp4::absmax8_bits(x2);
    m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
    m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
    if (!live[i]) continue;
    if ((p.turned >> (c >> 1)) & 1) {
      s_lo[i] = fp4::encode_scale(__uint_as_float(m1));
      s_hi[i] = fp4::encode_scale(__uint_as_float(m2));
      lo[i] = fp4::quantise8(x1, s_lo[i]);
      hi[i] = fp4::quantise8(x2, s_hi[i]);
    }
    uint32_t* kc = reinterpret_cast<uint32_t*>(k + to[i] + fp4::code_offset(to_row[i]));
    kc[c] = lo[i];
    kc[8 + c] = hi[i];
    uint8_t* ks = k + to[i] + fp4::scale_offset(to_row[i], p.block_size);
    if ((c & 1) == 0) ks[c >> 1] = (uint8_t)s_lo[i];
    else ks[4 + (c >> 1)] = (uint8_t)s_hi[i];
    if (v) {
      reinterpret_cast<uint2*>(v + to[i] + fp4::code_offset(to_row[i]))[c] = vc[i];
      v[to[i] + fp4::scale_offset(to_row[i], p.block_size) + c] = vs[i];
    }
  }
}

// inv_freq[j] in fp32 as the rotary table's builder has it: 1 / (theta ** (float(2j) / float(128))).
static float inv_freq_f32(float theta, int j) { return 1.0f / powf(theta, (float)(2 * j) / (float)HD); }

static bool power_of_two(float g) {
  int e;
  return std::isfinite(g) && g > 0.f && std::frexp(g, &e) == 0.5f && e >= -63 && e <= 65;
}

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
  if (head_dim != HD || block_size <= 0 || block_size % TILE != 0) return VLC_ERR_UNSUPPORTED;
  if (!power_of_two(k_scale) || !power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
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
  const dim3 grid((unsigned)(total_k / TILE + num_seqs), num_kv_heads, 2 * num_layers);
  gather_fp4_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  return launch_status();
}

extern "C" int vlc_mrope_shift_fp4(void* k_cache, void* v_cache, int64_t layer_stride, int num_layers,
                                   int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                                   const int32_t* src_slots, const int32_t* dst_slots, int num_rows,
                                   const int32_t* delta_thw, const int32_t* mrope_section, float rope_theta,
                                   void* stream) {
  if (num_rows < 0 || num_layers < 0 || num_kv_heads <= 0) return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % TILE != 0) return VLC_ERR_UNSUPPORTED;
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
  p.turned = 0;
  for (int j = 0; j < HD / 2; ++j) {
    const int axis = j < mrope_section[0] ? 0 : (j < mrope_section[0] + mrope_section[1] ? 1 : 2);
    const double a = (double)inv_freq_f32(rope_theta, j) * (double)delta_thw[axis];
    p.cos[j] = (float)cos(a);
    p.sin[j] = (float)sin(a);
    if (delta_thw[axis] != 0) p.turned |= 1u << (j / fp4::GROUP);
  }
  const dim3 grid((num_rows + 32 * kRows - 1) / (32 * kRows), num_kv_heads, num_layers);
  shift_fp4_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  return launch_status();
}
