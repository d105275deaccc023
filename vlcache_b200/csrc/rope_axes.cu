// Rotary embedding of new rows at positions with several axes (time, height, width), fused with
// the scatter into the paged cache, in bf16 or in 4 bits; and the 4-bit scatter without rotation.
//
// Pair j of the rotate-half split, j in [0, 64), belongs to the axis a(j) whose section of the
// pairs holds it (sections follow each other, as mrope_section lists them).  With
// c = table[pos[a(j)][i]][j] and s = table[pos[a(j)][i]][64 + j]:
//   y[j] = x[j] c - x[64 + j] s,   y[64 + j] = x[64 + j] c + x[j] s,
// every fp32 product and sum rounded by itself and the result rounded to bf16, as the one-axis
// kernel of this library does, so that equal positions on all axes give its bits.  The 4-bit
// cache holds the quantised bf16 row: the same rows whether the rotation is fused or not.
//
// Bound by HBM: each row element is read once and written once.  A warp takes one token and
// `kIters` groups of four consecutive heads (query, key and value heads counted through): eight
// lanes a head, eight pairs a lane, so a group's loads are 128-byte pieces, and every load of the
// warp's groups is issued before the first use.  A lane's cos/sin values depend on the token and
// its pairs only: they are loaded once and serve all its heads.
#include <cmath>

#include "fp4.cuh"
#include "runtime.h"

namespace vlc {
namespace rope_axes {

constexpr int HD = 128;
constexpr int HALF = 64;
constexpr int kMaxAxes = 4;
constexpr int kWarps = 8;
constexpr int kIters = 3;

enum Sink { kRows = 0, kBf16Cache = 1, kFp4Cache = 2 };

struct Params {
  const int64_t* positions;  // [axes][axis_stride]
  int64_t axis_stride;
  int num_axes;
  int section_end[kMaxAxes];  // first pair after each axis' section
  bool mixed;                 // a section border inside eight pairs
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* q_out;
  int64_t q_out_stride;
  const __nv_bfloat16* key;
  int64_t key_stride;
  const __nv_bfloat16* value;
  int64_t value_stride;
  const float* cos_sin;
  int64_t max_position;
  void* k_cache;  // or the rotated key rows (kRows), with out_stride
  void* v_cache;
  int64_t k_out_stride;
  const int32_t* slot_mapping;
  int64_t num_slots;
  int block_size;
  float k_inv_scale, v_inv_scale;
  int num_tokens, num_heads, num_kv_heads;
  int warps_per_token;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 u;
  u.x = pack_bf16x2(f[0], f[1]);
  u.y = pack_bf16x2(f[2], f[3]);
  u.z = pack_bf16x2(f[4], f[5]);
  u.w = pack_bf16x2(f[6], f[7]);
  return u;
}

// ROTATE false: no positions and no query heads (the plain 4-bit scatter).
template <int SINK, bool ROTATE>
__global__ void __launch_bounds__(kWarps * 32) rope_axes_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();  // the attention that follows may start its prologue
  const int64_t warp = (int64_t)blockIdx.x * kWarps + warp_id();
  const int64_t token = warp / p.warps_per_token;
  if (token >= p.num_tokens) return;
  const int slice = (int)(warp - token * p.warps_per_token);
  const int lane = lane_id();
  const int c = lane & 7;  // pairs 8c .. 8c + 7
  const int q_heads = ROTATE ? p.num_heads : 0;
  const int all_heads = q_heads + 2 * p.num_kv_heads;
  const int first = slice * kIters * 4 + (lane >> 3);

  uint4 a[kIters], b[kIters];
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int head = first + it * 4;
    a[it] = b[it] = make_uint4(0, 0, 0, 0);
    if (head >= all_heads) continue;
    const __nv_bfloat16* src;
    if (head < q_heads) {
      src = p.q + token * p.q_stride + head * HD;
    } else if (head < q_heads + p.num_kv_heads) {
      src = p.key + token * p.key_stride + (head - q_heads) * HD;
    } else {
      if (SINK == kRows) continue;  // value rows stay where they are
      src = p.value + token * p.value_stride + (head - q_heads - p.num_kv_heads) * HD;
    }
    a[it] = *reinterpret_cast<const uint4*>(src + 8 * c);
    b[it] = *reinterpret_cast<const uint4*>(src + HALF + 8 * c);
  }
  int slot = 0;
  bool stored = true;  // the row has a place in the cache
  if (SINK != kRows) {
    slot = __ldg(p.slot_mapping + token);
    stored = slot >= 0 && slot < p.num_slots;
    if (!stored && slot != -1 && lane == 0 && slice == 0) record_error(VLC_DEV_ERR_SLOT_RANGE);
  }
  float cv[8], sv[8];
  bool placed = true;  // every axis' position is inside the table
  if (ROTATE) {
    int64_t pos[kMaxAxes];
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x) {
      pos[x] = x < p.num_axes ? __ldg(p.positions + x * p.axis_stride + token) : 0;
      placed = placed && pos[x] >= 0 && pos[x] < p.max_position;
    }
    if (!placed) {
      if (lane == 0 && slice == 0) record_error(VLC_DEV_ERR_POSITION);
#pragma unroll
      for (int i = 0; i < 8; ++i) cv[i] = sv[i] = 0.f;
    } else if (!p.mixed) {
      int64_t at = pos[0];
#pragma unroll
      for (int x = 1; x < kMaxAxes; ++x)
        if (x < p.num_axes && 8 * c >= p.section_end[x - 1]) at = pos[x];
      const float4* row = reinterpret_cast<const float4*>(p.cos_sin + at * HD);
      *reinterpret_cast<float4*>(&cv[0]) = __ldg(row + 2 * c);
      *reinterpret_cast<float4*>(&cv[4]) = __ldg(row + 2 * c + 1);
      *reinterpret_cast<float4*>(&sv[0]) = __ldg(row + HALF / 4 + 2 * c);
      *reinterpret_cast<float4*>(&sv[4]) = __ldg(row + HALF / 4 + 2 * c + 1);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = 8 * c + i;
        int64_t at = pos[0];
#pragma unroll
        for (int x = 1; x < kMaxAxes; ++x)
          if (x < p.num_axes && j >= p.section_end[x - 1]) at = pos[x];
        cv[i] = __ldg(p.cos_sin + at * HD + j);
        sv[i] = __ldg(p.cos_sin + at * HD + HALF + j);
      }
    }
  }
  const int64_t page = SINK == kFp4Cache ? slot / p.block_size : 0;
  const int row = SINK == kFp4Cache ? (int)(slot - page * p.block_size) : 0;

#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int head = first + it * 4;
    const bool is_q = head < q_heads;
    const bool is_k = !is_q && head < q_heads + p.num_kv_heads;
    const bool is_v = !is_q && !is_k && head < all_heads;
    float x1[8], x2[8];
    if (ROTATE && (is_q || is_k)) {
      unpack8(a[it], x1);
      unpack8(b[it], x2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y1 = __fsub_rn(__fmul_rn(x1[i], cv[i]), __fmul_rn(x2[i], sv[i]));
        const float y2 = __fadd_rn(__fmul_rn(x2[i], cv[i]), __fmul_rn(x1[i], sv[i]));
        x1[i] = y1;
        x2[i] = y2;
      }
      a[it] = pack8(x1);
      b[it] = pack8(x2);
    }
    if (is_q) {
      if (placed) {
        __nv_bfloat16* dst = p.q_out + token * p.q_out_stride + head * HD;
        *reinterpret_cast<uint4*>(dst + 8 * c) = a[it];
        *reinterpret_cast<uint4*>(dst + HALF + 8 * c) = b[it];
      }
    }
    if (SINK != kFp4Cache) {
      const int kv_head = head - q_heads - (is_v ? p.num_kv_heads : 0);
      __nv_bfloat16* dst = nullptr;
      if (SINK == kRows) {
        if (is_k && placed) dst = (__nv_bfloat16*)p.k_cache + token * p.k_out_stride + kv_head * HD;
      } else if (stored && ((is_k && placed) || is_v)) {
        dst = (__nv_bfloat16*)(is_v ? p.v_cache : p.k_cache) + ((int64_t)slot * p.num_kv_heads + kv_head) * HD;
      }
      if (dst) {
        *reinterpret_cast<uint4*>(dst + 8 * c) = a[it];
        *reinterpret_cast<uint4*>(dst + HALF + 8 * c) = b[it];
      }
    } else if (__any_sync(0xffffffffu, is_k || is_v)) {
      // Lane c holds dims 8c.. of group c / 2 and dims 64 + 8c.. of group 4 + c / 2: a group's
      // maximum is that of two neighbouring lanes.
      const float inv = is_v ? p.v_inv_scale : p.k_inv_scale;
      unpack8(a[it], x1);
      unpack8(b[it], x2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x1[i] *= inv;
        x2[i] *= inv;
      }
      uint32_t m1 = fp4::absmax8_bits(x1), m2 = fp4::absmax8_bits(x2);
      m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
      m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
      if (stored && ((is_k && placed) || is_v)) {
        const int kv_head = head - q_heads - (is_v ? p.num_kv_heads : 0);
        const uint32_t s1 = fp4::encode_scale(__uint_as_float(m1));
        const uint32_t s2 = fp4::encode_scale(__uint_as_float(m2));
        uint8_t* dst = (uint8_t*)(is_v ? p.v_cache : p.k_cache) +
                       fp4::head_offset(page, p.num_kv_heads, kv_head, p.block_size);
        uint32_t* codes = reinterpret_cast<uint32_t*>(dst + fp4::code_offset(row));
        codes[c] = fp4::quantise8(x1, s1);
        codes[8 + c] = fp4::quantise8(x2, s2);
        uint8_t* scales = dst + fp4::scale_offset(row, p.block_size);
        if ((c & 1) == 0) scales[c >> 1] = (uint8_t)s1;
        else scales[4 + (c >> 1)] = (uint8_t)s2;
      }
    }
  }
}

// The caller's sections as ends; false when they do not fit the 64 pairs.
static bool set_sections(Params& p, const int32_t* sections, int num_axes) {
  int end = 0;
  p.mixed = false;
  for (int x = 0; x < kMaxAxes; ++x) {
    if (x < num_axes) {
      if (sections[x] < 0 || sections[x] > HALF) return false;
      end += sections[x];
    }
    p.section_end[x] = end;
    if (end % 8) p.mixed = true;
  }
  p.num_axes = num_axes;
  return end == HALF;
}

static bool power_of_two(float g) {
  int e;
  return std::isfinite(g) && g > 0.f && std::frexp(g, &e) == 0.5f && e >= -63 && e <= 65;
}

template <int SINK, bool ROTATE>
static int launch(Params& p, cudaStream_t stream) {
  const int heads = (ROTATE ? p.num_heads : 0) + (SINK == kRows ? 1 : 2) * p.num_kv_heads;
  p.warps_per_token = (heads + 4 * kIters - 1) / (4 * kIters);
  const int64_t grid = ((int64_t)p.num_tokens * p.warps_per_token + kWarps - 1) / kWarps;
  if (grid > 0x7fffffff) return VLC_ERR_SHAPE;
  rope_axes_kernel<SINK, ROTATE><<<(unsigned)grid, kWarps * 32, 0, stream>>>(p);
  return launch_status();
}

// Shared checks of the rotating entry points.
static int rotate_args(Params& p, const int64_t* positions, int64_t axis_stride, int num_axes,
                       const int32_t* sections, const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride,
                       const void* key, int64_t key_stride, const float* cos_sin_cache, int64_t max_position,
                       int num_tokens, int num_heads, int num_kv_heads, int head_dim) {
  if (num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_position <= 0) return VLC_ERR_SHAPE;
  if (num_heads > 65536 || num_kv_heads > 65536) return VLC_ERR_SHAPE;
  if (head_dim != HD || num_axes < 1 || num_axes > kMaxAxes) return VLC_ERR_UNSUPPORTED;
  if (!sections) return VLC_ERR_NULL;
  if (!set_sections(p, sections, num_axes)) return VLC_ERR_SHAPE;
  if (num_tokens == 0) return VLC_OK;
  if (!positions || !q || !q_out || !key || !cos_sin_cache) return VLC_ERR_NULL;
  if (num_axes > 1 && axis_stride < num_tokens && axis_stride != 0) return VLC_ERR_STRIDE;
  if (q_stride % 8 || q_out_stride % 8 || key_stride % 8) return VLC_ERR_STRIDE;
  if (q_stride < (int64_t)num_heads * HD || q_out_stride < (int64_t)num_heads * HD ||
      key_stride < (int64_t)num_kv_heads * HD)
    return VLC_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(key) || !aligned16(cos_sin_cache)) return VLC_ERR_ALIGN;
  p.positions = positions;
  p.axis_stride = axis_stride;
  p.q = (const __nv_bfloat16*)q;
  p.q_stride = q_stride;
  p.q_out = (__nv_bfloat16*)q_out;
  p.q_out_stride = q_out_stride;
  p.key = (const __nv_bfloat16*)key;
  p.key_stride = key_stride;
  p.cos_sin = cos_sin_cache;
  p.max_position = max_position;
  p.num_tokens = num_tokens;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  return VLC_OK;
}

static int cache_args(Params& p, const void* value, int64_t value_stride, void* k_cache, void* v_cache,
                      const int32_t* slot_mapping, int64_t num_slots, int num_kv_heads) {
  if (!value || !k_cache || !v_cache || !slot_mapping) return VLC_ERR_NULL;
  if (num_slots <= 0 || num_slots > 0x7fffffff) return VLC_ERR_SHAPE;
  if (value_stride % 8 || value_stride < (int64_t)num_kv_heads * HD) return VLC_ERR_STRIDE;
  if (!aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache)) return VLC_ERR_ALIGN;
  p.value = (const __nv_bfloat16*)value;
  p.value_stride = value_stride;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.slot_mapping = slot_mapping;
  p.num_slots = num_slots;
  return VLC_OK;
}

static int fp4_args(Params& p, int64_t num_pages, int block_size, float k_scale, float v_scale) {
  if (block_size <= 0 || block_size % 64 != 0) return VLC_ERR_UNSUPPORTED;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size) return VLC_ERR_SHAPE;
  if (!power_of_two(k_scale) || !power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
  p.block_size = block_size;
  p.k_inv_scale = 1.f / k_scale;
  p.v_inv_scale = 1.f / v_scale;
  return VLC_OK;
}

}  // namespace rope_axes
}  // namespace vlc

using namespace vlc;
using namespace vlc::rope_axes;

extern "C" int vlc_mrope_store_kvcache(const int64_t* positions, int64_t axis_stride, int num_axes,
                                       const int32_t* sections, const void* q, int64_t q_stride, void* q_out,
                                       int64_t q_out_stride, const void* key, int64_t key_stride, const void* value,
                                       int64_t value_stride, const float* cos_sin_cache, int64_t max_position,
                                       void* k_cache, void* v_cache, const int32_t* slot_mapping, int64_t num_slots,
                                       void* k_out, int64_t k_out_stride, int num_tokens, int num_heads,
                                       int num_kv_heads, int head_dim, void* stream) {
  Params p{};
  int rc = rotate_args(p, positions, axis_stride, num_axes, sections, q, q_stride, q_out, q_out_stride, key,
                       key_stride, cos_sin_cache, max_position, num_tokens, num_heads, num_kv_heads, head_dim);
  if (rc != VLC_OK || num_tokens == 0) return rc;
  if (slot_mapping) {
    rc = cache_args(p, value, value_stride, k_cache, v_cache, slot_mapping, num_slots, num_kv_heads);
    return rc != VLC_OK ? rc : launch<kBf16Cache, true>(p, (cudaStream_t)stream);
  }
  if (!k_out) return VLC_ERR_NULL;
  if (k_out_stride % 8 || k_out_stride < (int64_t)num_kv_heads * HD) return VLC_ERR_STRIDE;
  if (!aligned16(k_out)) return VLC_ERR_ALIGN;
  p.k_cache = k_out;
  p.k_out_stride = k_out_stride;
  return launch<kRows, true>(p, (cudaStream_t)stream);
}

extern "C" int vlc_rope_store_kvcache_fp4(const int64_t* positions, int64_t axis_stride, int num_axes,
                                          const int32_t* sections, const void* q, int64_t q_stride, void* q_out,
                                          int64_t q_out_stride, const void* key, int64_t key_stride,
                                          const void* value, int64_t value_stride, const float* cos_sin_cache,
                                          int64_t max_position, void* k_cache, void* v_cache,
                                          const int32_t* slot_mapping, int64_t num_pages, int block_size,
                                          float k_scale, float v_scale, int num_tokens, int num_heads,
                                          int num_kv_heads, int head_dim, void* stream) {
  Params p{};
  int rc = rotate_args(p, positions, axis_stride, num_axes, sections, q, q_stride, q_out, q_out_stride, key,
                       key_stride, cos_sin_cache, max_position, num_tokens, num_heads, num_kv_heads, head_dim);
  if (rc == VLC_OK) rc = fp4_args(p, num_pages, block_size, k_scale, v_scale);
  if (rc != VLC_OK || num_tokens == 0) return rc;
  rc = cache_args(p, value, value_stride, k_cache, v_cache, slot_mapping, num_pages * block_size, num_kv_heads);
  return rc != VLC_OK ? rc : launch<kFp4Cache, true>(p, (cudaStream_t)stream);
}

extern "C" int vlc_store_kvcache_fp4(const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                                     void* k_cache, void* v_cache, const int32_t* slot_mapping, int64_t num_pages,
                                     int block_size, float k_scale, float v_scale, int num_tokens,
                                     int num_kv_heads, int head_dim, void* stream) {
  Params p{};
  if (num_tokens < 0 || num_kv_heads <= 0 || num_kv_heads > 65536) return VLC_ERR_SHAPE;
  if (head_dim != HD) return VLC_ERR_UNSUPPORTED;
  int rc = fp4_args(p, num_pages, block_size, k_scale, v_scale);
  if (rc != VLC_OK || num_tokens == 0) return rc;
  if (!key) return VLC_ERR_NULL;
  if (key_stride % 8 || key_stride < (int64_t)num_kv_heads * HD) return VLC_ERR_STRIDE;
  if (!aligned16(key)) return VLC_ERR_ALIGN;
  rc = cache_args(p, value, value_stride, k_cache, v_cache, slot_mapping, num_pages * block_size, num_kv_heads);
  if (rc != VLC_OK) return rc;
  p.key = (const __nv_bfloat16*)key;
  p.key_stride = key_stride;
  p.num_tokens = num_tokens;
  p.num_kv_heads = num_kv_heads;
  return launch<kFp4Cache, false>(p, (cudaStream_t)stream);
}
