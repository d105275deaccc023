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
// Bound by HBM: each row element is read once and written once.  Two kernels:
//  * rope_axes_kernel, few tokens: a warp takes one token and kIters groups of four consecutive
//    heads (query, key and value heads counted through), eight lanes a head, eight pairs a lane;
//    every load of the warp's groups is issued before the first use, the cos/sin values are loaded
//    once for them.  A decode step's tokens spread over as many SMs as there are slices.
//  * rope_stream_kernel, many tokens: the same slices taken by persistent warps.  Every lane keeps
//    the row pieces of its next two slices in flight into a place of its own in shared memory
//    (16-byte asynchronous copies: no registers, no barrier, only its own copies to wait for), and
//    loads the positions two slices and the table values one slice ahead.
//    10617 tokens of 28 + 4 + 4 heads into bf16 pages: 34.6 us against 41 with the first kernel
//    (196 MB, 31 us at the copy rate); whole tokens brought and taken by bulk copies into rings of
//    eight warps measured 41 too, each token waiting for the stores of the one before.
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
  int block_shift;  // log2 of a block size that is a power of two, else -1
  float k_inv_scale, v_inv_scale;
  int num_tokens, num_heads, num_kv_heads;
  int warps_per_token;
};

// cos and sin of pairs 8c .. 8c + 7 as packed pairs, from the table rows of the axes.
template <typename RowOf>
__device__ __forceinline__ void load_angles(const Params& p, int c, RowOf row_of, uint64_t (&cs)[4],
                                            uint64_t (&sn)[4]) {
  if (!p.mixed) {
    int x = 0;
#pragma unroll
    for (int i = 1; i < kMaxAxes; ++i)
      if (i < p.num_axes && 8 * c >= p.section_end[i - 1]) x = i;
    const float4* row = reinterpret_cast<const float4*>(row_of(x));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 u = row[2 * c + i], v = row[HALF / 4 + 2 * c + i];
      cs[2 * i] = f2_pack(u.x, u.y);
      cs[2 * i + 1] = f2_pack(u.z, u.w);
      sn[2 * i] = f2_pack(v.x, v.y);
      sn[2 * i + 1] = f2_pack(v.z, v.w);
    }
  } else {
    float u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = 8 * c + i;
      int x = 0;
#pragma unroll
      for (int k = 1; k < kMaxAxes; ++k)
        if (k < p.num_axes && j >= p.section_end[k - 1]) x = k;
      u[i] = row_of(x)[j];
      v[i] = row_of(x)[HALF + j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = f2_pack(u[2 * i], u[2 * i + 1]);
      sn[i] = f2_pack(v[2 * i], v[2 * i + 1]);
    }
  }
}

// Dims 8c .. (a) and 64 + 8c .. (b) of a head's row into its place in the 4-bit cache.  The groups
// are c / 2 and 4 + c / 2, each shared by two neighbouring lanes: all lanes of the warp come here,
// those without a row (dst null) too.
__device__ __forceinline__ void store_fp4(uint8_t* dst, const uint4& a, const uint4& b, float inv_g, int c, int row,
                                          int block_size) {
  uint32_t m1 = fp4::absmax8(a), m2 = fp4::absmax8(b);
  m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
  m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
  if (!dst) return;
  const uint32_t s1 = fp4::encode_scale(m1, inv_g), s2 = fp4::encode_scale(m2, inv_g);
  uint32_t* codes = reinterpret_cast<uint32_t*>(dst + fp4::code_offset(row));
  codes[c] = fp4::quantise8(a, fp4::inverse_scale(s1, inv_g));
  codes[8 + c] = fp4::quantise8(b, fp4::inverse_scale(s2, inv_g));
  uint8_t* scales = dst + fp4::scale_offset(row, block_size);
  if ((c & 1) == 0) scales[c >> 1] = (uint8_t)s1;
  else scales[4 + (c >> 1)] = (uint8_t)s2;
}

// Eight pairs of a head's row (a: dims 8c.., b: 64 + 8c..) to where they belong: turned when the
// head is a query or key head, and quantised for the 4-bit cache.  All lanes of a warp come here.
template <int SINK, bool ROTATE>
__device__ __forceinline__ void put_head(const Params& p, int64_t token, int head, int c, uint4 a, uint4 b,
                                         const uint64_t (&cs)[4], const uint64_t (&sn)[4], bool placed, bool stored,
                                         int slot) {
  const int q_heads = ROTATE ? p.num_heads : 0;
  const bool is_q = head < q_heads;
  const bool is_k = !is_q && head < q_heads + p.num_kv_heads;
  const bool is_v = !is_q && !is_k && head < q_heads + 2 * p.num_kv_heads;
  if (ROTATE && (is_q || is_k)) {
    uint64_t x1[4], x2[4];
    fp4::unpack8(a, x1);
    fp4::unpack8(b, x2);
    fp4::rotate8(x1, x2, cs, sn);
    a = fp4::pack8(x1);
    b = fp4::pack8(x2);
  }
  const int kv_head = head - q_heads - (is_v ? p.num_kv_heads : 0);
  const bool keep = stored && ((is_k && placed) || is_v);  // a row for the cache
  __nv_bfloat16* dst = nullptr;
  if (is_q) {
    if (placed) dst = p.q_out + token * p.q_out_stride + head * HD;
  } else if (SINK == kRows) {
    if (is_k && placed) dst = (__nv_bfloat16*)p.k_cache + token * p.k_out_stride + kv_head * HD;
  } else if (SINK == kBf16Cache) {
    if (keep) dst = (__nv_bfloat16*)(is_v ? p.v_cache : p.k_cache) + ((int64_t)slot * p.num_kv_heads + kv_head) * HD;
  }
  if (dst) {
    *reinterpret_cast<uint4*>(dst + 8 * c) = a;
    *reinterpret_cast<uint4*>(dst + HALF + 8 * c) = b;
  }
  if (SINK == kFp4Cache && __any_sync(0xffffffffu, is_k || is_v)) {
    uint8_t* row = nullptr;
    int at = 0;
    if (keep) {
      const int page = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block_size;
      at = slot - page * p.block_size;
      row = (uint8_t*)(is_v ? p.v_cache : p.k_cache) + fp4::head_offset(page, p.num_kv_heads, kv_head, p.block_size);
    }
    store_fp4(row, a, b, is_v ? p.v_inv_scale : p.k_inv_scale, c, at, p.block_size);
  }
}

// ROTATE false: no positions and no query heads (the plain 4-bit scatter).
template <int SINK, bool ROTATE>
__global__ void __launch_bounds__(kWarps * 32, 4) rope_axes_kernel(const __grid_constant__ Params p) {
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
  uint64_t cs[4], sn[4];
  bool placed = true;  // every axis' position is inside the table
  if (ROTATE) {
    int64_t pos[kMaxAxes];
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x) {
      pos[x] = x < p.num_axes ? __ldg(p.positions + x * p.axis_stride + token) : 0;
      placed = placed && pos[x] >= 0 && pos[x] < p.max_position;
    }
    if (!placed && lane == 0 && slice == 0) record_error(VLC_DEV_ERR_POSITION);
    load_angles(
        p, c, [&](int x) {
          int64_t at = pos[0];
#pragma unroll
          for (int i = 1; i < kMaxAxes; ++i)
            if (x == i) at = pos[i];
          return p.cos_sin + (placed ? at : 0) * HD;
        }, cs, sn);
  }
#pragma unroll
  for (int it = 0; it < kIters; ++it)
    put_head<SINK, ROTATE>(p, token, first + it * 4, c, a[it], b[it], cs, sn, placed, stored, slot);
}

constexpr int kStreamWarps = 20;   // one block an SM: 102 registers a thread
constexpr int kStreamStages = 3;   // slices of rows a lane has in shared memory
constexpr int kStreamBytes = kStreamWarps * kStreamStages * kIters * 2 * 32 * 16;

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <int SINK>
__global__ void __launch_bounds__(kStreamWarps * 32, 1) rope_stream_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint4 rows[];  // [warp][stage][2 it + half][lane]
  pdl_launch_dependents();
  const int lane = lane_id(), c = lane & 7;
  uint4* const mine = rows + (warp_id() * kStreamStages) * (kIters * 2 * 32) + lane;
  const int heads = p.num_heads + 2 * p.num_kv_heads;
  // Slices of a token: this warp's are every (blocks * warps)-th of all.
  struct Unit {
    int token, slice;
  };
  const int per_token = p.warps_per_token;
  const int stride = gridDim.x * kStreamWarps, stride_tokens = stride / per_token,
            stride_slices = stride - stride_tokens * per_token;
  auto after = [&](const Unit& u) {
    Unit n{u.token + stride_tokens, u.slice + stride_slices};
    if (n.slice >= per_token) {
      n.slice -= per_token;
      ++n.token;
    }
    return n;
  };
  auto copy_rows = [&](const Unit& u, int stage) {
    if (u.token < p.num_tokens) {
      const int first = u.slice * (kIters * 4) + (lane >> 3);
      const int64_t token = u.token;
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        const int head = first + it * 4;
        const __nv_bfloat16* src;
        if (head < p.num_heads) src = p.q + token * p.q_stride + head * HD;
        else if (head < p.num_heads + p.num_kv_heads) src = p.key + token * p.key_stride + (head - p.num_heads) * HD;
        else if (SINK != kRows && head < heads)
          src = p.value + token * p.value_stride + (head - p.num_heads - p.num_kv_heads) * HD;
        else continue;
        uint4* dst = mine + (stage * kIters + it) * 64;
        copy_async16(dst, src + 8 * c);
        copy_async16(dst + 32, src + HALF + 8 * c);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // A lane's eight pairs belong to one axis (sections that split them go to the other kernel); that
  // every axis' position is inside the table is seen by the lanes together.
  int own = 0;
#pragma unroll
  for (int x = 1; x < kMaxAxes; ++x)
    if (x < p.num_axes && 8 * c >= p.section_end[x - 1]) own = x;
  const int64_t* const own_positions = p.positions + own * p.axis_stride;
  const int64_t* const any_positions = p.positions + min(lane & 3, p.num_axes - 1) * p.axis_stride;
  int64_t own_pos, any_pos;  // of the slice after the next, and its slot
  int slot_after = -1;
  auto load_positions = [&](const Unit& u) {
    const int token = u.token < p.num_tokens ? u.token : 0;
    own_pos = __ldg(own_positions + token);
    any_pos = __ldg(any_positions + token);
    if (SINK != kRows) slot_after = __ldg(p.slot_mapping + token);
  };
  uint64_t cs_next[4], sn_next[4];  // of the next slice
  bool placed_next;
  int slot_next = -1;
  auto load_table = [&]() {
    placed_next = __all_sync(0xffffffffu, (uint64_t)any_pos < (uint64_t)p.max_position);
    slot_next = slot_after;
    const float4* row = reinterpret_cast<const float4*>(p.cos_sin + (placed_next ? own_pos : 0) * HD) + 2 * c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 u = __ldg(row + i), v = __ldg(row + HALF / 4 + i);
      cs_next[2 * i] = f2_pack(u.x, u.y);
      cs_next[2 * i + 1] = f2_pack(u.z, u.w);
      sn_next[2 * i] = f2_pack(v.x, v.y);
      sn_next[2 * i + 1] = f2_pack(v.z, v.w);
    }
  };

  const int start = warp_id() * gridDim.x + blockIdx.x;
  Unit u0{start / per_token, start % per_token}, u1 = after(u0), u2 = after(u1);
  static_assert(kStreamStages == 3, "rows are two slices ahead, as positions are");
  copy_rows(u0, 0);
  copy_rows(u1, 1);
  load_positions(u0);
  load_table();
  load_positions(u1);
  for (int stage = 0; u0.token < p.num_tokens; stage = stage == 2 ? 0 : stage + 1) {
    uint64_t cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = cs_next[i];
      sn[i] = sn_next[i];
    }
    const bool placed = placed_next;
    const int slot = slot_next;
    load_table();
    load_positions(u2);
    copy_rows(u2, stage == 0 ? 2 : stage - 1);
    asm volatile("cp.async.wait_group 2;" ::: "memory");

    const int token = u0.token;
    const int first = u0.slice * (kIters * 4) + (lane >> 3);
    const bool stored = slot >= 0 && slot < p.num_slots;
    if (lane == 0 && u0.slice == 0) {
      if (!placed) record_error(VLC_DEV_ERR_POSITION);
      if (SINK != kRows && !stored && slot != -1) record_error(VLC_DEV_ERR_SLOT_RANGE);
    }
#pragma unroll
    for (int it = 0; it < kIters; ++it) {
      const uint4* src = mine + (stage * kIters + it) * 64;
      put_head<SINK, true>(p, token, first + it * 4, c, src[0], src[32], cs, sn, placed, stored, slot);
    }
    u0 = u1;
    u1 = u2;
    u2 = after(u2);
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

template <int SINK, bool ROTATE>
static int launch(Params& p, cudaStream_t stream) {
  const int heads = (ROTATE ? p.num_heads : 0) + (SINK == kRows ? 1 : 2) * p.num_kv_heads;
  p.warps_per_token = (heads + 4 * kIters - 1) / (4 * kIters);
  if constexpr (ROTATE) {
    // Where every persistent warp gets four slices and more: below, filling and draining their copies
    // costs more than it saves (36 heads: 3001 tokens 14.0 against 12.7 us, 4500 tokens 17.0 against
    // 18.5; 20 heads: 4500 tokens 13.0 against 11.4).
    const int sms = vlc_num_sms();
    if ((int64_t)p.num_tokens * p.warps_per_token >= 4ll * sms * kStreamWarps && p.num_tokens <= 0x3fffffff &&
        !p.mixed) {
      static std::atomic<uint64_t> smem_set{0};
      if (ensure_dynamic_smem((const void*)rope_stream_kernel<SINK>, kStreamBytes, smem_set) != VLC_OK)
        return VLC_ERR_CUDA;
      rope_stream_kernel<SINK><<<sms, kStreamWarps * 32, kStreamBytes, stream>>>(p);
      return launch_status();
    }
  }
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
  if (block_size <= 0 || block_size % 64 != 0 || block_size > fp4::MAX_BLOCK) return VLC_ERR_UNSUPPORTED;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size) return VLC_ERR_SHAPE;
  if (!fp4::power_of_two(k_scale) || !fp4::power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
  p.block_size = block_size;
  p.block_shift = -1;
  for (int s = 6; s < 31; ++s)
    if (block_size == 1 << s) p.block_shift = s;
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
