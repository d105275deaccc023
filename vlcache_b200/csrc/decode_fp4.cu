// Paged decode attention over the 4-bit KV cache (one query token per sequence), sm_100a.
//
//   o[h] = sum_j softmax_j(scale * g_k * q[h] . K[j]) * g_v * V[j],   K, V = s * code per group.
//
// The floor is HBM: 72 bytes per key and head for K and V each.  At that rate an SM has to take in
// 4 times the keys a second of the bf16 decode, so the work per element counts:
//   * K and V are the A operands (16 rows) of m16n8k16 f16 MMAs and the query heads of the KV head
//     the 8 columns: S^T = K Q^T and O^T = V^T P^T.  A KV head of up to 8 query heads then wastes
//     no rows, and an MMA consumes 256 cache elements, twice what the transposed products would.
//   * The contraction order is free, so a lane takes its A fragments from contiguous bytes: of a
//     key's 64 code bytes lane (r, t) loads bytes 16t..16t+15 (one 16-byte load for all eight
//     k-steps, Q permuted alike); of a key's V codes the 8 bytes of scale group r (a fragment's row
//     r is dim 16r + 2i of m-tile i, row r + 8 dim 16r + 2i + 1).
//   * e2m1 pairs convert to f16 pairs in one instruction and one multiplication by the scale makes
//     the exact value; V pairs hold the same dim of two keys, made by exchanging nibbles first.
//   * P^T in the layout of a B operand is S^T's accumulator transposed: one movmatrix an 8 x 8 tile.
// Layout of the work: grid (split of the keys, KV head, sequence), a warp takes chunks of CH keys
// of the CTA's split through a ring of its own (TMA tiles with the 64-byte swizzle for the codes,
// plain bulk copies for the scales), with its own running maximum and sum; the warps of a CTA join
// through shared memory, the splits in decode_fp4_combine_kernel.
//
// f16 operands: K and V are exact in f16.  q is scaled per head by a power of two that puts its
// largest element in [2^14, 2^15), so elements down to 2^-28 of it convert exactly; the power goes
// into the softmax scale.  P is 2^15 exp(s - max), so that it rounds to 11 bits down to 2^-29 of
// the largest; the factor is in P's sum too and cancels.  Sums are fp32.
#include <algorithm>
#include <cmath>

#include "fp4.cuh"
#include "runtime.h"

namespace vlc {
namespace decode_fp4 {

using fp4::HD;
constexpr int CH = 64;                          // keys a step of a warp
constexpr int TILES = CH / 16;
constexpr int WARPS = 4;
constexpr int STAGES = 3;
constexpr int CODE_TILE = CH * fp4::CODE_BYTES;
constexpr int SCALE_TILE = CH * fp4::SCALE_BYTES;
constexpr int STAGE_BYTES = 2 * (CODE_TILE + SCALE_TILE);
constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
constexpr int SMEM_BYTES = RING_BYTES + 1024;
constexpr int MAX_GROUP = 16;
constexpr float P_SHIFT = 15.f;

struct Params {
  CUtensorMap tm_k, tm_v;  // bytes {64, block_size, pages * Hk}, box {64, CH, 1}
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const __nv_bfloat16* q;
  int64_t q_seq_stride;
  const int32_t* block_tables;
  int64_t table_stride;
  int table_width;
  int block_size;
  int num_pages;
  const int32_t* context_lens;
  int split_keys, max_splits;
  int group, num_heads, num_kv_heads;
  float scale_log2;  // softmax scale * log2(e) * g_k
  float v_scale;
  __nv_bfloat16* out;
  int64_t out_seq_stride;
  float* part_o;   // [num_seqs][max_splits][num_heads][HD]
  float* part_ml;  // [num_seqs][max_splits][num_heads][2]
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lds64(uint32_t a, uint32_t& x, uint32_t& y) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x), "=r"(y) : "r"(a));
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}

// The key of a 16-key tile that S^T's row rho (0..7; rho + 8 is 8 keys on) stands for.  Any
// bijection gives the same sums; this one makes both the K loads (rows 2p, 2p + 1 in different
// 64-byte halves of the banks) and the V loads (rows 0, 2, 4, 6 and 1, 3, 5, 7 over all banks)
// free of conflicts under the 64-byte swizzle.
__device__ __forceinline__ int tile_key(int rho) {
  return (rho & 4) | (((rho >> 1) & 1) ^ ((rho & 1) * 3));
}
// Byte of 16-byte piece `piece` of key `key` in a swizzled code tile.
__device__ __forceinline__ uint32_t swizzled(int key, int piece) {
  return key * 64 + ((piece ^ ((key >> 1) & 3)) << 4);
}

template <int NT>  // 8-head column tiles
__global__ void __launch_bounds__(WARPS * 32, 2) decode_fp4_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_all[WARPS * STAGES];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int split = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int G = p.group;
  int len = __ldg(p.context_lens + b);
  // As in the bf16 decode: a length past the keys that the grid covers is recorded and cut.
  const int cap = p.max_splits * p.split_keys;
  if (len > cap) {
    if (split == 0 && g == 0 && threadIdx.x == 0) record_error(VLC_DEV_ERR_LENGTH);
    len = cap;
  }
  const int nsplit = len > 0 ? (len + p.split_keys - 1) / p.split_keys : 0;
  if (split >= nsplit) {
    if (len <= 0 && split == 0) {  // an empty sequence: zeros
      for (int i = threadIdx.x; i < G * HD / 2; i += blockDim.x)
        reinterpret_cast<uint32_t*>(p.out + (int64_t)b * p.out_seq_stride + (int64_t)g * G * HD)[i] = 0;
    }
    return;
  }
  const int warp = warp_id(), lane = lane_id();
  const int r = lane >> 2, t = lane & 3;
  uint64_t* const full = full_all + warp * STAGES;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(full + s, 1);
    fence_mbar_init();
  }
  __syncwarp();

  const int k_begin = split * p.split_keys;
  const int k_end = min(len, k_begin + p.split_keys);
  const int nchunks = (k_end - k_begin + CH - 1) / CH;
  const int mine = nchunks > warp ? (nchunks - warp + WARPS - 1) / WARPS : 0;  // chunks warp, warp + WARPS, ..
  uint8_t* const ring = smem + warp * (STAGES * STAGE_BYTES);
  const int32_t* const table = p.block_tables + (int64_t)b * p.table_stride;

  // Page of the warp's i-th chunk, or -1 when the table has no usable page there: such a chunk is
  // recorded and left out.
  auto page_of = [&](int i) {
    const int index = (k_begin + (warp + i * WARPS) * CH) / p.block_size;
    const int page = index < p.table_width ? __ldg(table + index) : -1;
    return page >= 0 && page < p.num_pages ? page : -1;
  };
  auto issue = [&](int i) {  // one lane
    const int page = page_of(i);
    if (page < 0) {
      record_error(VLC_DEV_ERR_BLOCK_RANGE);
      return;
    }
    uint64_t* bar = full + i % STAGES;
    uint8_t* st = ring + (i % STAGES) * STAGE_BYTES;
    const int row = (k_begin + (warp + i * WARPS) * CH) % p.block_size;
    const int piece = page * p.num_kv_heads + g;
    const int64_t scales = fp4::head_offset(page, p.num_kv_heads, g, p.block_size) +
                           fp4::scale_offset(row, p.block_size);
    mbar_expect_tx(bar, STAGE_BYTES);
    tma_load_3d(st, &p.tm_k, bar, 0, row, piece);
    bulk_load_1d(st + 2 * CODE_TILE, p.k_cache + scales, SCALE_TILE, bar);
    tma_load_3d(st + CODE_TILE, &p.tm_v, bar, 0, row, piece);
    bulk_load_1d(st + 2 * CODE_TILE + SCALE_TILE, p.v_cache + scales, SCALE_TILE, bar);
  };
  auto arrived = [&](int i) {
    const bool ok = mbar_wait_bounded(full + i % STAGES, (uint32_t)(i / STAGES) & 1u, VLC_DEV_ERR_TIMEOUT + 22,
                                      VLC_WAIT_LIMIT_CYCLES);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  if (lane == 0) {
    for (int i = 0; i < min(STAGES, mine); ++i) issue(i);
  }

  // Q as B fragments: lane (r, t) holds dims 32t .. 32t + 31 of head r (and 8 + r); head powers.
  uint32_t qb[NT][16];
  float head_scale[NT][2];  // of heads 2t and 2t + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int h = n * 8 + r;
    uint4 u[4] = {};
    if (h < G) {
      const uint4* src =
          reinterpret_cast<const uint4*>(p.q + (int64_t)b * p.q_seq_stride + (int64_t)(g * G + h) * HD + 32 * t);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __ldg(src + i);
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
    uint32_t top = 0;  // largest bf16 magnitude
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(141 - e) for a largest element with exponent field e puts it in [2^14, 2^15); e is kept
    // where both that power and its inverse are normal.  All-zero and non-finite rows: power 1.
    int e = (int)(top >> 7);
    e = (top == 0 || e == 255) ? 141 : max(e, 15);
    const float up = __uint_as_float((uint32_t)(127 + 141 - e) << 23);
    const float down = __uint_as_float((uint32_t)(127 - 141 + e) << 23);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      qb[n][i] = pack_f16x2(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
    head_scale[n][0] = p.scale_log2 * __shfl_sync(0xffffffffu, down, 8 * t);      // lane of head 2t
    head_scale[n][1] = p.scale_log2 * __shfl_sync(0xffffffffu, down, 8 * t + 4);  // of head 2t + 1
  }

  float o[NT][8][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }
  const uint32_t ring_u = smem_u32(ring);
  const int kr = tile_key(r);
  // V fragment columns 2t, 2t + 1 (and 8 more): keys of S^T's rows 2t and 2t + 1
  const int kv0 = tile_key(2 * t), kv1 = tile_key(2 * t + 1);

  for (int i = 0; i < mine; ++i) {
    if (page_of(i) < 0) {
      if (lane == 0) {
        mbar_arrive(full + i % STAGES);  // nothing was issued: the barrier's phase is turned over here
        if (i + STAGES < mine) issue(i + STAGES);
      }
      __syncwarp();
      continue;
    }
    if (!arrived(i)) {  // recorded; the copies still in flight are given the same time before the warp leaves
      for (int x = i + 1; x < min(i + STAGES, mine); ++x)
        if (page_of(x) >= 0) arrived(x);
      break;
    }
    const uint32_t st = ring_u + (i % STAGES) * STAGE_BYTES;
    const int valid = k_end - (k_begin + (warp + i * WARPS) * CH);  // keys of the chunk that count

    // ---- S^T = K Q^T
    float s[TILES][NT][4];
#pragma unroll
    for (int kt = 0; kt < TILES; ++kt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[kt][n][0] = s[kt][n][1] = s[kt][n][2] = s[kt][n][3] = 0.f;
      const int k0 = kt * 16 + kr, k1 = k0 + 8;
      uint32_t c0[4], c1[4];
      lds128(st + swizzled(k0, t), c0);
      lds128(st + swizzled(k1, t), c1);
      const uint32_t f0 = fp4::scales2_f16(lds_u16(st + 2 * CODE_TILE + k0 * 8 + 2 * t));
      const uint32_t f1 = fp4::scales2_f16(lds_u16(st + 2 * CODE_TILE + k1 * 8 + 2 * t));
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // four bytes: k-steps 2w and 2w + 1
        const uint32_t sc0 = __byte_perm(f0, 0, w < 2 ? 0x1010 : 0x3232);
        const uint32_t sc1 = __byte_perm(f1, 0, w < 2 ? 0x1010 : 0x3232);
        uint32_t h0[4], h1[4];
        fp4::decode8(c0[w], h0);
        fp4::decode8(c1[w], h1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          h0[x] = hmul2(h0[x], sc0);
          h1[x] = hmul2(h1[x], sc1);
        }
        const uint32_t a0[4] = {h0[0], h1[0], h0[1], h1[1]};
        const uint32_t a1[4] = {h0[2], h1[2], h0[3], h1[3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(s[kt][n], a0, qb[n][4 * w], qb[n][4 * w + 1]);
          mma_f16(s[kt][n], a1, qb[n][4 * w + 2], qb[n][4 * w + 3]);
        }
      }
    }
    // ---- running softmax, log2 domain; lane holds keys of rows r, r + 8 for heads 2t, 2t + 1
    uint32_t pb[TILES][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < TILES; ++kt) {
        float(&x)[4] = s[kt][n];
        x[0] *= head_scale[n][0];
        x[1] *= head_scale[n][1];
        x[2] *= head_scale[n][0];
        x[3] *= head_scale[n][1];
        if (valid < CH) {
          if (kt * 16 + kr >= valid) x[0] = x[1] = -INFINITY;
          if (kt * 16 + kr + 8 >= valid) x[2] = x[3] = -INFINITY;
        }
        top0 = fmaxf(top0, fmaxf(x[0], x[2]));
        top1 = fmaxf(top1, fmaxf(x[1], x[3]));
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
        top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
      }
      const float m0 = fmaxf(m[n][0], top0), m1 = fmaxf(m[n][1], top1);
      // (-inf: no key so far)
      const float f0 = m0 == -INFINITY ? 0.f : fast_exp2(m[n][0] - m0);
      const float f1 = m1 == -INFINITY ? 0.f : fast_exp2(m[n][1] - m1);
      const float r0 = m0 == -INFINITY ? 0.f : m0 - P_SHIFT, r1 = m1 == -INFINITY ? 0.f : m1 - P_SHIFT;
      m[n][0] = m0;
      m[n][1] = m1;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int kt = 0; kt < TILES; ++kt) {
        float(&x)[4] = s[kt][n];
        x[0] = fast_exp2(x[0] - r0);
        x[1] = fast_exp2(x[1] - r1);
        x[2] = fast_exp2(x[2] - r0);
        x[3] = fast_exp2(x[3] - r1);
        l0 += x[0] + x[2];
        l1 += x[1] + x[3];
        pb[kt][n][0] = transpose8x8(pack_f16x2(x[0], x[1]));
        pb[kt][n][1] = transpose8x8(pack_f16x2(x[2], x[3]));
      }
      l[n][0] = l[n][0] * f0 + l0;
      l[n][1] = l[n][1] * f1 + l1;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        o[n][mt][0] *= f0;
        o[n][mt][1] *= f1;
        o[n][mt][2] *= f0;
        o[n][mt][3] *= f1;
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int kt = 0; kt < TILES; ++kt) {
      const int key[4] = {kt * 16 + kv0, kt * 16 + kv1, kt * 16 + 8 + kv0, kt * 16 + 8 + kv1};
      uint32_t c[4][2], sb[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        lds64(st + CODE_TILE + swizzled(key[x], r >> 1) + 8 * (r & 1), c[x][0], c[x][1]);
        sb[x] = lds_u8(st + 2 * CODE_TILE + SCALE_TILE + key[x] * 8 + r);
        // rows past the end may hold anything: their P is 0, and a scale of 0 makes V 0
        if (valid < CH && key[x] >= valid) sb[x] = 0;
      }
      const uint32_t sc01 = fp4::scales2_f16(sb[0] | (sb[1] << 8)), sc23 = fp4::scales2_f16(sb[2] | (sb[3] << 8));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        // bytes of {key 0 or 2, key 1 or 3} x {low nibbles: dims 16r + 2i, high: 16r + 2i + 1}
        const uint32_t lo01 = (c[0][w] & 0x0f0f0f0fu) | ((c[1][w] << 4) & 0xf0f0f0f0u);
        const uint32_t hi01 = ((c[0][w] >> 4) & 0x0f0f0f0fu) | (c[1][w] & 0xf0f0f0f0u);
        const uint32_t lo23 = (c[2][w] & 0x0f0f0f0fu) | ((c[3][w] << 4) & 0xf0f0f0f0u);
        const uint32_t hi23 = ((c[2][w] >> 4) & 0x0f0f0f0fu) | (c[3][w] & 0xf0f0f0f0u);
        uint32_t a0[4], a1[4], a2[4], a3[4];
        fp4::decode8(lo01, a0);
        fp4::decode8(hi01, a1);
        fp4::decode8(lo23, a2);
        fp4::decode8(hi23, a3);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t a[4] = {hmul2(a0[x], sc01), hmul2(a1[x], sc01), hmul2(a2[x], sc23), hmul2(a3[x], sc23)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][4 * w + x], a, pb[kt][n][0], pb[kt][n][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0 && i + STAGES < mine) issue(i + STAGES);
  }

  // ---- join the warps: every copy into the ring was waited for, its memory is free
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], d);
      l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], d);
    }
  __syncthreads();
  constexpr int HEADS = NT * 8;
  float* sm_o = reinterpret_cast<float*>(smem);        // [WARPS][HEADS][HD]
  float* sm_ml = sm_o + WARPS * HEADS * HD;            // [WARPS][HEADS][2]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int h = n * 8 + 2 * t;
    float* d0 = sm_o + (warp * HEADS + h) * HD + 16 * r;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      *reinterpret_cast<float2*>(d0 + 2 * mt) = make_float2(o[n][mt][0], o[n][mt][2]);
      *reinterpret_cast<float2*>(d0 + HD + 2 * mt) = make_float2(o[n][mt][1], o[n][mt][3]);
    }
    if (r == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sm_ml[(warp * HEADS + h + x) * 2] = m[n][x];
        sm_ml[(warp * HEADS + h + x) * 2 + 1] = l[n][x];
      }
    }
  }
  __syncthreads();
  // four dims a thread, heads over the warps
  for (int h = warp; h < G; h += WARPS) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_ml[(w * HEADS + h) * 2]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = fast_exp2(sm_ml[(w * HEADS + h) * 2] - ref);
      L += f * sm_ml[(w * HEADS + h) * 2 + 1];
      const float4 x = reinterpret_cast<const float4*>(sm_o + (w * HEADS + h) * HD)[lane];
      acc.x += f * x.x;
      acc.y += f * x.y;
      acc.z += f * x.z;
      acc.w += f * x.w;
    }
    const int head = g * G + h;
    if (nsplit == 1) {
      const float inv = L != 0.f ? p.v_scale / L : 0.f;
      uint2 u;
      u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      reinterpret_cast<uint2*>(p.out + (int64_t)b * p.out_seq_stride + (int64_t)head * HD)[lane] = u;
    } else {
      const int64_t pi = ((int64_t)b * p.max_splits + split) * p.num_heads + head;
      reinterpret_cast<float4*>(p.part_o + pi * HD)[lane] = acc;
      if (lane == 0) reinterpret_cast<float2*>(p.part_ml)[pi] = make_float2(M, L);
    }
  }
}

// Joins the splits of each (sequence, head): one warp a head, four dims a lane.
__global__ void __launch_bounds__(128) decode_fp4_combine_kernel(const float* __restrict__ part_o,
                                                                 const float* __restrict__ part_ml,
                                                                 const int32_t* __restrict__ context_lens,
                                                                 int split_keys, int max_splits, int num_heads,
                                                                 float v_scale, __nv_bfloat16* __restrict__ out,
                                                                 int64_t out_seq_stride) {
  const int b = blockIdx.x;
  const int h = blockIdx.y * 4 + warp_id();
  const int lane = lane_id();
  if (h >= num_heads) return;
  const int len = min(__ldg(context_lens + b), max_splits * split_keys);
  const int nsplit = len > 0 ? (len + split_keys - 1) / split_keys : 0;
  if (nsplit <= 1) return;  // written by the decode kernel
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + (int64_t)b * max_splits * num_heads + h;
  const float4* po = reinterpret_cast<const float4*>(part_o) + ((int64_t)b * max_splits * num_heads + h) * (HD / 4);
  float M = -INFINITY;
  for (int s = lane; s < nsplit; s += 32) M = fmaxf(M, ml[(int64_t)s * num_heads].x);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < nsplit; ++s) {
    const float2 x = ml[(int64_t)s * num_heads];
    const float4 v = po[(int64_t)s * num_heads * (HD / 4) + lane];
    const float f = fast_exp2(x.x - ref);
    L += f * x.y;
    acc.x += f * v.x;
    acc.y += f * v.y;
    acc.z += f * v.z;
    acc.w += f * v.w;
  }
  const float inv = L != 0.f ? v_scale / L : 0.f;
  uint2 u;
  u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  reinterpret_cast<uint2*>(out + (int64_t)b * out_seq_stride + (int64_t)h * HD)[lane] = u;
}

// Keys of a split: from host values only, so that the grid is fixed for graph capture.
static int choose_split_keys(int num_seqs, int num_kv_heads, int max_context_len, int num_sms) {
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads;
  const int64_t target = 8LL * num_sms;
  const int64_t splits = std::max<int64_t>(1, (target + pairs - 1) / pairs);
  const int64_t step = WARPS * CH;
  int64_t sk = (max_context_len + splits - 1) / splits;
  sk = (sk + step - 1) / step * step;
  return (int)std::max<int64_t>(512, std::min<int64_t>(sk, 2048));
}

static bool power_of_two(float g) {
  int e;
  return std::isfinite(g) && g > 0.f && std::frexp(g, &e) == 0.5f && e >= -63 && e <= 65;
}

}  // namespace decode_fp4
}  // namespace vlc

using namespace vlc;
using namespace vlc::decode_fp4;

extern "C" int64_t vlc_decode_fp4_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int max_context_len) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_context_len <= 0) return 0;
  const int sk = choose_split_keys(num_seqs, num_kv_heads, max_context_len, vlc_num_sms());
  const int64_t max_splits = ((int64_t)max_context_len + sk - 1) / sk;
  if (max_splits <= 1) return 0;
  return (int64_t)num_seqs * max_splits * num_heads * (HD + 2) * (int64_t)sizeof(float);
}

extern "C" int vlc_decode_attn_fp4(const void* q, int64_t q_seq_stride, int num_seqs, int num_heads,
                                   const void* k_cache, const void* v_cache, int64_t num_pages, int block_size,
                                   int num_kv_heads, int head_dim, const int32_t* block_tables,
                                   int64_t block_table_stride, int block_table_width, const int32_t* context_lens,
                                   int max_context_len, float softmax_scale, float k_scale, float v_scale, void* out,
                                   int64_t out_seq_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || max_context_len < 0 || max_context_len > (1 << 30) || block_table_width < 0)
    return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % CH != 0) return VLC_ERR_UNSUPPORTED;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return VLC_ERR_SHAPE;
  const int G = num_heads / num_kv_heads;
  if (G > MAX_GROUP || !power_of_two(k_scale) || !power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0) return VLC_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out) return VLC_ERR_NULL;
  if (q_seq_stride % 8 || out_seq_stride % 8 || q_seq_stride < (int64_t)num_heads * HD ||
      out_seq_stride < (int64_t)num_heads * HD || block_table_stride < block_table_width)
    return VLC_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return VLC_ERR_ALIGN;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size || num_pages * num_kv_heads > 0x7fffffff)
    return VLC_ERR_SHAPE;
  if (num_kv_heads > 65535 || num_seqs > 65535) return VLC_ERR_SHAPE;
  if (max_context_len == 0) max_context_len = 1;
  const int sk = choose_split_keys(num_seqs, num_kv_heads, max_context_len, vlc_num_sms());
  const int max_splits = (max_context_len + sk - 1) / sk;
  const int64_t need = vlc_decode_fp4_workspace_size(num_seqs, num_heads, num_kv_heads, max_context_len);
  if (need > 0 && (!workspace || workspace_bytes < need)) return VLC_ERR_WORKSPACE;
  if (need > 0 && !aligned16(workspace)) return VLC_ERR_ALIGN;

  Params p;
  const uint64_t dims[3] = {(uint64_t)fp4::CODE_BYTES, (uint64_t)block_size, (uint64_t)(num_pages * num_kv_heads)};
  const uint64_t strides[2] = {(uint64_t)fp4::CODE_BYTES, (uint64_t)block_size * fp4::ROW_BYTES};
  const uint32_t box[3] = {(uint32_t)fp4::CODE_BYTES, (uint32_t)CH, 1};
  if (encode_tmap_u8(&p.tm_k, k_cache, 3, dims, strides, box, 64) != VLC_OK) return VLC_ERR_CUDA;
  if (encode_tmap_u8(&p.tm_v, v_cache, 3, dims, strides, box, 64) != VLC_OK) return VLC_ERR_CUDA;
  p.k_cache = (const uint8_t*)k_cache;
  p.v_cache = (const uint8_t*)v_cache;
  p.q = (const __nv_bfloat16*)q;
  p.q_seq_stride = q_seq_stride;
  p.block_tables = block_tables;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.block_size = block_size;
  p.num_pages = (int)num_pages;
  p.context_lens = context_lens;
  p.split_keys = sk;
  p.max_splits = max_splits;
  p.group = G;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.scale_log2 = softmax_scale * 1.4426950408889634f * k_scale;
  p.v_scale = v_scale;
  p.out = (__nv_bfloat16*)out;
  p.out_seq_stride = out_seq_stride;
  p.part_o = (float*)workspace;
  p.part_ml = workspace ? p.part_o + (int64_t)num_seqs * max_splits * num_heads * HD : nullptr;

  static std::atomic<uint64_t> smem1{0}, smem2{0};
  const dim3 grid(max_splits, num_kv_heads, num_seqs);
  cudaStream_t st = (cudaStream_t)stream;
  if (G <= 8) {
    if (ensure_dynamic_smem((const void*)decode_fp4_kernel<1>, SMEM_BYTES, smem1) != VLC_OK) return VLC_ERR_CUDA;
    decode_fp4_kernel<1><<<grid, WARPS * 32, SMEM_BYTES, st>>>(p);
  } else {
    if (ensure_dynamic_smem((const void*)decode_fp4_kernel<2>, SMEM_BYTES, smem2) != VLC_OK) return VLC_ERR_CUDA;
    decode_fp4_kernel<2><<<grid, WARPS * 32, SMEM_BYTES, st>>>(p);
  }
  const int rc = launch_status();
  if (rc != VLC_OK || max_splits <= 1) return rc;
  const dim3 cg(num_seqs, (num_heads + 3) / 4);
  decode_fp4_combine_kernel<<<cg, 128, 0, st>>>(p.part_o, p.part_ml, context_lens, sk, max_splits, num_heads, v_scale,
                                              p.out, out_seq_stride);
  return launch_status();
}
