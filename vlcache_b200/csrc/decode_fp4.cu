// Paged decode attention over the 4-bit KV cache (one query token per sequence), sm_100a.
//
//   o[h] = sum_j softmax_j(scale * g_k * q[h] . K[j]) * g_v * V[j],   K, V = s * code per group.
//
// The floor is HBM: 72 bytes per key and head for K and V each.  At that rate an SM has to take in
// 3.6 times the keys a second of the bf16 decode, so the work per element counts:
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
// Layout of the work: the keys of all (sequence, KV head) pairs, in chunks of 64, form one line that
// the grid's warps share out evenly, each a contiguous run of it.  The shares are equal whatever
// the lengths are (a grid of fixed splits left SMs idle at its end, paid a prologue and a join
// every few chunks and merged in shared memory: 267 us for 256 sequences of 2700 .. 10700 keys, 28
// query and 4 KV heads, against 178 us now).  A warp works alone: its own ring of chunks (TMA
// tiles, with the 64-byte swizzle for the codes and without one for the scales, issued by its lane
// 0), its own running maximum and sums, no barrier with any other warp.  A pair that a warp has to
// itself is written out; the parts of a pair that several warps share go to the workspace and
// decode_fp4_combine_kernel, launched as a programmatic dependent, joins them.
//
// f16 operands: K and V are exact in f16.  q is scaled per head by a power of two that puts its
// largest element in [2^14, 2^15), so elements down to 2^-28 of it convert exactly; the power goes
// into the softmax scale.  P is 2^12 exp(s - m) with m within 2^3 of the running maximum, so that it
// rounds to 11 bits down to 2^-26 of the largest; the factor is in P's sum too (an MMA with ones
// takes it) and cancels.  Sums are fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fp4.cuh"
#include "runtime.h"

namespace vlc {
namespace decode_fp4 {

using fp4::HD;
constexpr int CH = 64;                          // keys a step of a warp
constexpr int TILES = CH / 16;
constexpr int WARPS = 2;                        // a block's warps share nothing but the launch
constexpr int STAGES = 2;
constexpr int CODE_TILE = CH * fp4::CODE_BYTES;
constexpr int SCALE_TILE = CH * fp4::SCALE_BYTES;
constexpr int STAGE_BYTES = 2 * (CODE_TILE + SCALE_TILE);
constexpr int SMEM_BYTES = WARPS * STAGES * STAGE_BYTES + 512;  // + alignment to the swizzle's period
constexpr int MAX_GROUP = 16;
constexpr float P_SHIFT = 12.f;
constexpr float SLACK = 3.f;                    // log2 that the maximum may grow by before O is rescaled

// Blocks an SM holds: 12 warps of up to 168 registers with 8 query heads, 8 warps with 16.
constexpr int blocks_per_sm(int NT) { return NT == 1 ? 6 : 4; }

struct Params {
  // K's and V's codes {64, block_size, pages * Hk} and scales {64, block_size / 8, pages * Hk}, in
  // bytes (boxes {64, CH} and {64, CH / 8}).  Joined, codes[0] and scales[0] have a fourth dimension,
  // the two caches, whose stride is their distance: a chunk is then two copies instead of four (183
  // -> 179 us for 256 sequences).  v_first: V lies before K.
  CUtensorMap codes[2], scales[2];
  bool joined;
  bool v_first;
  const __nv_bfloat16* q;
  int64_t q_seq_stride;
  const int32_t* block_tables;
  int64_t table_stride;
  int table_width;
  int block_size;
  int num_pages;
  const int32_t* context_lens;
  int num_seqs, max_len;
  int group, num_heads, num_kv_heads;
  float scale_log2;  // |softmax scale| * log2(e) * g_k
  float q_sign;      // the softmax scale's sign
  float v_scale;
  __nv_bfloat16* out;
  int64_t out_seq_stride;
  int num_warps;
  // Workspace: a warp's first pair and its last leave parts when they are not whole.
  float* parts;    // [num_warps][2][group][HD] sums of P V
  float2* part_ml;  // [num_warps][2][group] (maximum, sum of P)
  int2* places;    // [num_seqs][num_kv_heads] of each pair with keys: (slot of its first part, parts)
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
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, __half2 b) {
  const __half2 d = __hmul2(as_half2(a), b);
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Bits of a where the mask is set, of b elsewhere: one instruction.
__device__ __forceinline__ uint32_t select_bits(uint32_t mask, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xca;" : "=r"(d) : "r"(mask), "r"(a), "r"(b));
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

// Chunks of a sequence.  A length past the host's bound is cut to it (recorded by the caller).
__device__ __forceinline__ int chunks_of(int len, int max_len) { return (min(max(len, 0), max_len) + CH - 1) / CH; }

// How the line of `total` chunks is shared: every warp takes each() of them and the first extra()
// one more.
struct Shares {
  int64_t each, extra;
  __device__ __forceinline__ Shares(int64_t total, int num_warps) : each(total / num_warps), extra(total % num_warps) {}
  __device__ __forceinline__ int64_t first(int64_t warp) const { return warp * each + min(warp, extra); }
  __device__ __forceinline__ int64_t count(int64_t warp) const { return each + (warp < extra ? 1 : 0); }
  __device__ __forceinline__ int64_t warp_of(int64_t chunk) const {
    const int64_t big = extra * (each + 1);
    return chunk < big ? chunk / (each + 1) : extra + (chunk - big) / each;
  }
};

// A query head group's state of a warp: S^T, O^T and the softmax, and the step over one chunk.
template <int NT>  // 8-head column tiles
struct State {
  uint32_t qb[NT][16];      // Q as B fragments: dims 32t .. 32t + 31 of head r (and 8 + r)
  float scale[NT][2];       // of scores, heads 2t and 2t + 1
  float o[NT][8][4];        // m-tile i: dims 16r + 2i (0, 1) and 16r + 2i + 1 (2, 3) of heads 2t, 2t + 1
  float l[NT][4];           // sums of P: 0 and 1 of heads 2t, 2t + 1
  float m[NT][2];           // the maximum that P is relative to
  float shift[NT][2];       // P_SHIFT - m (0 before the first key)

  __device__ __forceinline__ void start(const __nv_bfloat16* q, int G, int r, int t, float scale_log2, float sign) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = n * 8 + r;
      uint4 u[4] = {};
      if (h < G) {
        const uint4* src = reinterpret_cast<const uint4*>(q + (int64_t)h * HD + 32 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __ldg(src + i);
      }
      const uint32_t w[16] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w,
                              u[2].x, u[2].y, u[2].z, u[2].w, u[3].x, u[3].y, u[3].z, u[3].w};
      uint32_t top = 0;  // largest bf16 magnitude
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(141 - e) for a largest element with exponent field e puts it in [2^14, 2^15); e is kept
      // where both that power and its inverse are normal.  All-zero rows: power 1.  A row with an
      // infinity has scores of +-infinity or NaN only, whose softmax is NaN, also where all of them
      // are -infinity (which would read as no key): such rows become NaN here.
      int e = (int)(top >> 7);
      const bool finite = e != 255;
      e = (top == 0 || !finite) ? 141 : max(e, 15);
      const float up = finite ? __uint_as_float((uint32_t)(127 + 141 - e) << 23) * sign : __int_as_float(0x7fffffff);
      const float down = __uint_as_float((uint32_t)(127 - 141 + e) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        qb[n][i] = pack_f16x2(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
      scale[n][0] = scale_log2 * __shfl_sync(0xffffffffu, down, 8 * t);      // lane of head 2t
      scale[n][1] = scale_log2 * __shfl_sync(0xffffffffu, down, 8 * t + 4);  // of head 2t + 1
#pragma unroll
      for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      l[n][0] = l[n][1] = l[n][2] = l[n][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      shift[n][0] = shift[n][1] = 0.f;
    }
  }

  // One chunk at `st`.  CUT: only its first `valid` keys count.
  template <bool CUT>
  __device__ __forceinline__ void step(uint32_t st, uint32_t k_at, int valid, int r, int t) {
    const int kr = tile_key(r);
    // k_at: 0 or 1, K's place among the two
    const uint32_t k_codes = st + k_at * CODE_TILE + swizzled(kr, t);
    const uint32_t k_scales = st + 2 * CODE_TILE + k_at * SCALE_TILE + kr * 8 + 2 * t;
    const uint32_t v_at = k_at ^ 1;
    // ---- S^T = K Q^T
    float s[TILES][NT][4];
#pragma unroll
    for (int kt = 0; kt < TILES; ++kt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[kt][n][0] = s[kt][n][1] = s[kt][n][2] = s[kt][n][3] = 0.f;
      uint32_t c0[4], c1[4];  // keys kr and kr + 8 of the tile (8 keys on, the swizzle is the same)
      lds128(k_codes + kt * 1024, c0);
      lds128(k_codes + kt * 1024 + 512, c1);
      const __half2 f0 = as_half2(fp4::scales2_f16(lds_u16(k_scales + kt * 128)));
      const __half2 f1 = as_half2(fp4::scales2_f16(lds_u16(k_scales + kt * 128 + 64)));
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // four bytes: k-steps 2w and 2w + 1
        // (a half on both sides of a multiplication is an operand's form, not an instruction)
        const __half2 sc0 = w < 2 ? __low2half2(f0) : __high2half2(f0);
        const __half2 sc1 = w < 2 ? __low2half2(f1) : __high2half2(f1);
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
    // ---- running softmax, log2 domain; a lane holds keys of rows r, r + 8 for heads 2t, 2t + 1
    uint32_t pb[TILES][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < TILES; ++kt) {
        float(&x)[4] = s[kt][n];
        if (CUT) {
          if (kt * 16 + kr >= valid) x[0] = x[1] = -INFINITY;
          if (kt * 16 + kr + 8 >= valid) x[2] = x[3] = -INFINITY;
        }
        top0 = fmax3(top0, x[0], x[2]);
        top1 = fmax3(top1, x[1], x[3]);
      }
      top0 *= scale[n][0];
      top1 *= scale[n][1];
      // The lanes' own maxima tell whether any grew past the slack; only then are they joined.
      if (__any_sync(0xffffffffu, top0 > m[n][0] + SLACK || top1 > m[n][1] + SLACK)) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
        }
        const float m0 = fmaxf(m[n][0], top0), m1 = fmaxf(m[n][1], top1);
        const float f0 = m0 == -INFINITY ? 0.f : fast_exp2(m[n][0] - m0);  // (-inf: no key so far)
        const float f1 = m1 == -INFINITY ? 0.f : fast_exp2(m[n][1] - m1);
        m[n][0] = m0;
        m[n][1] = m1;
        shift[n][0] = m0 == -INFINITY ? 0.f : P_SHIFT - m0;
        shift[n][1] = m1 == -INFINITY ? 0.f : P_SHIFT - m1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[n][i][0] *= f0;
          o[n][i][1] *= f1;
          o[n][i][2] *= f0;
          o[n][i][3] *= f1;
        }
        l[n][0] *= f0;
        l[n][1] *= f1;
      }
#pragma unroll
      for (int kt = 0; kt < TILES; ++kt) {
        float(&x)[4] = s[kt][n];
        x[0] = fast_exp2(fmaf(x[0], scale[n][0], shift[n][0]));
        x[1] = fast_exp2(fmaf(x[1], scale[n][1], shift[n][1]));
        x[2] = fast_exp2(fmaf(x[2], scale[n][0], shift[n][0]));
        x[3] = fast_exp2(fmaf(x[3], scale[n][1], shift[n][1]));
        if (CUT) {  // (not left to exp2(-inf): a scale of 0 would make it exp2(NaN))
          if (kt * 16 + kr >= valid) x[0] = x[1] = 0.f;
          if (kt * 16 + kr + 8 >= valid) x[2] = x[3] = 0.f;
        }
        pb[kt][n][0] = transpose8x8(pack_f16x2(x[0], x[1]));
        pb[kt][n][1] = transpose8x8(pack_f16x2(x[2], x[3]));
      }
    }
    // ---- O^T += V^T P^T; V's columns 2t, 2t + 1 (and 8 more) are the keys of S^T's rows of that number
    const int kv[2] = {tile_key(2 * t), tile_key(2 * t + 1)};
    uint32_t v_codes[2], v_scales[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      v_codes[x] = st + v_at * CODE_TILE + swizzled(kv[x], r >> 1) + 8 * (r & 1);
      v_scales[x] = st + 2 * CODE_TILE + v_at * SCALE_TILE + kv[x] * 8 + r;
    }
    const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
    for (int kt = 0; kt < TILES; ++kt) {
      uint32_t c[4][2], sb[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        lds64(v_codes[x & 1] + kt * 1024 + (x >> 1) * 512, c[x][0], c[x][1]);
        sb[x] = lds_u8(v_scales[x & 1] + kt * 128 + (x >> 1) * 64);
        // rows past the end may hold anything: their P is 0, and a scale of 0 makes V 0
        if (CUT && kt * 16 + kv[x & 1] + (x >> 1) * 8 >= valid) sb[x] = 0;
      }
      const __half2 sc01 = as_half2(fp4::scales2_f16(__byte_perm(sb[0], sb[1], 0x0040)));
      const __half2 sc23 = as_half2(fp4::scales2_f16(__byte_perm(sb[2], sb[3], 0x0040)));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(l[n], ones, pb[kt][n][0], pb[kt][n][1]);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        // bytes of {key 0 or 2, key 1 or 3} x {low nibbles: dims 16r + 2i, high: 16r + 2i + 1}
        constexpr uint32_t LOW = 0x0f0f0f0fu;
        const uint32_t lo01 = select_bits(LOW, c[0][w], c[1][w] << 4);
        const uint32_t hi01 = select_bits(LOW, c[0][w] >> 4, c[1][w]);
        const uint32_t lo23 = select_bits(LOW, c[2][w], c[3][w] << 4);
        const uint32_t hi23 = select_bits(LOW, c[2][w] >> 4, c[3][w]);
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
  }
};

// A running (maximum, sum of P, four dims of O) and its union with another part's.
struct Joined {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float m2, float l2, const float4& o2) {
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
    const float f = fast_exp2(m - ref), g = fast_exp2(m2 - ref);
    m = top;
    l = l * f + l2 * g;
    o = make_float4(o.x * f + o2.x * g, o.y * f + o2.y * g, o.z * f + o2.z * g, o.w * f + o2.w * g);
  }
  __device__ __forceinline__ uint2 result(float v_scale) const {
    const float inv = l != 0.f ? v_scale / l : 0.f;
    return make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
};

// Both caches' chunk at `row` of a head's piece into a stage.
__device__ __forceinline__ void copy_chunk(const Params& p, uint8_t* st, uint64_t* bar, int row, int piece) {
  tma_load_4d(st, &p.codes[0], bar, 0, row, piece, 0);
  tma_load_4d(st + 2 * CODE_TILE, &p.scales[0], bar, 0, row >> 3, piece, 0);
  if (!p.joined) {
    tma_load_4d(st + CODE_TILE, &p.codes[1], bar, 0, row, piece, 0);
    tma_load_4d(st + 2 * CODE_TILE + SCALE_TILE, &p.scales[1], bar, 0, row >> 3, piece, 0);
  }
}

// Few pairs of few keys: a cluster of four blocks takes a pair, each of its warps one chunk of the
// keys (chunk i block i % 4, so that few chunks spread over the SMs), and the warps join through the
// blocks' shared memory, where a warp's O takes the place of its chunk: four blocks an SM.  One launch
// where the line of chunks takes two, and a scheduler for every warp: one sequence of 700 keys, 16
// query and 2 KV heads: 4.8 us against 7.1 with the line (and against 7.2 with sixteen warps in one
// block).  Several chunks a warp, in clusters of 4 or 8, took a microsecond more for the loop and
// gained 5 .. 14 % on the line at 2000 .. 4000 keys.
constexpr int PAIR_BLOCKS = 4, PAIR_WARPS = 4;
constexpr int PAIR_SMEM = PAIR_WARPS * STAGE_BYTES + 512;
constexpr int PAIR_KEYS = PAIR_BLOCKS * PAIR_WARPS * CH;

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <int NT>
__global__ void __launch_bounds__(PAIR_WARPS * 32) __cluster_dims__(PAIR_BLOCKS, 1, 1)
    decode_fp4_pair_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int HEADS = NT * 8;
  static_assert(HEADS * HD * sizeof(float) <= STAGE_BYTES, "a warp's O takes the place of its chunk");
  __shared__ __align__(8) uint64_t full_all[PAIR_WARPS];
  __shared__ __align__(8) float2 sm_ml[PAIR_WARPS][HEADS];
  const int warp = warp_id(), lane = lane_id();
  const int r = lane >> 2, t = lane & 3;
  const int rank = (int)cluster_ctarank();
  const int head = blockIdx.x / PAIR_BLOCKS, seq = blockIdx.y, G = p.group;
  // (at the same place in every block)
  uint8_t* const first = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 511) & ~uintptr_t(511));
  uint8_t* const st = first + warp * STAGE_BYTES;
  uint64_t* const full = full_all + warp;
  const int key = (warp * PAIR_BLOCKS + rank) * CH, index = key / p.block_size, row = key - index * p.block_size;
  // loaded beside the length; unused where the chunk is past it
  const int page = index < p.table_width ? __ldg(p.block_tables + (int64_t)seq * p.table_stride + index) : -1;
  int len = __ldg(p.context_lens + seq);
  if (lane == 0) {
    mbar_init(full, 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (len > p.max_len) {
    if (threadIdx.x == 0 && blockIdx.x == 0) record_error(VLC_DEV_ERR_LENGTH);
    len = p.max_len;
  }
  int valid = min(CH, len - key);
  if (valid > 0 && (uint32_t)page >= (uint32_t)p.num_pages) {
    if (lane == 0) record_error(VLC_DEV_ERR_BLOCK_RANGE);
    valid = 0;  // its keys are left out
  }
  if (valid > 0 && lane == 0) {
    mbar_expect_tx(full, STAGE_BYTES);
    copy_chunk(p, st, full, row, page * p.num_kv_heads + head);
  }
  State<NT> state;
  state.start(p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * G * HD, G, r, t, p.scale_log2, p.q_sign);
  if (valid > 0) {
    const bool came = mbar_wait_bounded(full, 0, VLC_DEV_ERR_TIMEOUT + 24, VLC_WAIT_LIMIT_CYCLES);
    if (__all_sync(0xffffffffu, came)) state.template step<true>(smem_u32(st), p.v_first, valid, r, t);
    else mbar_wait_bounded(full, 0, VLC_DEV_ERR_TIMEOUT + 24, VLC_WAIT_LIMIT_CYCLES);  // before O takes its place
    __syncwarp();  // every lane has read the chunk
  }
  float(*const sm_o)[HD] = reinterpret_cast<float(*)[HD]>(st);
#pragma unroll
  for (int x = 0; x < NT * 2; ++x) {
    const int nt = x >> 1, odd = x & 1, h = nt * 8 + 2 * t + odd;
    float4* dst = reinterpret_cast<float4*>(&sm_o[h][16 * r]);
#pragma unroll
    for (int mt = 0; mt < 8; mt += 2)
      dst[mt / 2] = make_float4(state.o[nt][mt][odd], state.o[nt][mt][2 + odd], state.o[nt][mt + 1][odd],
                                state.o[nt][mt + 1][2 + odd]);
    if (r == 0) sm_ml[warp][h] = make_float2(state.m[nt][odd], state.l[nt][odd]);
  }
  cluster_sync();
  const int h = rank * PAIR_WARPS + warp;  // a warp joins a head (at most 16)
  if (h < G) {
    const uint32_t o_at = smem_u32(first) + (h * HD + 4 * lane) * (uint32_t)sizeof(float);
    Joined sum;
    auto join = [&](auto rounds) {
#pragma unroll
      for (int w = 0; w < decltype(rounds)::value; ++w)  // in the order of the chunks
#pragma unroll
        for (int b = 0; b < PAIR_BLOCKS; ++b) {
          const float2 x = ld_cluster_v2(mapa_shared(smem_u32(&sm_ml[w][h]), b));
          const float4 v = ld_cluster_v4(mapa_shared(o_at + w * STAGE_BYTES, b));
          sum.add(x.x, x.y, v);
        }
    };
    static_assert(PAIR_WARPS == 4, "the rounds below");
    if (len <= PAIR_BLOCKS * CH) join(std::integral_constant<int, 1>());
    else if (len <= 2 * PAIR_BLOCKS * CH) join(std::integral_constant<int, 2>());
    else join(std::integral_constant<int, 4>());
    reinterpret_cast<uint2*>(p.out + (int64_t)seq * p.out_seq_stride + ((int64_t)head * G + h) * HD)[lane] =
        sum.result(p.v_scale);  // (no key: zeros)
  }
  cluster_sync();  // the others have read this block's shared memory
}

template <int NT>
__global__ void __launch_bounds__(WARPS * 32, blocks_per_sm(NT)) decode_fp4_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_all[WARPS * STAGES];
  __shared__ int valid_all[WARPS * STAGES];
  pdl_launch_dependents();  // the join waits for this grid's end before it reads
  const int warp = warp_id(), lane = lane_id();
  const int r = lane >> 2, t = lane & 3;
  const int G = p.group, Hk = p.num_kv_heads;
  const int64_t my = (int64_t)blockIdx.x * WARPS + warp;
  uint64_t* const full = full_all + warp * STAGES;
  volatile int* const valid_of = valid_all + warp * STAGES;

  // ---- this warp's run [c0, c1) of the line, and the sequence that c0 lies in
  int64_t total = 0;
  for (int i = lane; i < p.num_seqs; i += 32) {
    const int len = __ldg(p.context_lens + i);
    if (my == 0 && len > p.max_len) record_error(VLC_DEV_ERR_LENGTH);
    total += chunks_of(len, p.max_len);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  total *= Hk;
  const Shares shares(total, p.num_warps);
  const int64_t c0 = shares.first(my);
  const int count = (int)shares.count(my);
  if (my >= p.num_warps || count == 0) return;
  int seq = 0;
  int64_t at = c0;  // c0's place among the chunks from the sequence's first on
  for (int base = 0;; base += 32) {
    int64_t n = base + lane < p.num_seqs ? (int64_t)chunks_of(__ldg(p.context_lens + base + lane), p.max_len) * Hk : 0;
    int64_t upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, upto > at);
    if (past) {
      const int first = __ffs(past) - 1;
      seq = base + first;
      at -= __shfl_sync(0xffffffffu, upto - n, first);
      break;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
    if (base + 32 >= p.num_seqs) return;  // not reached: c0 < total
  }
  int len = min(__ldg(p.context_lens + seq), p.max_len);
  int n = (len + CH - 1) / CH;
  int head = (int)(at / n), j = (int)(at - (int64_t)head * n);

  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 511) & ~uintptr_t(511)) +
                        warp * (STAGES * STAGE_BYTES);
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(full + s, 1);
    fence_mbar_init();
  }
  __syncwarp();

  // ---- the issuing side (lane 0): a cursor of its own, STAGES chunks ahead of the other
  struct {
    int seq, head, left, keys;  // chunks and keys of the pair from here on
    int row, index;             // row in the page, page of the sequence
    int page;                   // its number in the cache, loaded when the cursor comes to it
  } ahead = {seq, head, n - j, len - j * CH, (j * CH) % p.block_size, (j * CH) / p.block_size, 0};
  auto load_page = [&]() {
    ahead.page = ahead.index < p.table_width ? __ldg(p.block_tables + ahead.seq * p.table_stride + ahead.index) : -1;
  };
  if (lane == 0) load_page();
  auto issue = [&](int stage, bool more) {
    uint64_t* bar = full + stage;
    uint8_t* st = ring + stage * STAGE_BYTES;
    if ((uint32_t)ahead.page < (uint32_t)p.num_pages) {
      const int piece = ahead.page * Hk + ahead.head;
      valid_of[stage] = min(CH, ahead.keys);
      mbar_expect_tx(bar, STAGE_BYTES);
      copy_chunk(p, st, bar, ahead.row, piece);
    } else {  // the table has no usable page there: recorded, and none of the chunk's keys counts
      valid_of[stage] = 0;
      record_error(VLC_DEV_ERR_BLOCK_RANGE);
      mbar_arrive(bar);
    }
    if (!more) return;
    ahead.row += CH;
    ahead.keys -= CH;
    if (--ahead.left > 0) {
      if (ahead.row < p.block_size) return;
      ahead.row = 0;
      ++ahead.index;
    } else {
      ahead.row = ahead.index = 0;
      if (++ahead.head == Hk) {
        ahead.head = 0;
        do {
          ++ahead.seq;
        } while (__ldg(p.context_lens + ahead.seq) <= 0);  // a chunk follows: so does a sequence with keys
      }
      ahead.keys = min(__ldg(p.context_lens + ahead.seq), p.max_len);
      ahead.left = (ahead.keys + CH - 1) / CH;
    }
    load_page();  // used at the next issue
  };
  if (lane == 0) {
    for (int i = 0; i < min(STAGES, count); ++i) issue(i, i + 1 < count);
  }
  // Whether chunk i came (recorded where it did not).
  auto arrived = [&](int i) {
    const uint32_t parity = (uint32_t)(i / STAGES) & 1u;
    if (mbar_try_wait(full + i % STAGES, parity)) return true;
    return mbar_wait_bounded(full + i % STAGES, parity, VLC_DEV_ERR_TIMEOUT + 22, VLC_WAIT_LIMIT_CYCLES);
  };

  const uint32_t ring_u = smem_u32(ring);
  State<NT> state;
  auto q_of = [&]() { return p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * G * HD; };
  state.start(q_of(), G, r, t, p.scale_log2, p.q_sign);
  // The warp with a pair's first chunk notes where its parts will be: one for each warp up to that of
  // its last chunk, in slot 0 but for this warp's.
  auto note = [&](int64_t chunk, int slot) {
    if (lane == 0)
      p.places[(int64_t)seq * Hk + head] =
          make_int2((int)my * 2 + slot, (int)(shares.warp_of(chunk + n - 1) - my) + 1);
  };
  if (j == 0) note(c0, 0);
  int begin = j;       // first chunk of the pair that is in the state
  int first_slot = 0;  // the part's slot: 0 for the one that holds the warp's first chunk

  for (int i = 0; i < count; ++i) {
    if (!__all_sync(0xffffffffu, arrived(i))) {  // the copies still in flight, this one's too, are given more time
      for (int x = i; x < min(i + STAGES, count); ++x) arrived(x);
      return;
    }
    const uint32_t st = ring_u + (i % STAGES) * STAGE_BYTES;
    const int valid = valid_of[i % STAGES];
    if (valid == CH) state.template step<false>(st, p.v_first, valid, r, t);
    else state.template step<true>(st, p.v_first, valid, r, t);
    __syncwarp();  // every lane has read the stage
    if (lane == 0 && i + STAGES < count) issue(i % STAGES, i + STAGES + 1 < count);
    if (++j < n && i + 1 < count) continue;

    // ---- the pair ends, or the run does
    const bool whole = begin == 0 && j == n;
    float* const part_o = p.parts + (my * 2 + first_slot) * G * HD;
    float2* const part_ml = p.part_ml + (my * 2 + first_slot) * G;
#pragma unroll
    for (int x = 0; x < NT * 2; ++x) {
      const int nt = x >> 1, odd = x & 1;
      const int h = nt * 8 + 2 * t + odd;
      if (h >= G) continue;
      const float sum = state.l[nt][odd];
      if (whole) {
        const float inv = sum != 0.f ? p.v_scale / sum : 0.f;
        uint32_t u[8];
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
          u[mt] = pack_bf16x2(state.o[nt][mt][odd] * inv, state.o[nt][mt][2 + odd] * inv);
        uint4* dst = reinterpret_cast<uint4*>(p.out + (int64_t)seq * p.out_seq_stride + ((int64_t)head * G + h) * HD +
                                              16 * r);
        dst[0] = make_uint4(u[0], u[1], u[2], u[3]);
        dst[1] = make_uint4(u[4], u[5], u[6], u[7]);
      } else {
#pragma unroll
        for (int mt = 0; mt < 8; mt += 4) {  // 32 bytes a store: whole sectors
          uint32_t u[8];
#pragma unroll
          for (int x4 = 0; x4 < 4; ++x4) {
            u[2 * x4] = __float_as_uint(state.o[nt][mt + x4][odd]);
            u[2 * x4 + 1] = __float_as_uint(state.o[nt][mt + x4][2 + odd]);
          }
          st_global_v8(part_o + h * HD + 16 * r + 2 * mt, u);
        }
        if (r == 0) part_ml[h] = make_float2(state.m[nt][odd], sum);
      }
    }
    if (i + 1 == count) break;
    j = begin = 0;
    first_slot = 1;
    if (++head == Hk) {
      head = 0;
      do {
        len = min(__ldg(p.context_lens + ++seq), p.max_len);
      } while (len <= 0);
      n = (len + CH - 1) / CH;
    }
    note(c0 + i + 1, 1);
    state.start(q_of(), G, r, t, p.scale_log2, p.q_sign);
  }
}

// Joins the parts of the pairs that several warps shared and writes zeros for empty sequences.
// kFewParts: a block takes eight heads of a sequence, a warp each, and loads eight parts at once.
// kSomeParts: a block takes one head, and its warps take the parts in turn.  kManyParts: a block takes a
// quarter of one head's dims, and its 32 groups of eight lanes take the parts in turn.  The decode kernel
// fills the SMs to its end, so what a block does before the wait is not hidden: where a pair's parts are
// was noted by the warp that began it.
// Decode and join, us (few : some : many), 28 heads of 4 unless noted: parts 2, 256 sequences of
// 100-1000 keys 35.1 : 47.5 : 101; parts 7, 64 of 3000-5000 37.5 : 40.2 : 55.2; parts 14, 32 of 3000-5000
// 26.6 : 26.5 : 33.2; parts 28, 16 of 5000-8000 25.4 : 21.8 : 25.8; parts 112, 4 of 8000 25.8 : 13.9 : 14.0;
// parts 223, 8 heads of 8, one of 32000 43 : 19.1 : 17.0; parts 445, one of 32000 67 : 18.6 : 14.9.
enum Join { kFewParts, kSomeParts, kManyParts };
template <Join JOIN>
__global__ void __launch_bounds__(256, 3) decode_fp4_combine_kernel(const float* parts, const float2* part_ml,
                                                                 const int2* places, const int32_t* context_lens,
                                                                 int num_warps, int num_heads, int num_kv_heads, float v_scale,
                                                                 __nv_bfloat16* out, int64_t out_seq_stride) {
  constexpr bool SPREAD = JOIN != kFewParts;
  constexpr int LANES = JOIN == kManyParts ? 8 : 32;  // four dims each, of one part
  constexpr int PARTS = 8;  // of a head, loaded at once by a warp of kFewParts
  __shared__ float4 s_o[8][LANES];
  __shared__ float2 s_ml[8];
  const int seq = blockIdx.x, warp = warp_id(), lane = lane_id();
  const int G = num_heads / num_kv_heads;
  const int dim4 = blockIdx.z * LANES + lane % LANES;  // all of the dims, or a quarter
  const float4* po = reinterpret_cast<const float4*>(parts) + dim4;
  uint2* const dst = reinterpret_cast<uint2*>(out + (int64_t)seq * out_seq_stride) + dim4;
  const bool empty = __ldg(context_lens + seq) <= 0;
  // Every block waits, those with nothing to join too: what follows in the stream may rely on this
  // grid's end for the decode kernel's.
  pdl_wait();
  const int h = SPREAD ? blockIdx.y : blockIdx.y * 8 + warp;
  int2 place = make_int2(0, 0);
  if (h < num_heads && !empty) place = places[(int64_t)seq * num_kv_heads + h / G];
  // A warp that gave up waiting for its copies (recorded) leaves pairs unnoted: nothing is read for them.
  if ((uint32_t)place.x >= 2u * num_warps || (uint32_t)place.y > (uint32_t)(num_warps - (place.x >> 1)))
    place = make_int2(0, 1);
  const int64_t first = (int64_t)place.x * G + h % G, rest = (int64_t)(place.x & ~1) * G + h % G;
  const int count = place.y;  // parts of the head, of which part i > 0 is row rest + 2 G i
  if constexpr (SPREAD) {
    if (empty && threadIdx.x < LANES) dst[h * (HD / 4)] = make_uint2(0, 0);
    if (count <= 1) return;  // empty, or written by its warp
    Joined sum;
#pragma unroll 4
    for (int i = threadIdx.x / LANES; i < count; i += 256 / LANES) {
      const int64_t s = i == 0 ? first : rest + (int64_t)i * 2 * G;
      const float2 x = part_ml[s];
      const float4 v = po[s * (HD / 4)];
      sum.add(x.x, x.y, v);
    }
#pragma unroll
    for (int d = LANES; d < 32; d <<= 1) {
      const float m = __shfl_xor_sync(0xffffffffu, sum.m, d), l = __shfl_xor_sync(0xffffffffu, sum.l, d);
      float4 v;
      v.x = __shfl_xor_sync(0xffffffffu, sum.o.x, d);
      v.y = __shfl_xor_sync(0xffffffffu, sum.o.y, d);
      v.z = __shfl_xor_sync(0xffffffffu, sum.o.z, d);
      v.w = __shfl_xor_sync(0xffffffffu, sum.o.w, d);
      sum.add(m, l, v);
    }
    if (lane < LANES) s_o[warp][lane] = sum.o;
    if (lane == 0) s_ml[warp] = make_float2(sum.m, sum.l);
    __syncthreads();
    if (threadIdx.x >= LANES) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) sum.add(s_ml[w].x, s_ml[w].y, s_o[w][lane]);
    dst[h * (HD / 4)] = sum.result(v_scale);
  }
  if constexpr (!SPREAD) {
    if (h >= num_heads || count == 1) return;  // (0 parts: zeros)
    Joined sum;
    for (int i0 = 0; i0 < count; i0 += PARTS) {
      float2 x[PARTS];
      float4 v[PARTS];
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        if (i0 + i >= count) continue;
        const int64_t s = i0 + i == 0 ? first : rest + (int64_t)(i0 + i) * 2 * G;
        x[i] = part_ml[s];
        v[i] = po[s * (HD / 4)];
      }
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        if (i0 + i < count) sum.add(x[i].x, x[i].y, v[i]);
    }
    dst[h * (HD / 4)] = sum.result(v_scale);
  }
}

// Warps of the grid: from host values only, so that it is fixed for graph capture.
static int grid_warps(int num_seqs, int num_heads, int num_kv_heads, int max_context_len, int num_sms) {
  const int64_t most = (int64_t)num_seqs * num_kv_heads * (((int64_t)max_context_len + CH - 1) / CH);
  const int64_t resident = (int64_t)num_sms * WARPS * blocks_per_sm(num_heads / num_kv_heads <= 8 ? 1 : 2);
  return (int)std::max<int64_t>(1, std::min(resident, most));
}

// Whether clusters take whole pairs.  Measured against the line of chunks, us, of 1000 keys (of 200): 28
// heads of 4, 4 pairs 5.2 : 7.2 (4.2 : 7.1), 64 pairs 7.3 : 9.4 (5.4 : 8.5), 128 pairs 10.4 : 13.8
// (6.4 : 9.0), 256 pairs 19.9 : 19.0 (11.6 : 10.1).  With over 8 query heads a KV head (32 of 2) a block
// takes more registers: 64 pairs 10.0 : 13.3 (6.9 : 10.1), 128 pairs 17.3 : 15.8 (13.4 : 11.4).
static bool whole_pairs(int num_seqs, int num_heads, int num_kv_heads, int max_context_len, int num_sms) {
  const int64_t most = num_heads / num_kv_heads <= 8 ? num_sms : num_sms / 2;
  return max_context_len <= PAIR_KEYS && (int64_t)num_seqs * num_kv_heads <= most;
}

// A bound of 0 (every sequence empty) runs as a bound of 1: the join writes the zeros.
static int bound_of(int max_context_len) { return std::max(1, max_context_len); }

static int64_t workspace_bytes_for(int64_t warps, int group, int64_t pairs) {
  return warps * 2 * group * (HD + 2) * (int64_t)sizeof(float) + pairs * (int64_t)sizeof(int2);
}

}  // namespace decode_fp4
}  // namespace vlc

using namespace vlc;
using namespace vlc::decode_fp4;

extern "C" int64_t vlc_decode_fp4_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int max_context_len) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_context_len < 0) return 0;
  max_context_len = bound_of(max_context_len);
  const int sms = vlc_num_sms();
  if (whole_pairs(num_seqs, num_heads, num_kv_heads, max_context_len, sms)) return 0;
  return workspace_bytes_for(grid_warps(num_seqs, num_heads, num_kv_heads, max_context_len, sms),
                             num_heads / num_kv_heads, (int64_t)num_seqs * num_kv_heads);
}

extern "C" int vlc_decode_attn_fp4(const void* q, int64_t q_seq_stride, int num_seqs, int num_heads,
                                   const void* k_cache, const void* v_cache, int64_t num_pages, int block_size,
                                   int num_kv_heads, int head_dim, const int32_t* block_tables,
                                   int64_t block_table_stride, int block_table_width, const int32_t* context_lens,
                                   int max_context_len, float softmax_scale, float k_scale, float v_scale, void* out,
                                   int64_t out_seq_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || max_context_len < 0 || max_context_len > (1 << 30) || block_table_width < 0)
    return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % CH != 0 || block_size > fp4::MAX_BLOCK) return VLC_ERR_UNSUPPORTED;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return VLC_ERR_SHAPE;
  const int G = num_heads / num_kv_heads;
  if (G > MAX_GROUP || !fp4::power_of_two(k_scale) || !fp4::power_of_two(v_scale)) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0) return VLC_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out) return VLC_ERR_NULL;
  if (q_seq_stride % 8 || out_seq_stride % 8 || q_seq_stride < (int64_t)num_heads * HD ||
      out_seq_stride < (int64_t)num_heads * HD || block_table_stride < block_table_width)
    return VLC_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return VLC_ERR_ALIGN;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size || num_pages * num_kv_heads > 0x7fffffff)
    return VLC_ERR_SHAPE;
  if (num_kv_heads > 65535 || num_seqs > 65535 || num_heads > 65535) return VLC_ERR_SHAPE;
  max_context_len = bound_of(max_context_len);
  const int sms = vlc_num_sms();
  const bool whole = whole_pairs(num_seqs, num_heads, num_kv_heads, max_context_len, sms);
  const int warps = whole ? 0 : grid_warps(num_seqs, num_heads, num_kv_heads, max_context_len, sms);
  if (!whole) {
    if (!workspace || workspace_bytes < workspace_bytes_for(warps, G, (int64_t)num_seqs * num_kv_heads))
      return VLC_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 32) return VLC_ERR_ALIGN;
  }

  Params p;
  const uint8_t* caches[2] = {(const uint8_t*)k_cache, (const uint8_t*)v_cache};
  const uint64_t pieces = (uint64_t)(num_pages * num_kv_heads), page_head = (uint64_t)block_size * fp4::ROW_BYTES;
  p.v_first = caches[1] < caches[0];
  if (p.v_first) std::swap(caches[0], caches[1]);
  const uint64_t apart = (uint64_t)(caches[1] - caches[0]);
  p.joined = apart > 0 && apart < 1ull << 40;  // as a tensor map's strides may be
  if (!p.joined && p.v_first) {
    std::swap(caches[0], caches[1]);
    p.v_first = false;
  }
  for (int i = 0; i < (p.joined ? 1 : 2); ++i) {
    const uint64_t both = p.joined ? 2 : 1, last = p.joined ? apart : pieces * page_head;
    const uint64_t dims[4] = {(uint64_t)fp4::CODE_BYTES, (uint64_t)block_size, pieces, both};
    const uint64_t strides[3] = {(uint64_t)fp4::CODE_BYTES, page_head, last};
    const uint32_t box[4] = {(uint32_t)fp4::CODE_BYTES, (uint32_t)CH, 1, (uint32_t)both};
    if (encode_tmap_u8(&p.codes[i], caches[i], 4, dims, strides, box, 64) != VLC_OK) return VLC_ERR_CUDA;
    const uint64_t sdims[4] = {64, (uint64_t)block_size / 8, pieces, both};
    const uint64_t sstrides[3] = {64, page_head, last};
    const uint32_t sbox[4] = {64, (uint32_t)CH / 8, 1, (uint32_t)both};
    if (encode_tmap_u8(&p.scales[i], caches[i] + (int64_t)block_size * fp4::CODE_BYTES, 4, sdims, sstrides, sbox, 0) !=
        VLC_OK)
      return VLC_ERR_CUDA;
  }
  p.q = (const __nv_bfloat16*)q;
  p.q_seq_stride = q_seq_stride;
  p.block_tables = block_tables;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.block_size = block_size;
  p.num_pages = (int)num_pages;
  p.context_lens = context_lens;
  p.num_seqs = num_seqs;
  p.max_len = max_context_len;
  p.group = G;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.scale_log2 = std::fabs(softmax_scale) * 1.4426950408889634f * k_scale;
  p.q_sign = softmax_scale < 0.f ? -1.f : 1.f;
  p.v_scale = v_scale;
  p.out = (__nv_bfloat16*)out;
  p.out_seq_stride = out_seq_stride;
  p.num_warps = warps;
  p.parts = (float*)workspace;
  p.part_ml = (float2*)(p.parts + (int64_t)warps * 2 * G * HD);
  p.places = (int2*)(p.part_ml + (int64_t)warps * 2 * G);

  static std::atomic<uint64_t> smem1{0}, smem2{0}, pair1{0}, pair2{0};
  const int grid = (warps + WARPS - 1) / WARPS;
  cudaStream_t st = (cudaStream_t)stream;
  if (whole) {
    const dim3 pairs(num_kv_heads * PAIR_BLOCKS, num_seqs);
    auto kernel = G <= 8 ? decode_fp4_pair_kernel<1> : decode_fp4_pair_kernel<2>;
    if (ensure_dynamic_smem((const void*)kernel, PAIR_SMEM, G <= 8 ? pair1 : pair2) != VLC_OK) return VLC_ERR_CUDA;
    kernel<<<pairs, PAIR_WARPS * 32, PAIR_SMEM, st>>>(p);
    return launch_status();
  }
  if (G <= 8) {
    if (ensure_dynamic_smem((const void*)decode_fp4_kernel<1>, SMEM_BYTES, smem1) != VLC_OK) return VLC_ERR_CUDA;
    decode_fp4_kernel<1><<<grid, WARPS * 32, SMEM_BYTES, st>>>(p);
  } else {
    if (ensure_dynamic_smem((const void*)decode_fp4_kernel<2>, SMEM_BYTES, smem2) != VLC_OK) return VLC_ERR_CUDA;
    decode_fp4_kernel<2><<<grid, WARPS * 32, SMEM_BYTES, st>>>(p);
  }
  int rc = launch_status();
  if (rc != VLC_OK) return rc;
  // By the parts of a pair on average, and where quarters of all heads are at most two blocks an SM.
  const int64_t parts = warps / ((int64_t)num_seqs * num_kv_heads) + 1;
  const Join join = parts <= 10 ? kFewParts : (int64_t)num_seqs * num_heads <= sms / 2 ? kManyParts : kSomeParts;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = join == kFewParts ? dim3(num_seqs, (num_heads + 7) / 8)
                                  : dim3(num_seqs, num_heads, join == kManyParts ? 4 : 1);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg,
                         join == kFewParts    ? decode_fp4_combine_kernel<kFewParts>
                         : join == kSomeParts ? decode_fp4_combine_kernel<kSomeParts>
                                              : decode_fp4_combine_kernel<kManyParts>,
                         (const float*)p.parts, (const float2*)p.part_ml, (const int2*)p.places, context_lens, warps,
                         num_heads, num_kv_heads, v_scale, p.out, out_seq_stride) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}
