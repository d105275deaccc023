// Paged decode attention of the last 1 .. n tokens of each sequence, with a sliding window and first
// tokens (sinks) that stay visible, sm_100a.
//
//   Row r of a sequence's n has position t = len - n + r and sees key j iff j <= t and
//   (window == 0 or j > t - window or j < sinks):   o = sum_j softmax_j(scale * q . K[j]) * V[j].
//
// The floor is HBM: 512 bytes a key and KV head, each key that any of the n rows sees read once.  So
// the n tokens of a sequence and the G query heads of a KV head are the rows of one product, and a key
// goes through shared memory once for all of them:
//   * K and V are the A operands (16 rows) of m16n8k16 bf16 MMAs, the query rows (token-major, G heads
//     each) the 8 columns: S^T = K Q^T and O^T = V^T P^T.  A tile of 8 rows wastes at most 7, where a
//     tile of 16 would waste half of one token's 7 or 8 heads.
//   * P^T in the layout of a B operand is S^T's accumulator transposed: one movmatrix an 8 x 8 tile.
//   * The keys that a sequence sees are chunks of 16: those of the sinks, then those from the
//     window's first on; what lies between is skipped, its pages are not touched.
// The chunks of all (sequence, KV head) pairs form one line that the grid's blocks share out evenly,
// each a contiguous run of it, so that the shares are equal whatever the lengths are.  In a block a
// warp takes every fourth chunk of the run, with a ring of its own (one TMA copy a chunk, K and V
// together) and a running softmax of its own; at the end of a pair the warps' sums are added through
// shared memory, lane by lane.  A pair that a block has to itself is written out; the parts of a pair
// that several blocks share go to the workspace, and window_join_kernel, a programmatic dependent,
// joins them.  Few pairs of few keys are taken by clusters instead, a pair each, whose blocks join through
// their shared memory: one launch.  A tile of 8 rows takes 32 registers of accumulators and 16 of Q: up to three
// tiles, 24 rows, are here; more go to decode_window_wide.cu, which shares the line and the join.
//
// P is rounded to bf16, V's type, as an operand of its MMA has to be (by 2^-8 of itself at most); its sum
// is taken over the rounded values, so that the error does not add up with the keys.  Scores, maxima
// and sums are fp32.
//
// Measured (64 sequences of 2700 .. 10700 keys, window 4096, 28 query and 4 KV heads; floor 82 .. 83 us): one token
// 86.6 us, two 91, three 95 (decode_window_wide.cu: two 93.6, three 95.1); four, which it takes, 94 (here, by teams of
// two warps: 96), five 96 (106), eight 101 (142).  One token is bound by HBM (76 % of DRAM's nominal rate); with more
// the steps' latency counts: 8 warps an SM, whose registers hold the rows.
#include <algorithm>
#include <cmath>
#include <limits>

#include "decode_window.cuh"
#include "runtime.h"

namespace vlc {
namespace decode_window {

constexpr int WARPS = 4;                 // of a block
constexpr int RING_BYTES = 64 << 10;     // of a block, shared out among its warps
constexpr int CK = 16;                   // keys of a chunk
constexpr int BLOCKS_PER_SM = 2;
constexpr int WIDE_ROWS = 24;            // more rows go to decode_window_wide.cu, whatever the lengths are (wide_of)

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// A warp's rows: S^T, O^T and the softmax, and the step over one chunk.  Lane (r, t) = (lane / 4,
// lane % 4) holds keys r and r + 8 of a chunk, dims 8c + r, and rows 2t and 2t + 1 of each tile.
template <int NT>  // tiles of 8 rows
struct State {
  static constexpr int HALF_BYTES = CK * 128;   // 64 dims of its keys
  uint32_t qb[NT][8][2];  // Q as B fragments: dims 16k + 2t, + 1 (and 8 more) of row r
  float o[NT][8][4];                   // m-tile i: dims 16i + r of rows 2t, 2t + 1 (0, 1), 16i + 8 + r (2, 3)
  float l[NT][4];                      // sums of P: 0 and 1 of rows 2t, 2t + 1
  float m[NT][2];                      // the maximum that P is relative to

  // The pair's rows, row x being token x / G's head x % G.
  __device__ __forceinline__ void start(const Params& p, int seq, int head, int r, int t) {
    const int G = p.group;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = n * 8 + r;
      const int tok = p.token_of(row);
      const bool live = row < p.rows;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          p.q + ((int64_t)seq * p.tokens + (live ? tok : 0)) * p.q_token_stride +
          ((int64_t)head * G + (live ? row - tok * G : 0)) * HD) + t;
      uint32_t top = 0;  // largest bf16 magnitude
      uint32_t u[8][2];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u[k][x] = live ? __ldg(src + 8 * k + 4 * x) ^ p.q_flip : 0u;
          top = max(top, max(u[k][x] & 0x7fffu, (u[k][x] >> 16) & 0x7fffu));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // A row with an infinity has scores of +-infinity or NaN only, whose softmax is NaN, also where
      // all of them are -infinity (which would read as no key): such rows become NaN here.
      const uint32_t spoil = top >= 0x7f80u ? 0x7fff7fffu : 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x) qb[n][k][x] = u[k][x] | spoil;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      l[n][0] = l[n][1] = l[n][2] = l[n][3] = 0.f;
      m[n][0] = m[n][1] = NO_MAX;
    }
  }

  // One chunk whose K and V tiles are at kt and vt; key0 is its first key.  `cut`: not every row sees all of it.
  __device__ __forceinline__ void step(const Params& p, uint32_t kt, uint32_t vt, int key0, bool cut,
                                       const Span<CK>& span, int lane) {
    const int r = lane >> 2, t = lane & 3, mi = lane >> 3, ri = lane & 7;
    // ---- S^T = K Q^T
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    {
      float s2[4] = {0.f, 0.f, 0.f, 0.f};  // one tile alone: two chains of MMAs
      // piece 2k + x of row ri is at (2k + x) ^ ri = 2k ^ (x ^ ri): an address, with bits of k exchanged
      const uint32_t at = ((mi & 1) * 8 + ri) * 128 + (((mi >> 1) ^ ri) << 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t a[4];
        ldsm_x4(((kt + at) ^ ((k & 3) << 5)) + (k >> 2) * HALF_BYTES, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_bf16(NT == 1 && (k & 1) ? s2 : s[n], a, qb[n][k][0], qb[n][k][1]);
      }
      if (NT == 1) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[0][x] += s2[x];
      }
    }
    if (cut) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const int pos = span.len - p.tokens + p.token_of(n * 8 + 2 * t + odd);
#pragma unroll
          for (int e = odd; e < 4; e += 2) {
            const int key = key0 + r + (e >> 1) * 8;
            if (key > pos || (p.window > 0 && key <= pos - p.window && key >= p.sinks)) s[n][e] = -INFINITY;
          }
        }
      // V rows that no row of the sequence sees may hold anything: their P is 0, and so V is made.
      const int key = key0 + lane % CK;  // (a lane half a row)
      if (key >= span.len || (key < span.low && key >= p.sinks)) {
#pragma unroll
        for (int y = 0; y < 8; ++y)
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vt + lane * 128 + y * 16), "r"(0) : "memory");
      }
      fence_proxy_async_smem();  // before the next copy into the stage
      __syncwarp();
    }
    // ---- running softmax, log2 domain
    float top[NT][2], most = NO_MAX;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n][0] = fmaxf(s[n][0], s[n][2]);
      top[n][1] = fmaxf(s[n][1], s[n][3]);
      most = fmax3(most, fmaf(top[n][0], p.scale_log2, -m[n][0]), fmaf(top[n][1], p.scale_log2, -m[n][1]));
    }
    // The lanes' own maxima tell whether any grew past the slack; only then are they joined.
    if (__any_sync(0xffffffffu, most > SLACK)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top[n][0] = fmaxf(top[n][0], __shfl_xor_sync(0xffffffffu, top[n][0], d));
          top[n][1] = fmaxf(top[n][1], __shfl_xor_sync(0xffffffffu, top[n][1], d));
        }
        rescale(n, fmaxf(m[n][0], top[n][0] * p.scale_log2), fmaxf(m[n][1], top[n][1] * p.scale_log2));
      }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float(&x)[4] = s[n];
      x[0] = fast_exp2(fmaf(x[0], p.scale_log2, -m[n][0]));
      x[1] = fast_exp2(fmaf(x[1], p.scale_log2, -m[n][1]));
      x[2] = fast_exp2(fmaf(x[2], p.scale_log2, -m[n][0]));
      x[3] = fast_exp2(fmaf(x[3], p.scale_log2, -m[n][1]));
      pb[n][0] = transpose8x8(pack_bf16x2(x[0], x[1]));
      pb[n][1] = transpose8x8(pack_bf16x2(x[2], x[3]));
    }
    // ---- O^T += V^T P^T
    const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const uint32_t at = ((mi >> 1) * 8 + ri) * 128 + (((mi & 1) ^ ri) << 4);
#pragma unroll
    for (int n = 0; n < NT; ++n) mma_bf16(l[n], ones, pb[n][0], pb[n][1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a[4];
      ldsm_x4_t(((vt + at) ^ ((i & 3) << 5)) + (i >> 2) * HALF_BYTES, a);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16(o[n][i], a, pb[n][0], pb[n][1]);
    }
  }

  // Tile n relative to other maxima.
  __device__ __forceinline__ void rescale(int n, float m0, float m1) {
    const float f0 = fast_exp2(m[n][0] - m0), f1 = fast_exp2(m[n][1] - m1);
    m[n][0] = m0;
    m[n][1] = m1;
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

  // The sums to and from another warp's same lane, for one tile.
  __device__ __forceinline__ void put(int n, float4* to, int lane) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i * 32 + lane] = make_float4(o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
    to[8 * 32 + lane] = make_float4(m[n][0], m[n][1], l[n][0], l[n][1]);
  }
  __device__ __forceinline__ void add(int n, const float4* from, int lane) {
    const float4 ml = from[8 * 32 + lane];
    rescale(n, fmaxf(m[n][0], ml.x), fmaxf(m[n][1], ml.y));
    const float g0 = fast_exp2(ml.x - m[n][0]), g1 = fast_exp2(ml.y - m[n][1]);
    l[n][0] = fmaf(ml.z, g0, l[n][0]);
    l[n][1] = fmaf(ml.w, g1, l[n][1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 v = from[i * 32 + lane];
      o[n][i][0] = fmaf(v.x, g0, o[n][i][0]);
      o[n][i][1] = fmaf(v.y, g1, o[n][i][1]);
      o[n][i][2] = fmaf(v.z, g0, o[n][i][2]);
      o[n][i][3] = fmaf(v.w, g1, o[n][i][3]);
    }
  }
};

// Behind the ring are the sums that half of the block's warps hand over to the other.
constexpr int SUM_BYTES = 9 * 32 * 16;  // of a tile
constexpr int smem_bytes(int tiles) {
  return RING_BYTES + WARPS / 2 * (tiles < 2 ? 2 : tiles) * SUM_BYTES + 1024;  // + alignment to the swizzle's period
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Grid: blocks of WARPS warps, each with a ring and every WARPS-th chunk of the block's.  PAIR: clusters, each with a
// pair (y: sequence, x: head and rank) whose chunks its blocks share; else blocks with equal shares of the line.
template <int NT, bool PAIR>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS_PER_SM) window_decode_kernel(const __grid_constant__ Params p) {
  constexpr int TILE_BYTES = CK * HD * 2, STAGE_BYTES = 2 * TILE_BYTES;  // K or V, and both
  constexpr int STAGES = RING_BYTES / WARPS / STAGE_BYTES;
  using Span = Span<CK>;
  auto span_of = [&](int len) { return decode_window::span_of<CK>(p, len); };
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_all[WARPS * STAGES];
  if (!PAIR) pdl_launch_dependents();  // the join waits for this grid's end before it reads
  const int warp = warp_id(), lane = lane_id();
  const int r = lane >> 2, t = lane & 3;
  const int G = p.group, Hk = p.num_kv_heads;
  uint64_t* const full = full_all + warp * STAGES;
  if (threadIdx.x < WARPS * STAGES) {
    mbar_init(full_all + threadIdx.x, 1);
    fence_mbar_init();
  }
  __syncthreads();

  // ---- this block's run [c0, c0 + count) of the line, and the sequence that c0 lies in (each warp for itself)
  int seq = 0, head = 0, j0 = 0, count = 0;
  int64_t c0 = 0;
  Span span;
  const Shares shares = [&] {
    if constexpr (PAIR) {
      seq = blockIdx.y;
      head = blockIdx.x / p.cluster;
      const int len = __ldg(p.context_lens + seq), rank = (int)cluster_ctarank();
      if (blockIdx.x == 0 && threadIdx.x == 0 && len > p.max_len) record_error(VLC_DEV_ERR_LENGTH);
      span = span_of(len);
      j0 = (int)((int64_t)span.count * rank / p.cluster);
      count = (int)((int64_t)span.count * (rank + 1) / p.cluster) - j0;
      return Shares(0, 1);
    }
    Run<CK> run;
    const Shares all = run_of(p, run, warp, lane);
    seq = run.seq;
    head = run.head;
    j0 = run.j0;
    count = run.count;
    c0 = run.c0;
    span = run.span;
    return all;
  }();
  if (!PAIR && count == 0) return;

  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const ring = smem + warp * (STAGES * STAGE_BYTES);
  float4* const sums = reinterpret_cast<float4*>(smem + RING_BYTES);

  // ---- the issuing side (lane 0): a cursor over the warp's chunks
  const int mine = (count - warp + WARPS - 1) / WARPS;  // chunks warp, warp + WARPS, .. of the run
  Span ahead = span;
  int a_seq = seq, a_head = head, a_j = j0 + warp, issued = 0;
  int a_row = 0, a_index = 0, a_page = -1;  // its row in its page, the page of the sequence, the page's number
  auto load_page = [&]() {
    a_page = a_index < p.table_width ? __ldg(p.block_tables + a_seq * p.table_stride + a_index) : -1;
  };
  auto place = [&]() {  // a_j of another pair, or behind the sinks
    while (a_j >= ahead.count) {  // past the pair's end: on to the pair that it lies in
      a_j -= ahead.count;
      if (++a_head < Hk) continue;
      a_head = 0;
      do {
        ahead = span_of(__ldg(p.context_lens + ++a_seq));  // the chunk follows: so does a sequence with keys
      } while (ahead.count <= 0);
    }
    const int key = (a_j < ahead.first ? a_j : a_j + ahead.jump) * CK;
    a_index = key / p.block_size;
    a_row = key - a_index * p.block_size;
    load_page();
  };
  auto issue = [&]() {  // chunk `issued` of the warp
    const int stage = issued % STAGES;
    uint64_t* bar = full + stage;
    uint8_t* st = ring + stage * STAGE_BYTES;
    int slot = a_page * p.block_size + a_row;
    if ((uint32_t)a_page >= (uint32_t)p.num_pages) {  // the table has no usable page there: recorded, zeros come
      record_error(VLC_DEV_ERR_BLOCK_RANGE);
      slot = p.num_pages * p.block_size;
    }
    mbar_expect_tx(bar, STAGE_BYTES);
    tma_load_5d(st, &p.kv[0], bar, 0, a_head, slot, 0, 0);
    if (!p.joined) tma_load_5d(st + TILE_BYTES, &p.kv[1], bar, 0, a_head, slot, 0, 0);
    if (++issued == mine) return;
    // the next chunk's place, whose page is there by the next call
    a_j += WARPS;
    a_row += WARPS * CK;
    if (a_j >= ahead.count || (a_j >= ahead.first && a_j - WARPS < ahead.first)) {
      place();
    } else if (a_row >= p.block_size) {
      do {
        a_row -= p.block_size;
        ++a_index;
      } while (a_row >= p.block_size);
      load_page();
    }
  };
  if (lane == 0 && mine > 0) {
    place();
    for (int i = 0; i < min(STAGES, mine); ++i) issue();
  }
  // Whether the warp's chunk i came (recorded where it did not).
  auto arrived = [&](int i) {
    const uint32_t parity = (uint32_t)(i / STAGES) & 1u;
    if (mbar_try_wait(full + i % STAGES, parity)) return true;
    return mbar_wait_bounded(full + i % STAGES, parity, VLC_DEV_ERR_TIMEOUT + 26, VLC_WAIT_LIMIT_CYCLES);
  };

  const uint32_t ring_u = smem_u32(ring);
  State<NT> state;
  int i = 0;        // the warp's chunks so far
  bool ok = true;   // its waits so far: a warp that gave up takes no more chunks
  for (int done = 0, first_slot = 0; PAIR || done < count; first_slot = 1) {
    // ---- the pair's chunks [done, done + n) of the run
    const int n = PAIR ? count : min(span.count - j0, count - done);
    // The block with a pair's first chunk notes where its parts will be: one for each block up to that
    // of its last chunk, in slot 0 but for this block's.
    if (!PAIR && j0 == 0 && threadIdx.x == 0)
      p.places[(int64_t)seq * Hk + head] = make_int2((int)blockIdx.x * 2 + first_slot,
                                                     (int)(shares.block_of(c0 + done + span.count - 1) - blockIdx.x) + 1);
    state.start(p, seq, head, r, t);
    const int all0 = span.all0(p), all1 = span.all1(p), all2 = span.all2(p);
    const uint32_t k_off = p.v_first ? TILE_BYTES : 0, v_off = p.v_first ? 0 : TILE_BYTES;
    for (int j = j0 + i * WARPS + warp - done; ok && j < j0 + n; j += WARPS, ++i) {
      if (!__all_sync(0xffffffffu, arrived(i))) {
        ok = false;
        break;
      }
      const int stage = i % STAGES;
      const uint32_t st = ring_u + stage * STAGE_BYTES;
      const int key0 = (j < span.first ? j : j + span.jump) * CK;
      const bool all_seen = j < all0 || (j >= all1 && j < all2);
      state.step(p, st + k_off, st + v_off, key0, !all_seen, span, lane);
      __syncwarp();  // every lane has read the stage
      if (lane == 0 && issued < mine) issue();
    }
    // ---- the warps' sums: the upper half hand theirs over until one warp has them
#pragma unroll
    for (int half = WARPS / 2; half >= 1; half /= 2) {
      float4* const to = sums + (warp % half) * (NT * 9 * 32);
      __syncthreads();
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int x = 0; x < NT; ++x) state.put(x, to + x * (9 * 32), lane);
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int x = 0; x < NT; ++x) state.add(x, to + x * (9 * 32), lane);
      }
    }
    if constexpr (PAIR) {
      // ---- the blocks' sums: each block leaves its in its shared memory and adds some dims of all of them
      if (!ok && lane == 0) {  // (copies still in flight are given more time before the sums take their place)
        for (; i < issued; ++i) arrived(i);
      }
      __syncthreads();
      float4* const own = reinterpret_cast<float4*>(smem);
      if (warp == 0) {
#pragma unroll
        for (int x = 0; x < NT; ++x) state.put(x, own + x * (9 * 32), lane);
      }
      cluster_sync();
      for (int tile = warp; tile * 8 < p.rows; tile += WARPS) {
        const uint32_t at = smem_u32(own + tile * (9 * 32) + lane);
        for (int mt = (int)cluster_ctarank(); mt < 8; mt += p.cluster) {
          float4 ml[8], v[8];
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            if (b >= p.cluster) continue;
            const uint32_t from = mapa_shared(at, b);
            ml[b] = ld_cluster_v4(from + 8 * 32 * 16);
            v[b] = ld_cluster_v4(from + mt * 32 * 16);
          }
          float m0 = NO_MAX, m1 = NO_MAX, l0 = 0.f, l1 = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            if (b >= p.cluster) continue;
            m0 = fmaxf(m0, ml[b].x);
            m1 = fmaxf(m1, ml[b].y);
          }
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            if (b >= p.cluster) continue;
            const float f0 = fast_exp2(ml[b].x - m0), f1 = fast_exp2(ml[b].y - m1);
            l0 = fmaf(ml[b].z, f0, l0);
            l1 = fmaf(ml[b].w, f1, l1);
            o = make_float4(fmaf(v[b].x, f0, o.x), fmaf(v[b].y, f1, o.y), fmaf(v[b].z, f0, o.z), fmaf(v[b].w, f1, o.w));
          }
          const float inv0 = l0 != 0.f ? 1.f / l0 : 0.f, inv1 = l1 != 0.f ? 1.f / l1 : 0.f;  // (NaN stays NaN)
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const int row = tile * 8 + 2 * t + odd, tok = p.token_of(row);
            if (row >= p.rows) continue;
            __nv_bfloat16* dst = p.out + ((int64_t)seq * p.tokens + tok) * p.out_token_stride +
                                 ((int64_t)head * G + row - tok * G) * HD + r + 16 * mt;
            dst[0] = __float2bfloat16(odd ? o.y * inv1 : o.x * inv0);
            dst[8] = __float2bfloat16(odd ? o.w * inv1 : o.z * inv0);
          }
        }
      }
      cluster_sync();  // the others have read this block's sums
      return;
    }
    if (!PAIR && warp == 0) {
      const bool whole = j0 == 0 && n == span.count;
      const int64_t slot = ((int64_t)blockIdx.x * 2 + first_slot) * p.rows;
#pragma unroll
      for (int x = 0; x < NT * 2; ++x) {
        const int nt = x >> 1, odd = x & 1;
        const int row = nt * 8 + 2 * t + odd;
        if (row >= p.rows) continue;
        const float sum = state.l[nt][odd];
        if (whole) {
          const int tok = p.token_of(row);
          const float inv = sum != 0.f ? 1.f / sum : 0.f;  // (NaN stays NaN)
          __nv_bfloat16* dst = p.out + ((int64_t)seq * p.tokens + tok) * p.out_token_stride +
                               ((int64_t)head * G + row - tok * G) * HD + r;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            dst[16 * mt] = __float2bfloat16(state.o[nt][mt][odd] * inv);
            dst[16 * mt + 8] = __float2bfloat16(state.o[nt][mt][2 + odd] * inv);
          }
        } else {
          float* dst = p.parts + (slot + row) * HD + r;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {  // (eight lanes write a sector)
            dst[16 * mt] = state.o[nt][mt][odd];
            dst[16 * mt + 8] = state.o[nt][mt][2 + odd];
          }
          if (r == 0) p.part_ml[slot + row] = make_float2(state.m[nt][odd], sum);
        }
      }
    }
    done += n;
    j0 = 0;
    if (done < count && ++head == Hk) {
      head = 0;
      do {
        span = span_of(__ldg(p.context_lens + ++seq));
      } while (span.count <= 0);
    }
  }
  // Copies still in flight are given more time before the block ends.
  if (!ok && lane == 0) {
    for (; i < issued; ++i) arrived(i);
  }
}

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
  __device__ __forceinline__ uint2 result() const {
    const float inv = l != 0.f ? 1.f / l : 0.f;
    return make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
};

// Joins the parts of the pairs that several blocks shared and writes zeros for empty sequences.  Grid
// (pair, rows).  SPREAD: a block takes one row, its eight warps the row's parts in turn; else eight
// rows, a warp each, which loads eight parts at once.
template <bool SPREAD>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ Params p) {
  constexpr int PARTS = 8;
  __shared__ float4 s_o[8][32];
  __shared__ float2 s_ml[8];
  const int pair = blockIdx.x, warp = warp_id(), lane = lane_id();
  const int seq = pair / p.num_kv_heads, head = pair - seq * p.num_kv_heads;
  const int row = SPREAD ? blockIdx.y : blockIdx.y * 8 + warp;
  const bool empty = __ldg(p.context_lens + seq) <= 0;
  // Every block waits, those with nothing to join too: what follows in the stream may rely on this
  // grid's end for the decode kernel's.
  pdl_wait();
  if (row >= p.rows) return;
  int2 place = make_int2(0, 0);
  if (!empty) place = p.places[pair];
  if ((uint32_t)place.x >= 2u * p.num_blocks || (uint32_t)place.y > (uint32_t)(p.num_blocks - (place.x >> 1)))
    place = make_int2(0, 1);  // (not reached: every pair with keys is noted)
  const int count = place.y;
  if (count == 1) return;  // written by its block
  const int tok = p.token_of(row);
  uint2* const dst = reinterpret_cast<uint2*>(p.out + ((int64_t)seq * p.tokens + tok) * p.out_token_stride +
                                              ((int64_t)head * p.group + row - tok * p.group) * HD) + lane;
  // part i > 0 is in slot 0 of the block i after the first's
  const int64_t first = (int64_t)place.x * p.rows + row, rest = (int64_t)(place.x & ~1) * p.rows + row;
  const float4* const po = reinterpret_cast<const float4*>(p.parts) + lane;
  Joined sum;
  if constexpr (SPREAD) {
#pragma unroll 4
    for (int i = warp; i < count; i += 8) {
      const int64_t s = i == 0 ? first : rest + (int64_t)i * 2 * p.rows;
      const float2 x = p.part_ml[s];
      const float4 v = po[s * (HD / 4)];
      sum.add(x.x, x.y, v);
    }
    s_o[warp][lane] = sum.o;
    if (lane == 0) s_ml[warp] = make_float2(sum.m, sum.l);
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) sum.add(s_ml[w].x, s_ml[w].y, s_o[w][lane]);
    *dst = sum.result();  // (0 parts: zeros)
  } else {
    for (int i0 = 0; i0 < count; i0 += PARTS) {
      float2 x[PARTS];
      float4 v[PARTS];
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        if (i0 + i >= count) continue;
        const int64_t s = i0 + i == 0 ? first : rest + (int64_t)(i0 + i) * 2 * p.rows;
        x[i] = p.part_ml[s];
        v[i] = po[s * (HD / 4)];
      }
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        if (i0 + i < count) sum.add(x[i].x, x[i].y, v[i]);
    }
    *dst = sum.result();
  }
}

// Whether decode_window_wide.cu takes the call: it does where the rows are more than three tiles here.  Below that both
// could; here : there, us (WIDE_ROWS lowered), 16 query and 2 KV heads without a window, caches out of L2.  16 rows: one
// sequence of 500 keys 7.2 : 8.4, of 2000 9.3 : 9.4, of 8000 13.3 : 10.9; eight of 2000 11.4 : 13.3; sixteen of 8000
// 28.4 : 30.1.  24 rows: 8.8 : 8.7, 11.0 : 9.4, 15.9 : 11.4, 13.7 : 13.7, 30.6 : 29.9.  64 sequences under a window (28 and 4
// heads): 14 rows 91.2 : 93.6, 21 rows 95.5 : 95.1.  So up to 16 rows batches are faster here, and 24 are near even but
// for one long sequence.
static bool wide_of(int rows) { return rows > WIDE_ROWS; }

// Most chunks that any sequence has under the host's bound.
static int64_t most_chunks(int CK, int tokens, int max_context_len, int window, int sinks) {
  const int64_t chunks = ((int64_t)max_context_len + CK - 1) / CK;
  if (window == 0) return chunks;
  return std::min(chunks, ((int64_t)sinks + CK - 1) / CK + ((int64_t)window + tokens + CK - 2) / CK + 1);
}

// Blocks of the cluster that takes a pair, or 0 for the line.  The line's shares are even whatever the lengths
// are, and its blocks many where the pairs are few; a pair's cluster saves the second launch.  Pair : line, us, of
// 16 query and 2 KV heads, one token: one sequence of 500 keys 6.3 : 8.0, of 2000 7.8 : 9.9, of 4000 9.9 : 9.6, of
// 8000 14.3 : 10.6; eight of 4000 11.1 : 13.1; sixteen of 8000 26.2 : 30.8; 64 of 4000 46.3 : 48.4.  So a warp takes
// up to 8 chunks, or 16 where the clusters fill half of the GPU (beyond that ragged lengths would leave it idle).
static int cluster_of(int num_seqs, int num_kv_heads, int rows, int tokens, int max_context_len, int window, int sinks,
                      int num_sms) {
  if (wide_of(rows)) return 0;
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads, resident = (int64_t)num_sms * BLOCKS_PER_SM;
  int cluster = 8;
  while (cluster > 1 && pairs * cluster > resident) cluster /= 2;
  const int64_t chunks = most_chunks(CK, tokens, max_context_len, window, sinks);
  const int64_t most = (2 * pairs * cluster >= resident ? 16 : 8) * cluster * WARPS;
  return cluster > 1 && chunks <= most ? cluster : 0;
}

// Blocks of the grid: from host values only, so that it is fixed for graph capture.  A block has at least
// MIN_CHUNKS for each of its warps: few chunks, but fewer parts to join.
constexpr int MIN_CHUNKS = 2;
static int grid_blocks(int num_seqs, int num_kv_heads, int rows, int tokens, int max_context_len, int window, int sinks,
                       int num_sms) {
  const bool wide = wide_of(rows);
  const int64_t chunks = most_chunks(wide ? WIDE_CHUNK : CK, tokens, max_context_len, window, sinks);
  const int least = wide ? 1 : MIN_CHUNKS * WARPS;
  const int64_t most = (num_seqs * num_kv_heads * chunks + least - 1) / least;
  return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)num_sms * (wide ? 1 : BLOCKS_PER_SM), most));
}

static int64_t workspace_bytes_for(int64_t blocks, int rows, int64_t pairs) {
  return blocks * 2 * rows * (HD + 2) * (int64_t)sizeof(float) + pairs * (int64_t)sizeof(int2);
}

// Bounds of the sizes that both entry points take.
static bool sizes_ok(int num_seqs, int tokens, int num_heads, int num_kv_heads, int max_context_len, int window,
                     int sinks) {
  return num_seqs >= 0 && num_seqs <= 65535 && tokens > 0 && num_heads > 0 && num_kv_heads > 0 &&
         num_heads % num_kv_heads == 0 && num_kv_heads <= 65535 && max_context_len >= 0 &&
         max_context_len <= (1 << 30) && window >= 0 && sinks >= 0 && window <= (1 << 30) && sinks <= (1 << 30) &&
         (int64_t)num_seqs * num_kv_heads <= 0x7fffffff;
}

template <int NT>
static int launch(const Params& p, cudaStream_t st) {
  static std::atomic<uint64_t> smem[2];
  const bool pair = p.cluster > 0;
  const auto kernel = pair ? window_decode_kernel<NT, true> : window_decode_kernel<NT, false>;
  if (ensure_dynamic_smem((const void*)kernel, smem_bytes(NT), smem[pair]) != VLC_OK) return VLC_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = pair ? dim3(p.cluster * p.num_kv_heads, p.num_seqs) : dim3(p.num_blocks);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem_bytes(NT);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pair ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}

}  // namespace decode_window
}  // namespace vlc

using namespace vlc;
using namespace vlc::decode_window;

extern "C" int64_t vlc_decode_window_workspace_size(int num_seqs, int num_tokens, int num_heads, int num_kv_heads,
                                                    int max_context_len, int window, int sinks) {
  if (num_seqs <= 0 || !sizes_ok(num_seqs, num_tokens, num_heads, num_kv_heads, max_context_len, window, sinks)) return 0;
  const int64_t rows = (int64_t)num_heads / num_kv_heads * num_tokens;
  if (rows > MAX_ROWS) return 0;
  const int sms = vlc_num_sms();
  max_context_len = std::max(1, max_context_len);
  if (cluster_of(num_seqs, num_kv_heads, (int)rows, num_tokens, max_context_len, window, sinks, sms)) return 0;
  const int blocks = grid_blocks(num_seqs, num_kv_heads, (int)rows, num_tokens, max_context_len, window, sinks, sms);
  return workspace_bytes_for(blocks, (int)rows, (int64_t)num_seqs * num_kv_heads);
}

extern "C" int vlc_decode_attn_window(const void* q, int64_t q_token_stride, int num_seqs, int num_tokens,
                                      int num_heads, const void* k_cache, const void* v_cache, int64_t num_pages,
                                      int block_size, int num_kv_heads, int head_dim, const int32_t* block_tables,
                                      int64_t block_table_stride, int block_table_width, const int32_t* context_lens,
                                      int max_context_len, int window, int sinks, float softmax_scale, void* out,
                                      int64_t out_token_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes_ok(num_seqs, num_tokens, num_heads, num_kv_heads, max_context_len, window, sinks) || block_table_width < 0)
    return VLC_ERR_SHAPE;
  if (head_dim != HD || block_size <= 0 || block_size % MIN_BLOCK != 0) return VLC_ERR_UNSUPPORTED;
  const int G = num_heads / num_kv_heads;
  if ((int64_t)G * num_tokens > MAX_ROWS || !std::isfinite(softmax_scale)) return VLC_ERR_UNSUPPORTED;
  if (num_seqs == 0) return VLC_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out) return VLC_ERR_NULL;
  if (q_token_stride % 8 || out_token_stride % 8 || q_token_stride < (int64_t)num_heads * HD ||
      out_token_stride < (int64_t)num_heads * HD || block_table_stride < block_table_width)
    return VLC_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return VLC_ERR_ALIGN;
  if (num_pages <= 0 || num_pages > 0x7fffffff / block_size) return VLC_ERR_SHAPE;
  max_context_len = std::max(1, max_context_len);
  const int sms = vlc_num_sms(), rows = G * num_tokens;
  const int blocks = grid_blocks(num_seqs, num_kv_heads, rows, num_tokens, max_context_len, window, sinks, sms);
  const int cluster = cluster_of(num_seqs, num_kv_heads, rows, num_tokens, max_context_len, window, sinks, sms);
  if (!cluster) {
    if (!workspace || workspace_bytes < workspace_bytes_for(blocks, rows, (int64_t)num_seqs * num_kv_heads))
      return VLC_ERR_WORKSPACE;
    if (!aligned16(workspace)) return VLC_ERR_ALIGN;
  }

  const bool wide = wide_of(rows);
  Params p;
  const uint8_t* caches[2] = {(const uint8_t*)k_cache, (const uint8_t*)v_cache};
  p.v_first = !wide && caches[1] < caches[0];
  if (p.v_first) std::swap(caches[0], caches[1]);
  const uint64_t apart = (uint64_t)(caches[1] - caches[0]);
  p.joined = !wide && apart > 0 && apart < 1ull << 40;  // as a tensor map's strides may be
  if (!p.joined && p.v_first) {
    std::swap(caches[0], caches[1]);
    p.v_first = false;
  }
  const uint64_t slots = (uint64_t)num_pages * block_size, row = (uint64_t)num_kv_heads * HD * 2;
  for (int i = 0; i < (p.joined ? 1 : 2); ++i) {
    const uint64_t both = p.joined ? 2 : 1;
    const uint64_t dims[5] = {64, (uint64_t)num_kv_heads, slots, 2, both};
    const uint64_t strides[4] = {HD * 2, row, 128, p.joined ? apart : 256};
    const uint32_t box[5] = {64, 1, (uint32_t)(wide ? WIDE_BOX : CK), wide ? 1u : 2u, (uint32_t)both};
    if (encode_tmap_bf16(&p.kv[i], caches[i], wide ? 4 : 5, dims, strides, box, 128) != VLC_OK) return VLC_ERR_CUDA;
  }
  p.q = (const __nv_bfloat16*)q;
  p.q_token_stride = q_token_stride;
  p.block_tables = block_tables;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.block_size = block_size;
  p.num_pages = (int)num_pages;
  p.context_lens = context_lens;
  p.num_seqs = num_seqs;
  p.max_len = max_context_len;
  p.tokens = num_tokens;
  p.window = window;
  p.sinks = window > 0 ? sinks : 0;
  p.group = G;
  p.group_inverse = (65536 + G - 1) / G;
  p.num_kv_heads = num_kv_heads;
  p.rows = rows;
  p.cluster = cluster;
  p.scale_log2 = std::max(std::fabs(softmax_scale) * 1.4426950408889634f, std::numeric_limits<float>::min());
  p.q_flip = softmax_scale < 0.f ? 0x80008000u : 0u;
  p.out = (__nv_bfloat16*)out;
  p.out_token_stride = out_token_stride;
  p.num_blocks = blocks;
  p.parts = (float*)workspace;
  p.part_ml = (float2*)(p.parts + (int64_t)blocks * 2 * rows * HD);
  p.places = (int2*)(p.part_ml + (int64_t)blocks * 2 * rows);

  cudaStream_t st = (cudaStream_t)stream;
  const int rc = wide ? launch_wide(p, st) : rows <= 8 ? launch<1>(p, st) : rows <= 16 ? launch<2>(p, st) : launch<3>(p, st);
  if (rc != VLC_OK || cluster) return rc;
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads;
  const bool spread = blocks / pairs + 1 > 10;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)pairs, spread ? rows : (rows + 7) / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, spread ? window_join_kernel<true> : window_join_kernel<false>, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return VLC_ERR_CUDA;
  }
  return VLC_OK;
}
