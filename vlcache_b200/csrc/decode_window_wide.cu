// Paged decode attention of many rows a KV head (drafted tokens x query heads), with a window and sinks: the line of
// decode_window.cu on tcgen05 products.
//
//   S^T [128 keys x N rows] = K Q^T,   O^T [128 dims x N rows] += V^T P^T
//
// A chunk is 128 keys, and the keys and dims take the accumulators' 128 lanes, so that the products' time goes with
// the rows (N = 32 .. 128 columns) where a tile of 128 rows would be empty for the most part.  K is read K-major, V
// as it lies in the cache, MN-major.  A softmax thread has one key and half of the rows: the maxima are lazy and
// shared by all keys of a row, so that a step has no reductions over keys but for one vote whether any score grew past
// its row's maximum by 2^8; P goes to shared memory as the second product's B operand, 16 bytes a store.  Roles (a
// block an SM, 12 warps): K and V copies, products, Q, softmax (8).  The next chunk's S is made while this one's
// softmax runs; S, O and Q have two buffers each, so that the next pair starts while this one's O is written.
//
// P is rounded to bf16 as an operand has to be, and its sums are of the rounded values; scores, maxima, sums and O are
// fp32.
//
// Measured (64 sequences of 2700 .. 10700 keys, window 4096, 28 query and 4 KV heads; floor 83 us): 28 rows 93 .. 95 us by
// the GPU, 35 95 .. 97, 56 100 .. 102, 63 102, 91 121, 112 178.  Up to 48 rows HBM bounds it: 4.5 us until the first S, the
// join and the last chunks 5, between them 0.97 of the floor (a ring of 4 slots instead of 5 costs 0.5).  Copies of 32
// keys: of 64, a window's ends waste more (35 rows 97.9 against 96.6), of 16 the copies count (112); chunks that lie in a
// page in one copy: no change.  With more rows the softmax's time counts (2000 cycles a chunk of 64 rows), then
// registers: a thread's sums of P.  Tried: the exponentials or the products left out, for a time only: no change, so
// the chains of waits count and not the pipes; pages' numbers four chunks ahead, unrolled: 98 and 104 for 35 and 56
// rows (more code, which the roles' caches feel); P and the slow path in one loop, one copy of each: 99 and 107; four
// shares of the rows: no change for 56, 127 for 91, but 178 instead of 195 for 112.  Rows' output offsets and 1 / sum made
// once, not by each thread, and maxima and sums over lanes that halve the columns: 112 -> 96.
#include <algorithm>
#include <cmath>

#include "decode_window.cuh"
#include "runtime.h"

namespace vlc {
namespace decode_window {
namespace wide {

constexpr int CK = WIDE_CHUNK;
constexpr int FIRST_SOFTMAX = 4;              // warp; four for each share of the rows from there on
constexpr int HALF_BYTES = CK * 128;          // 64 dims of a chunk's keys
constexpr int TILE_BYTES = 2 * HALF_BYTES;    // K or V
constexpr uint32_t DESC_HI = umma_desc_sw128_hi(1024);

template <int N>
struct Layout {
  static constexpr int SIDES = N <= 96 ? 2 : 4;  // shares of the rows: a thread's sums of P are registers
  static constexpr int THREADS = (FIRST_SOFTMAX + 4 * SIDES) * 32;
  static constexpr int SLOTS = N <= 64 ? 5 : 4;  // of the ring of K and V
  static constexpr int Q_BUFFERS = N <= 96 ? 2 : 1, Q_BYTES = N * HD * 2;
  static constexpr int P_BYTES = (N + 63) / 64 * HALF_BYTES;  // 64 rows of each key, then the next 64
  static constexpr int Q = SLOTS * TILE_BYTES, P = Q + Q_BUFFERS * Q_BYTES;
  static constexpr int ROWS = P + P_BYTES;       // where a row's output is, from the pair's on
  static constexpr int FLOATS = ROWS + N * 8;    // m[N], factor[N], tops[SIDES][4 warps][N / SIDES]
  static constexpr int BARS = FLOATS + 6 * N * 4;
  static constexpr int NUM_BARS = 2 * SLOTS + 13;
  static constexpr int MISC = BARS + NUM_BARS * 8;
  static constexpr int BYTES = MISC + 16 + 1024;  // + alignment to the swizzle's period
  static_assert(BYTES <= 232448, "shared memory");
};

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Whether `yes` holds in any thread of the named barrier.
__device__ __forceinline__ bool named_bar_any(int id, int threads, bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.b32 a, %3, 0;\n\t"
      "barrier.cta.red.or.pred b, %1, %2, a;\n\t"
      "selp.b32 %0, 1, 0, b;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(threads), "r"((uint32_t)yes)
      : "memory");
  return any != 0;
}

template <int NC>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[NC]) {
#pragma unroll
  for (int c = 0; c + 16 <= NC; c += 16) tmem_ld16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
  if constexpr (NC % 16 != 0) tmem_ld8(taddr + NC - 8, *reinterpret_cast<uint32_t(*)[8]>(&r[NC - 8]));
  tmem_wait_ld();
}

// Each column's union over the warp's lanes, to to[column]: the lanes halve the columns among them three times.
template <int NC, typename V, typename F>
__device__ __forceinline__ void columns_over_warp(V&& value, F&& join, float* to, int lane) {
  float v[NC / 2];
#pragma unroll
  for (int c = 0; c < NC / 2; ++c) {
    const float low = value(c), high = value(c + NC / 2);
    v[c] = join(lane & 16 ? high : low, __shfl_xor_sync(0xffffffffu, lane & 16 ? low : high, 16));
  }
#pragma unroll
  for (int c = 0; c < NC / 4; ++c)
    v[c] = join(lane & 8 ? v[c + NC / 4] : v[c], __shfl_xor_sync(0xffffffffu, lane & 8 ? v[c] : v[c + NC / 4], 8));
#pragma unroll
  for (int c = 0; c < NC / 8; ++c)
    v[c] = join(lane & 4 ? v[c + NC / 8] : v[c], __shfl_xor_sync(0xffffffffu, lane & 4 ? v[c] : v[c + NC / 8], 4));
  to += ((lane & 16 ? 4 : 0) + (lane & 8 ? 2 : 0) + (lane & 4 ? 1 : 0)) * (NC / 8);
#pragma unroll
  for (int c = 0; c < NC / 8; ++c) {
    v[c] = join(v[c], __shfl_xor_sync(0xffffffffu, v[c], 2));
    v[c] = join(v[c], __shfl_xor_sync(0xffffffffu, v[c], 1));
    if (lane % 4 == 0) to[c] = v[c];
  }
}

// Place in the ring of chunk i of n: K0, K1, V0, K2, V1, ..: the order in which they are wanted.
__device__ __forceinline__ int k_load(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int v_load(int i, int n) { return i + 1 < n ? 2 * i + 2 : 2 * n - 1; }

template <int N>  // columns: rows, padded
__global__ void __launch_bounds__(Layout<N>::THREADS, 1) window_decode_wide_kernel(const __grid_constant__ Params p) {
  using L = Layout<N>;
  constexpr int SIDES = L::SIDES, THREADS = L::THREADS;
  constexpr int NC = N / SIDES;  // of a softmax thread
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, N, false, false);
  constexpr uint32_t IDESC_O = umma_idesc_bf16(128, N, true, true);
  extern __shared__ uint8_t smem_raw[];
  pdl_launch_dependents();  // the join waits for this grid's end before it reads
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* const empty = full + L::SLOTS;
  uint64_t* const q_full = empty + L::SLOTS;  // two of each from here on
  uint64_t* const q_empty = q_full + 2;
  uint64_t* const s_full = q_full + 4;
  uint64_t* const s_empty = q_full + 6;
  uint64_t* const o_empty = q_full + 8;
  uint64_t* const p_full = q_full + 10;
  uint64_t* const p_empty = q_full + 11;
  uint64_t* const drain = q_full + 12;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const int warp = warp_id(), lane = lane_id();

  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int x = 0; x < 2 * L::SLOTS; ++x) mbar_init(full + x, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(q_full + x, 64);
      mbar_init(q_empty + x, 1);
      mbar_init(s_full + x, 1);
      mbar_init(s_empty + x, 4 * SIDES);
      mbar_init(o_empty + x, 4 * SIDES);
    }
    mbar_init(p_full, 4 * SIDES);
    mbar_init(p_empty, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  int64_t* const row_at = reinterpret_cast<int64_t*>(smem + L::ROWS);
  if (threadIdx.x >= THREADS - N) {
    const int row = threadIdx.x - (THREADS - N), tok = p.token_of(row);
    row_at[row] = tok * p.out_token_stride + (row - tok * p.group) * HD;
  }
  Run<CK> run;
  const Shares shares = run_of(p, run, warp, lane);
  const int count = run.count;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S: columns [0, N) and [N, 2N), O: [2N, 3N) and [3N, 4N)
  auto wait = [&](uint64_t* bar, int phase, int role) {
    return wait_or_abort(bar, (uint32_t)phase & 1u, VLC_DEV_ERR_TIMEOUT + role, abort_flag);
  };
  // By a warp that leaves its role where it gave up: its lanes leave together or not at all.
  auto warp_wait = [&](uint64_t* bar, int phase, int role) {
    return warp_wait_or_abort(bar, (uint32_t)phase & 1u, VLC_DEV_ERR_TIMEOUT + role, abort_flag);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ K and V copies: a lane each box of keys
    constexpr int BOXES = CK / WIDE_BOX;
    static_assert(MIN_BLOCK % WIDE_BOX == 0, "a box lies in one page");
    struct Entry {
      int page, row, head;
      bool seen;  // some row sees some key of the box
    };
    Run<CK> at = run;
    int left = count;
    auto fetch = [&]() {  // the box of the cursor's chunk, and on
      const int j = at.j0, key = (j < at.span.first ? j : j + at.span.jump) * CK + lane * WIDE_BOX;
      const int index = key / p.block_size;
      Entry e{-1, key - index * p.block_size, at.head,
              key < at.span.len && (key + WIDE_BOX > at.span.low || key < p.sinks)};
      if (lane < BOXES && e.seen && index < p.table_width)
        e.page = __ldg(p.block_tables + at.seq * p.table_stride + index);
      if (--left > 0 && ++at.j0 == at.span.count) at.next_pair(p);
      return e;
    };
    int loads = 0;
    auto issue = [&](const CUtensorMap* map, const Entry& e) {
      const int slot = loads % L::SLOTS;
      const bool empty_now = loads < L::SLOTS || wait(empty + slot, loads / L::SLOTS - 1, 27);
      if (lane == 0 && empty_now) mbar_expect_tx(full + slot, TILE_BYTES);
      if (!__all_sync(0xffffffffu, empty_now)) return false;  // (a lane alone may have given up: all leave, or none)
      if (lane < BOXES) {
        int row = e.page * p.block_size + e.row;
        if ((uint32_t)e.page >= (uint32_t)p.num_pages) {  // no usable page there: zeros come
          if (e.seen) record_error(VLC_DEV_ERR_BLOCK_RANGE);
          row = p.num_pages * p.block_size;
        }
        uint8_t* const to = smem + slot * TILE_BYTES + lane * WIDE_BOX * 128;
        tma_load_4d(to, map, full + slot, 0, e.head, row, 0);
        tma_load_4d(to + HALF_BYTES, map, full + slot, 0, e.head, row, 1);
      }
      ++loads;
      return true;
    };
    bool ok = true;
    if (count > 0) {
      Entry now = fetch(), next = now;
      if (count > 1) next = fetch();
      ok = issue(&p.kv[0], now);
      for (int i = 0; ok && i < count; ++i) {
        Entry behind = next;
        if (i + 2 < count) behind = fetch();
        ok = (i + 1 >= count || issue(&p.kv[0], next)) && issue(&p.kv[1], now);
        now = next;
        next = behind;
      }
    }
    // Where a role gave up, the copies in flight are given more time before the block ends.
    if (!ok || *abort_flag) drain_ring(full, loads, L::SLOTS, VLC_DEV_ERR_TIMEOUT + 28);
  } else if (warp == 1) {
    // ------------------------------------------------------------ products, by one lane
    if (lane == 0 && count > 0) {
      const uint32_t ring = umma_desc_sw128_lo(smem_u32(smem), 16);
      const uint32_t ring_v = umma_desc_sw128_lo(smem_u32(smem), HALF_BYTES);
      const uint32_t q_at = umma_desc_sw128_lo(smem_u32(smem + L::Q), 16);
      const uint32_t p_at = umma_desc_sw128_lo(smem_u32(smem + L::P), HALF_BYTES);
      // Cursors over the run: of S (one chunk ahead) and of O.
      Run<CK> at = run;
      int left = min(at.span.count - at.j0, count), s_pair = 0;  // chunks of S's pair that are left
      bool s_first = true;
      auto product_s = [&](int i) {
        const int load = k_load(i), slot = load % L::SLOTS, b = s_pair % L::Q_BUFFERS;
        if (s_first && !wait(q_full + b, s_pair / L::Q_BUFFERS, 29)) return false;
        if (!wait(full + slot, load / L::SLOTS, 30) || (i >= 2 && !wait(s_empty + (i & 1), i / 2 - 1, 31))) return false;
        tc_fence_after();
        const uint32_t a = ring + slot * (TILE_BYTES >> 4), q = q_at + b * (L::Q_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          umma_ss_w(tmem + (i & 1) * N, a + (uint32_t)(((k >> 2) * HALF_BYTES + (k & 3) * 32) >> 4), DESC_HI,
                    q + (uint32_t)(((k >> 2) * (N * 128) + (k & 3) * 32) >> 4), DESC_HI, IDESC_S, k > 0 ? 1u : 0u);
        umma_commit(s_full + (i & 1));
        umma_commit(empty + slot);
        s_first = --left == 0;
        if (s_first) {
          umma_commit(q_empty + b);
          ++s_pair;
          if (i + 1 < count) {
            at.next_pair(p);
            left = min(at.span.count, count - i - 1);
          }
        }
        return true;
      };
      int o_pair = 0, o_left = left;
      Run<CK> o_run = run;
      bool o_first = true, ok = product_s(0);
      for (int i = 0; ok && i < count; ++i) {
        if (i + 1 < count && !product_s(i + 1)) break;
        const int load = v_load(i, count), slot = load % L::SLOTS, b = o_pair & 1;
        if (!wait(p_full, i, 32) || !wait(full + slot, load / L::SLOTS, 30) ||
            (o_first && o_pair >= 2 && !wait(o_empty + b, o_pair / 2 - 1, 33)))
          break;
        tc_fence_after();
        const uint32_t a = ring_v + slot * (TILE_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < CK / 16; ++k)
          umma_ss_w(tmem + (2 + b) * N, a + (uint32_t)((k * 2048) >> 4), DESC_HI, p_at + (uint32_t)((k * 2048) >> 4),
                    DESC_HI, IDESC_O, o_first && k == 0 ? 0u : 1u);
        umma_commit(p_empty);
        umma_commit(empty + slot);
        o_first = --o_left == 0;
        if (o_first) {
          ++o_pair;
          if (i + 1 < count) {
            o_run.next_pair(p);
            o_left = min(o_run.span.count, count - i - 1);
          }
        }
      }
      umma_commit(drain);  // every product is done before the block ends
      mbar_wait_bounded(drain, 0, VLC_DEV_ERR_TIMEOUT + 34, VLC_WAIT_LIMIT_CYCLES);
    }
  } else if (warp < FIRST_SOFTMAX) {
    // ------------------------------------------------------------ Q: 16 lanes a row
    const int row0 = (warp - 2) * 2 + (lane >> 4), piece = lane & 15;
    Run<CK> at = run;
    for (int done = 0, pair = 0; done < count; ++pair) {
      const int b = pair % L::Q_BUFFERS;
      if (pair >= L::Q_BUFFERS && !warp_wait(q_empty + b, pair / L::Q_BUFFERS - 1, 35)) break;
      uint8_t* const to = smem + L::Q + b * L::Q_BYTES + (piece >> 3) * (N * 128);
      constexpr int LOADS = N <= 64 ? N / 4 : 8;  // at once
#pragma unroll
      for (int first = 0; first < N; first += LOADS * 4) {
        uint4 v[LOADS];
#pragma unroll
        for (int x = 0; x < LOADS; ++x) {
          const int row = row0 + first + x * 4, tok = p.token_of(row);
          v[x] = make_uint4(0, 0, 0, 0);
          if (row < p.rows)
            v[x] = __ldg(reinterpret_cast<const uint4*>(p.q + ((int64_t)at.seq * p.tokens + tok) * p.q_token_stride +
                                                        ((int64_t)at.head * p.group + row - tok * p.group) * HD) + piece);
        }
#pragma unroll
        for (int x = 0; x < LOADS; ++x) {
          const int row = row0 + first + x * 4;
          const uint32_t u[4] = {v[x].x ^ p.q_flip, v[x].y ^ p.q_flip, v[x].z ^ p.q_flip, v[x].w ^ p.q_flip};
          bool huge = false;
#pragma unroll
          for (int y = 0; y < 4; ++y) huge |= (u[y] & 0x7fffu) >= 0x7f80u || (u[y] & 0x7fff0000u) >= 0x7f800000u;
          // A row with an infinity has scores of +-infinity or NaN only, whose softmax is NaN: it becomes NaN here.
          const uint32_t any = __ballot_sync(0xffffffffu, huge) >> (lane & 16) & 0xffffu;
          const uint32_t spoil = any ? 0x7fff7fffu : 0u;
          *reinterpret_cast<uint4*>(to + row * 128 + (((piece & 7) ^ (row & 7)) << 4)) =
              make_uint4(u[0] | spoil, u[1] | spoil, u[2] | spoil, u[3] | spoil);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full + b);
      done += min(at.span.count - at.j0, count - done);
      if (done < count) at.next_pair(p);
    }
  } else {
    // ------------------------------------------------------------ softmax: a thread has a key, and a share of the rows.
    // After a wait that gave up a thread goes on through all chunks (later waits end at once), so that the named
    // barriers stay matched.
    const int side = (warp - FIRST_SOFTMAX) >> 2, quarter = warp & 3, key_lane = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lanes + side * NC, o_at = lanes + 2 * N + side * NC;
    float* const floats = reinterpret_cast<float*>(smem + L::FLOATS);
    float* const ms = floats + side * NC;
    float* const fs = floats + N + side * NC;
    float* const tops = floats + 2 * N + side * (4 * NC);
    uint8_t* const p_row = smem + L::P + key_lane * 128;
    const int bar = 1 + side, row0 = side * NC;
    auto arrive = [&](uint64_t* b) {  // for the warp
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    Run<CK> at = run;
    int i = 0;
    for (int done = 0, pair = 0; done < count; ++pair) {
      const Span<CK>& span = at.span;
      const int n = min(span.count - at.j0, count - done);
      const int slot = (int)blockIdx.x * 2 + (pair > 0 ? 1 : 0);
      const bool whole = at.j0 == 0 && n == span.count;
      if (at.j0 == 0 && threadIdx.x == FIRST_SOFTMAX * 32)  // where the pair's parts will be
        p.places[(int64_t)at.seq * p.num_kv_heads + at.head] =
            make_int2(slot, (int)(shares.block_of(run.c0 + done + span.count - 1) - blockIdx.x) + 1);
      const int all0 = span.all0(p), all1 = span.all1(p), all2 = span.all2(p);
      const uint32_t o_now = o_at + (pair & 1) * N;
      float l[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) l[c] = 0.f;
      for (int j = at.j0; j < at.j0 + n; ++j, ++i) {
        const bool fresh = j == at.j0;
        wait(s_full + (i & 1), i / 2, 36);
        tc_fence_after();
        uint32_t s[NC];
        tmem_load(s_at + (i & 1) * N, s);
        tc_fence_before();
        arrive(s_empty + (i & 1));
        const bool cut = !(j < all0 || (j >= all1 && j < all2));
        const int key = (j < span.first ? j : j + span.jump) * CK + key_lane;
        if (cut) {  // rows of the tokens [a, a + window) see the key, and the later ones where it is a sink
          const int a = key - (span.len - p.tokens);
          const int lo = min(max(a, 0), MAX_ROWS) * p.group - row0;
          const int hi = (p.window == 0 || key < p.sinks ? MAX_ROWS : min(max(a + p.window, 0), MAX_ROWS)) * p.group - row0;
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (c < lo || c >= hi) s[c] = 0xff800000u;
        }
        // ---- P, rounded, and whether a score is past its row's maximum
        uint32_t packed[NC / 2];
        float most = NO_MAX;
        auto make_p = [&]() {
#pragma unroll
          for (int c = 0; c < NC; c += 4) {
            const float4 m = *reinterpret_cast<const float4*>(ms + c);
            const float x0 = fmaf(__uint_as_float(s[c]), p.scale_log2, -m.x);
            const float x1 = fmaf(__uint_as_float(s[c + 1]), p.scale_log2, -m.y);
            const float x2 = fmaf(__uint_as_float(s[c + 2]), p.scale_log2, -m.z);
            const float x3 = fmaf(__uint_as_float(s[c + 3]), p.scale_log2, -m.w);
            most = fmax3(fmax3(most, x0, x1), x2, x3);
            packed[c / 2] = pack_bf16x2(fast_exp2(x0), fast_exp2(x1));
            packed[c / 2 + 1] = pack_bf16x2(fast_exp2(x2), fast_exp2(x3));
          }
        };
        bool grown = fresh;
        if (!fresh) {
          make_p();
          grown = named_bar_any(bar, 128, most > SLACK);
        }
        bool product_done = i == 0;  // the one before, which reads P and adds to O
        if (grown) {
          columns_over_warp<NC>([&](int c) { return __uint_as_float(s[c]); }, [](float a, float b) { return fmaxf(a, b); },
                                tops + quarter * NC, lane);
          named_bar_sync(bar, 128);
          if (key_lane < NC) {
            const float top = fmaxf(fmaxf(tops[key_lane], tops[NC + key_lane]),
                                    fmaxf(tops[2 * NC + key_lane], tops[3 * NC + key_lane]));
            const float before = fresh ? NO_MAX : ms[key_lane], now = fmaxf(before, top * p.scale_log2);
            ms[key_lane] = now;
            fs[key_lane] = fast_exp2(before - now);
          }
          named_bar_sync(bar, 128);
          if (!fresh) {
            wait(p_empty, i - 1, 37);
            product_done = true;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < NC; c += 8) {
              uint32_t o[8];
              tmem_ld8(o_now + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float f = fs[c + x];
                l[c + x] *= f;
                o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              }
              tmem_st8(o_now + c, o);
            }
            tmem_wait_st();
            tc_fence_before();
          }
          make_p();
        }
#pragma unroll
        for (int c = 0; c < NC; c += 2) {
          l[c] += __uint_as_float(packed[c / 2] << 16);
          l[c + 1] += __uint_as_float(packed[c / 2] & 0xffff0000u);
        }
        if (!product_done) wait(p_empty, i - 1, 37);
#pragma unroll
        for (int c = 0; c < NC; c += 8) {
          const int piece = (row0 + c) >> 3;
          *reinterpret_cast<uint4*>(p_row + (piece >> 3) * HALF_BYTES + (((piece & 7) ^ (key_lane & 7)) << 4)) =
              make_uint4(packed[c / 2], packed[c / 2 + 1], packed[c / 2 + 2], packed[c / 2 + 3]);
        }
        if (cut) {
          // V rows that no row of the sequence sees may hold anything: their P is 0, and so V is made.
          const int load = v_load(i, count), ring_slot = load % L::SLOTS;
          wait(full + ring_slot, load / L::SLOTS, 38);
          if (key >= span.len || (key < span.low && key >= p.sinks)) {
            uint4* const v = reinterpret_cast<uint4*>(smem + ring_slot * TILE_BYTES + side * 2 / SIDES * HALF_BYTES +
                                                          key_lane * 128 + side % (SIDES / 2) * (256 / SIDES));
#pragma unroll
            for (int x = 0; x < 16 / SIDES; ++x) v[x] = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        arrive(p_full);
      }
      // ---- the pair's sums of P over the keys, then its O
      columns_over_warp<NC>([&](int c) { return l[c]; }, [](float a, float b) { return a + b; }, tops + quarter * NC, lane);
      named_bar_sync(bar, 128);
      const int64_t part = (int64_t)slot * p.rows + row0;
      if (key_lane < NC) {
        const float sum = (tops[key_lane] + tops[NC + key_lane]) + (tops[2 * NC + key_lane] + tops[3 * NC + key_lane]);
        fs[key_lane] = sum != 0.f ? 1.f / sum : 0.f;  // (NaN stays NaN)
        if (!whole && row0 + key_lane < p.rows) p.part_ml[part + key_lane] = make_float2(ms[key_lane], sum);
      }
      named_bar_sync(bar, 128);
      wait(p_empty, i - 1, 37);
      tc_fence_after();
      uint32_t o[NC];
      tmem_load(o_now, o);
      tc_fence_before();
      arrive(o_empty + (pair & 1));
      const int rows = min(NC, p.rows - row0);
      if (whole) {
        __nv_bfloat16* const out =
            p.out + (int64_t)at.seq * p.tokens * p.out_token_stride + (int64_t)at.head * p.group * HD + key_lane;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c < rows) out[row_at[row0 + c]] = __float2bfloat16(__uint_as_float(o[c]) * fs[c]);
      } else {
        float* const parts = p.parts + part * HD + key_lane;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c < rows) parts[c * HD] = __uint_as_float(o[c]);
      }
      done += n;
      if (done < count) at.next_pair(p);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int N>
static int launch(const Params& p, cudaStream_t st) {
  static std::atomic<uint64_t> smem{0};
  const auto kernel = window_decode_wide_kernel<N>;
  if (ensure_dynamic_smem((const void*)kernel, Layout<N>::BYTES, smem) != VLC_OK) return VLC_ERR_CUDA;
  kernel<<<p.num_blocks, Layout<N>::THREADS, Layout<N>::BYTES, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? VLC_OK : VLC_ERR_CUDA;
}

}  // namespace wide

int launch_wide(const Params& p, cudaStream_t st) {
  if (p.rows <= 32) return wide::launch<32>(p, st);
  if (p.rows <= 48) return wide::launch<48>(p, st);
  if (p.rows <= 64) return wide::launch<64>(p, st);
  if (p.rows <= 96) return wide::launch<96>(p, st);
  return wide::launch<128>(p, st);
}

}  // namespace decode_window
}  // namespace vlc
