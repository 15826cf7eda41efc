// Sliding-window attention on the fifth-generation tensor cores, for float16 and bfloat16 rows
// that are whole 16-byte vectors. The mathematics and the masks are those of nt_attention.cu.
//
// One warp of a block copies tiles, one issues the products, the others (16; 8 where two blocks share
// an SM) compute. Scores accumulate in TMEM; the weights go back to TMEM over them as 16-bit values and are the first
// operand of the second product. The backward is two passes of one kernel, each with S and dP
// computed again; sums that cross blocks exist only for split key blocks and are added in order
// afterwards.
//
// Roundings below 32 bits: the weights and dS are rounded to the inputs' type because the second
// products take their operand in it; every sum, maximum and statistic is float32. Where a row sees
// kFineKeys keys or fewer, dS is what is left of nearly equal numbers (P dP - P delta), and its
// rounding would show: there it goes in as the sum of two 16-bit values, in two products (window 2:
// dq has 1.15 times the error of rounding the exact gradient instead of 1.53; the backward of 2 x 4096
// tokens of 16 heads of 128 takes 160 us instead of 144; from 16 keys on the ratio is below 1.5 with
// one value).
// Three kinds of calls have such rows in number: narrow windows; batches with lengths, whose queries past
// a sequence's end see what is left of it (8 sequences up to 777 tokens, window 100: 1.15 instead of
// 1.53, 50 us the backward instead of 46); and short sequences, whose first rows, with the largest
// weights, have most of the gradients' norm (64 causal tokens of one head: 1.06 instead of 1.39 to 1.57,
// as the sample falls; 4 x 256 tokens of 8 heads of 64 take 17.4 us instead of 15.4). Longer calls take
// one value (1.41 to 1.46): the choice alone costs them 4 to 12 % (4096 causal tokens of 16 heads of
// 64: 327 us for 292).
//
// float16 holds 40 powers of two, and dS has the size of the upstream gradient times that of v times a
// weight. Its backward therefore rounds dS times a power of two (one of each query for dq, one of each
// block of keys for dk) and P times 2^14, and takes them out of the float32 sums at the end: the ratio
// is below 1.5 for gradients and values of any size (without it 3.4 at gradients of 1e-3 over 2048 causal
// tokens, and infinities where dS passes 65504). The norms and their maxima cost the backward 83 -> 93 us
// (8 x 1024 tokens of 12 heads of 64, window 256) and 220 -> 232 (4096 causal of 16 of 128); bfloat16 has
// float32's range and takes neither.
#include <cmath>
#include <utility>

#include "nt_attention.cuh"
#include "nt_tc.cuh"

namespace nt {

constexpr int kTcRows = 128;
constexpr uint32_t kTmemColumns = 512;
constexpr float kRaiseSum = 8192.0f;
constexpr int64_t kFineKeys = 16;
constexpr int kShortQueries = 512;

// Whether one of queries [i0, i1) sees at most kFineKeys keys. Along the queries the number of keys
// first grows, then stays and then, past the sequence's length, falls: the least is at an end.
__device__ __forceinline__ bool attn_few_keys(const AttnParams& P, int length, int i0, int i1) {
  return attn_key_count(P, length, i0) <= kFineKeys || attn_key_count(P, length, i1 - 1) <= kFineKeys;
}
// float16: weights are at most 1, so that 2^14 times them stays below 65504 and those from 2^-28 on are
// normal numbers.
constexpr int kWeightPower = 14;

// The power of two e for dS = P (dP - delta) of rows whose norms of g and v are at most g and v: |dP| and
// |delta| (delta is a mean of dP) are at most g v, so 2^e |dS| is below 2^14 and not far below it.
// Norms of 0 have nothing to scale.
__device__ __forceinline__ int gradient_power(float g, float v) {
  const int exponent = (__float_as_int(2.0f * g * v) >> 23 & 255) - 127;
  return min(max(13 - exponent, -100), 100);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }   // -126 <= e <= 127
// The largest of the entries that hold rows [lo, hi), 0 if there are none. A whole warp.
__device__ __forceinline__ float largest_norm(const float* tops, int dim, int lo, int hi, int lane) {
  float top = 0.0f;
  const int end = norm_tiles(hi, dim);
#pragma unroll 8
  for (int i = lo / norm_rows(dim) + lane; i < end; i += 32) top = fmaxf(top, tops[i]);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // (not negative)
}
// The largest norm of v among the keys that queries [q0, q1) see.
__device__ __forceinline__ float largest_value_norm(const AttnParams& P, int length, int b, int hk, int q0, int q1, int lane) {
  const AttnKeys range(P, length, q0, q1);
  const float* tops = P.v_top + ((int64_t)b * P.kv_heads + hk) * norm_tiles(P.keys, P.dim);
  return fmaxf(largest_norm(tops, P.dim, 0, range.sink_end, lane), largest_norm(tops, P.dim, range.lo, range.hi, lane));
}

// Which columns of a tile a row sees: c < end and (c >= begin or c < sink). word(c0) has bit e set
// for column c0 + e, so that a masked tile costs one bit test and one select per element.
struct ColumnMask {
  int begin, end, sink;
  static __device__ __forceinline__ uint32_t below(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  }
  __device__ __forceinline__ uint32_t word(int c0) const {
    return below(end - c0) & (~below(begin - c0) | below(sink - c0));
  }
};

// A wait of a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity));
}
// Phase of slot use n of a ring of `size`.
__device__ __forceinline__ uint32_t ring_phase(int n, int size) { return (uint32_t)(n / size) & 1u; }

template <int N, int... C>
__device__ __forceinline__ void exponentials(float (&x)[N], std::integer_sequence<int, C...>) {
  (ex2_mixed<C>(x[2 * C], x[2 * C + 1]), ...);
}

// Rows [rows, next multiple of 16) of a tile are cleared: their weights are 0, but what lies there
// may be anything, and 0 * NaN must not reach a sum. One warp.
template <int DP>
__device__ __forceinline__ void clear_tail(uint8_t* tile, int rows, int lane) {
  const int tail = (rows + 15) / 16 * 16 - rows;
  if (tail == 0) return;
  for (int i = lane; i < tail * (DP / 8); i += 32) {
    const int row = rows + i / (DP / 8), c = i % (DP / 8);
    *reinterpret_cast<uint4*>(tile + (c / 8) * kTcRows * 128 + row * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  __syncwarp();
}

// ---- forward -------------------------------------------------------------------------
// o = sum_j exp(scale s_j - m) v_j / sum_j exp(scale s_j - m) in one pass over the keys, 128 at a time.
// Heads of up to 128: a block owns two groups of 128 queries of one head, which share the key and value
// tiles (a tile fetched for 128 queries alone would ask the L2 for 64 KB per 1024 cycles of products).
// Eight warps do the softmax of a group: two threads share a row, 64 columns each. The products of one
// group run under the exponentials of the other:
//   s0(0) s1(0) | o0 += w0(0) v, s0(1) | o1 += w1(0) v, s1(1) | o0 += w0(1) v, ...
// TMEM: s0, s1 (the weights over them), o0, o1. (16 heads of 128, 4096 causal tokens: 69 us, 1.0 PFLOP/s
// of the visible pairs, the tensor pipe active for 47 % of the time, the exponentials' for 36, issue 44:
// no pipe is full; what is left are the waits between a tile's scores, weights and product. With a
// window of 512 of 2 x 2048 tokens 43 us, where a block's start and end, some 5 us of 20, are bare.)
// Heads of up to 64: half of the bytes and of TMEM, so one group to a block and two blocks on an SM,
// and the start and end of one lie under the other's work (8 x 1024 tokens of 12 heads, window 256: 40
// us with two groups to a block, 34 so; 8192 tokens of 16 heads, window 128: 46, 34; 2 x 4096 causal of
// 16: 119, 113).
// SPLIT: where there are too few blocks of queries for the device, a cluster of blocks shares the
// tiles of one; each leaves its unnormalised output, maxima and sums in its shared memory, and they
// are joined from there, rows dealt to the blocks, always in the same order.
template <int DP> struct FwdShared {
  static constexpr int kGroups = DP <= 64 ? 1 : 2, kResident = 2 / kGroups;   // of 128 queries; blocks on an SM
  static constexpr int kRows = kGroups * kTcRows;
  static constexpr int kWarps = 8 * kGroups, kCopyWarp = kWarps, kMmaWarp = kWarps + 1, kThreads = (kWarps + 2) * 32;
  static constexpr int kTmem = kTmemColumns / kResident;
  static constexpr int kTile = kTcRows * DP * 2;
  static constexpr int kRing = 2;
  static constexpr int kK = kGroups * kTile, kV = kK + kRing * kTile, kControl = kV + kRing * kTile;
  struct Control {
    float exchange[kGroups][2][2][kTcRows];   // group, use (maximum, sum), half of the columns, row
    float statistics[kRows][2];   // SPLIT: maximum and sum
    uint64_t q_full, k_full[kRing], k_free[kRing], v_full[kRing], v_free[kRing], s_full[kGroups], w_full[kGroups], o_full[kGroups];
    uint32_t tmem;
  };
  static constexpr int kPartRow = DP + 4;   // floats; SPLIT: a row of the unnormalised output
  static_assert(kRows * kPartRow * 4 <= kControl, "the output takes the tiles' place");
  static constexpr int kBytes = kControl + (int)sizeof(Control);
};

template <int DT, int DP, bool SPLIT>
__global__ void __launch_bounds__(FwdShared<DP>::kThreads, FwdShared<DP>::kResident)
attention_tc_forward(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using Shape = FwdShared<DP>;
  constexpr int TILE = Shape::kTile, RING = Shape::kRing, GROUPS = Shape::kGroups, ROWS = Shape::kRows;
  constexpr int kCopyWarp = Shape::kCopyWarp, kMmaWarp = Shape::kMmaWarp;
  // No static shared memory: the dynamic block starts where shared memory does, 1024 bytes in.
  extern __shared__ __align__(1024) uint8_t aligned[];
  typename Shape::Control& ctl = *reinterpret_cast<typename Shape::Control*>(aligned + Shape::kControl);
  const uint32_t base = smem_u32(aligned);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Blocks in the order of their work: the last queries of every head first.
  const int splits = SPLIT ? P.splits : 1, rank = SPLIT ? (int)cluster_rank() : 0;
  const uint32_t block = blockIdx.x / splits;
  const uint32_t pairs = (uint32_t)P.heads * P.batch, tiles = gridDim.x / splits / pairs;
  const int b = block % pairs / P.heads, h = block % P.heads, hk = h / P.group;
  const int i0 = (tiles - 1 - block / pairs) * ROWS, i1 = min(P.queries, i0 + ROWS);
  const int length = attn_length(P, b);
  const AttnKeys range(P, length, i0, i1);
  // The block's tiles: all, or its share.
  const int all = range.blocks(kTcRows), first = all * rank / splits, blocks = all * (rank + 1) / splits - first;
  auto tile_of = [&](int j, int& begin, int& end) { range.block(first + j, kTcRows, begin, end); };
  // Whether a query of group g sees a key of [begin, end) (group 1 may be past the last query).
  const AttnKeys range0(P, length, i0, min(i1, i0 + kTcRows)), range1(P, length, min(i1, i0 + kTcRows), i1);
  auto active = [&](int g, int begin, int end) {
    if (GROUPS == 1) return true;
    const AttnKeys& r = g ? range1 : range0;
    return (g == 0 || i1 > i0 + kTcRows) && ((begin < r.hi && end > r.lo) || begin < r.sink_end);
  };

  // The copying warp sets up the barriers and issues the first copies while the rest is set up.
  auto load = [&](const CUtensorMap& map, int at, int token, int head, uint64_t* bar) {
#pragma unroll
    for (int half = 0; half < DP / 64; ++half)
      tma_load(aligned + at + half * kTcRows * 128, &map, half * 64, token, head, b, bar);
  };
  auto fill = [&](const CUtensorMap& map, int at, uint64_t* full, int j) {
    int begin, end;
    tile_of(j, begin, end);
    mbar_arrive_expect_tx(&full[j % RING], TILE);
    load(map, at + j % RING * TILE, begin, hk, &full[j % RING]);
  };
  if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, Shape::kTmem);
  if (warp == kCopyWarp && lane == 0) {
    mbar_init(&ctl.q_full, 1);
#pragma unroll
    for (int i = 0; i < RING; ++i) {
      mbar_init(&ctl.k_full[i], 1); mbar_init(&ctl.k_free[i], 1); mbar_init(&ctl.v_full[i], 1); mbar_init(&ctl.v_free[i], 1);
    }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(&ctl.s_full[i], 1); mbar_init(&ctl.w_full[i], 8); mbar_init(&ctl.o_full[i], 1);
    }
    fence_mbar_init();
    if (blocks > 0) {
      // The second group's rows may all lie past the last query: the copy then writes zeros.
      mbar_arrive_expect_tx(&ctl.q_full, GROUPS * TILE);
      load(map_q, 0, i0, h, &ctl.q_full);
      fill(map_k, Shape::kK, ctl.k_full, 0);
      if constexpr (GROUPS == 2) load(map_q, TILE, i0 + kTcRows, h, &ctl.q_full);
      fill(map_v, Shape::kV, ctl.v_full, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  bool ok = true;

  if (warp == kCopyWarp) {
    if (lane == 0 && blocks > 0) {
      int n1 = 1, n2 = 1;
      for (int j = 1; j < blocks; ++j) {
        if (j >= RING) ok = wait_bar(&ctl.k_free[j % RING], ring_phase(j - RING, RING));
        if (!ok) break;
        fill(map_k, Shape::kK, ctl.k_full, j);
        n1 = j + 1;
        if (j >= RING) ok = wait_bar(&ctl.v_free[j % RING], ring_phase(j - RING, RING));
        if (!ok) break;
        fill(map_v, Shape::kV, ctl.v_full, j);
        n2 = j + 1;
      }
      if (!ok) {   // the copies in flight land before the block may end
        wait_bar(&ctl.q_full, 0);
        for (int i = max(0, n1 - RING); i < n1; ++i) wait_bar(&ctl.k_full[i % RING], ring_phase(i, RING));
        for (int i = max(0, n2 - RING); i < n2; ++i) wait_bar(&ctl.v_full[i % RING], ring_phase(i, RING));
      }
    }
  } else if (warp == kMmaWarp) {
    const int width16 = (P.dim + 15) / 16;
    const uint32_t pv = tc_instruction<DT>(width16 * 16, true);
    auto scores = [&](int g, int at, int rows) {
      if (elect_one()) {
        const uint32_t qk = tc_instruction<DT>((rows + 15) / 16 * 16, false);
        const uint64_t q = tc_columns(base + g * TILE), k = tc_columns(base + at);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          if (s < width16)
            tc_mma(tmem + g * kTcRows, q + tc_column_step(kTcRows, s), k + tc_column_step(kTcRows, s), qk, s > 0);
        tc_commit(&ctl.s_full[g]);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    int done[GROUPS] = {};   // tiles of each group
    bool finished = false;   // group 0, before the last tile
    int begin = 0, end = 0;
    if (blocks > 0) {
      tile_of(0, begin, end);
      ok = wait_warp(&ctl.q_full, 0) && wait_warp(&ctl.k_full[0], 0);
      if (ok) {
        if (active(0, begin, end)) scores(0, Shape::kK, end - begin);
        if (GROUPS == 2 && active(1, begin, end)) scores(1, Shape::kK, end - begin);
        commit(&ctl.k_free[0]);
      }
    }
    for (int j = 0; j < blocks && ok; ++j) {
      int next_begin = 0, next_end = 0;
      const int slot = j % RING, next = (j + 1) % RING;
      if (j + 1 < blocks) {
        tile_of(j + 1, next_begin, next_end);
        ok = wait_warp(&ctl.k_full[next], ring_phase(j + 1, RING));
      }
      ok = ok && wait_warp(&ctl.v_full[slot], ring_phase(j, RING));
      if (!ok) break;
      clear_tail<DP>(aligned + Shape::kV + slot * TILE, end - begin, lane);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (active(g, begin, end)) {
          ok = ok && wait_warp(&ctl.w_full[g], done[g] & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t v = tc_rows(base + Shape::kV + slot * TILE, kTcRows);
#pragma unroll
            for (int s = 0; s < kTcRows / 16; ++s)   // the weights lie in two halves of 64 columns
              if (s * 16 < end - begin)
                tc_mma_tmem(tmem + ROWS + g * DP, tmem + g * kTcRows + (s >> 2) * 64 + (s & 3) * 8,
                            v + tc_row_step(s), pv, done[g] > 0 || s > 0);
          }
          __syncwarp();
          ++done[g];
        }
        if (j + 1 < blocks && active(g, next_begin, next_end)) {
          scores(g, Shape::kK + next * TILE, next_end - next_begin);
        } else if (GROUPS == 2 && g == 0 && j + 2 == blocks) {
          // The first group sees nothing of the last tile (of causal attention): its output is ready.
          commit(&ctl.o_full[0]);
          finished = true;
        }
      }
      if (!ok) break;
      commit(&ctl.v_free[slot]);
      if (j + 1 < blocks) commit(&ctl.k_free[next]);
      begin = next_begin;
      end = next_end;
    }
    // (A block without tiles commits nothing: no one would wait for the arrival, and the block may end.)
    if (blocks > 0) {
      if (!finished) commit(&ctl.o_full[0]);
      if constexpr (GROUPS == 2) commit(&ctl.o_full[1]);
      if (!ok) wait_bar(&ctl.o_full[GROUPS - 1], 0);   // no product is in flight when TMEM is given back
    }
  } else {
    const int g = GROUPS == 2 ? warp >> 3 : 0, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // lane 32 (w % 4) in the address's upper half
    const uint32_t t_s = tmem + g * kTcRows + lanes + half * 64;
    const uint32_t t_o = tmem + ROWS + g * DP + lanes + half * (DP / 2);
    const int q0 = i0 + g * kTcRows, q1 = min(i1, q0 + kTcRows);
    const int p = P.offset + q0 + row;
    const int full_lo = P.window == 0 ? 0 : P.offset + q1 - P.window;   // first key the last query sees
    const int full_hi = P.offset + q0;                                   // last key the first query sees
    const int pair = 1 + g * 4 + (warp & 3);
    float m = -INFINITY, l = 0.0f, shift = 0.0f, minus = 0.0f;
    bool extreme = false;
    int done = 0;
    for (int j = 0; j < blocks; ++j) {
      int begin, end;
      tile_of(j, begin, end);
      if (!active(g, begin, end)) continue;
      // A wait that ran out is remembered and not waited for again; the warp still takes part in
      // every barrier, so that no other warp is left waiting for it.
      if (ok) ok = wait_bar(&ctl.s_full[g], done & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      const bool full = end - begin == kTcRows && end - 1 <= full_hi && (begin >= full_lo || end <= P.sinks);
      if (!full) {
        const ColumnMask mask{P.window == 0 ? 0 : p - P.window + 1 - begin, min(end, p + 1) - begin, P.sinks - begin};
        seen[0] = mask.word(half * 64);
        seen[1] = mask.word(half * 64 + 32);
      }
      // The reference maximum only has to keep the weights in range, so the one of the first tile
      // stays until a row's weights of one tile sum to more than 2^13 (float16 holds 2^15). In the
      // first tile, in that rare case, and where a row sees its first key, the two warps of the rows
      // agree on a new maximum, rescale the output and form the weights (again).
      bool again = done == 0;
      while (true) {
        if (again) {
          float top = -INFINITY;
#pragma unroll
          for (int c0 = 0; c0 < 64; c0 += 32) {
            uint32_t s[32];
            tmem_load32(t_s + c0, s);
            tmem_wait_load();
#pragma unroll
            for (int c = 0; c < 32; ++c) top = fmaxf(top, seen[c0 / 32] >> c & 1 ? __uint_as_float(s[c]) : -INFINITY);
          }
          ctl.exchange[g][0][half][row] = top;
          named_barrier(pair, 64);
          top = fmaxf(m, fmaxf(top, ctl.exchange[g][0][half ^ 1][row]));
          const float f = top == -INFINITY ? 1.0f : ex2_approx((m - top) * P.scale_log2);
          m = top;
          l *= f;
          if (done > 0) {
            // Products complete in order: s of this tile is there, so o of the last one is too.
#pragma unroll 1
            for (int c = 0; c < DP / 2; c += 32) {
              uint32_t o[32];
              tmem_load32(t_o + c, o);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_store32(t_o + c, o);
            }
          }
          shift = m == -INFINITY ? 0.0f : m;
          // Scores near the ends of float32 are subtracted before they are scaled.
          extreme = __any_sync(0xffffffffu, isinf(shift * P.scale_log2));
          minus = extreme ? 0.0f : -shift * P.scale_log2;
        }
        Pair sum(0.0f, 0.0f);
        uint32_t w[32];
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          uint32_t s[32];
          tmem_load32(t_s + c0, s);
          tmem_wait_load();
          if (extreme) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = __float_as_uint(__uint_as_float(s[c]) - shift);
          }
          float x[32];
          const Pair scale2(P.scale_log2, P.scale_log2), minus2(minus, minus);
#pragma unroll
          for (int c = 0; c < 32; c += 2)
            fma2(Pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, minus2).get(x[c], x[c + 1]);
          exponentials(x, std::make_integer_sequence<int, 16>{});
          if (!full) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = seen[c0 / 32] >> c & 1 ? x[c] : 0.0f;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            sum = add2(sum, Pair(x[c], x[c + 1]));
            w[(c0 + c) / 2] = pack2<DT>(x[c], x[c + 1]);
          }
        }
        float a, b;
        sum.get(a, b);
        if (!again) {
          again = named_barrier_or(pair, 64, a + b > kRaiseSum || (m == -INFINITY && (seen[0] | seen[1])));
          if (again) continue;
        }
        tmem_store32(t_s, w);   // over scores that are no longer needed
        l += a + b;
        break;
      }
      ++done;
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.w_full[g]);
    }
    if (ok && blocks > 0) ok = wait_bar(&ctl.o_full[g], 0);
    __syncwarp();
    tc_fence_after();
    ctl.exchange[g][1][half][row] = l;
    named_barrier(pair, 64);
    // Halves in a fixed order, so that both threads of a row have the same sum.
    l = ctl.exchange[g][1][0][row] + ctl.exchange[g][1][1][row];
    if constexpr (SPLIT) {
      if (GROUPS == 2 && ok && blocks > 0) ok = wait_bar(&ctl.o_full[GROUPS - 1 - g], 0);   // every tile is free
      __syncwarp();
      const int r = g * kTcRows + row;
      if (done > 0) {
        float* part = reinterpret_cast<float*>(aligned) + r * Shape::kPartRow + half * (DP / 2);
#pragma unroll
        for (int c = 0; c < DP / 2; c += 32) {
          uint32_t o[32];
          tmem_load32(t_o + c, o);
          tmem_wait_load();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(part + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      if (half == 0) {
        ctl.statistics[r][0] = m;
        ctl.statistics[r][1] = l;
      }
    } else {
      const float f = l == 0.0f ? 0.0f : 1.0f / l;
      // The group's tile of queries is free now: 32 rows x half of the columns of each warp.
      constexpr int WIDTH = DP / 2, CH = WIDTH / 8;
      uint8_t* stage = aligned + warp * 32 * WIDTH * 2;
      const int row0 = q0 + (warp & 3) * 32, rows = q1 - row0, vectors = (P.dim - half * WIDTH + 7) / 8;
      const int64_t at = (P.os.at(b, h, row0) + half * WIDTH) * 2;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        char* dst = static_cast<char*>(which ? P.o_low : P.o);
        if (dst == nullptr) continue;
#pragma unroll
        for (int c = 0; c < WIDTH; c += 32) {
          uint32_t o[32];
          if (done > 0) {
            tmem_load32(t_o + c, o);
            tmem_wait_load();
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // A row without keys is 0 whatever the accumulator holds.
              const float x = f == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * k]) * f;
              const float y = f == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * k + 1]) * f;
              v[k] = pack2<DT>(x, y);
              if (which) {
                const float2 r = unpack2<DT>(v[k]);
                v[k] = pack2<DT>(x - r.x, y - r.y);
              }
            }
            stage_vector<CH>(stage, lane, (c + e) / 8, make_uint4(v[0], v[1], v[2], v[3]));
          }
        }
        store_staged<CH>(stage, lane, dst + at, P.os.t * 2, rows, vectors);
      }
      const bool live = q0 + row < q1;
      if (live && half == 0 && P.lse != nullptr)
        P.lse[((int64_t)b * P.heads + h) * P.queries + q0 + row] =
            l == 0.0f ? -INFINITY : fmaf(m, P.scale, log2f(l) * kLn2F);
    }
  }
  if (!ok && P.error != nullptr) atomicOr(P.error, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_free(tmem, Shape::kTmem);
  if constexpr (SPLIT) {
    cluster_sync_all();
    constexpr int LPR = DP / 4, RPW = 32 / LPR;   // four columns a lane
    const float* part = reinterpret_cast<const float*>(aligned);
    for (int r0 = (rank + splits * warp) * RPW; warp < Shape::kWarps && r0 < i1 - i0; r0 += splits * Shape::kWarps * RPW) {
      const int r = r0 + lane / LPR, c = lane % LPR * 4;
      if (r >= i1 - i0) continue;
      const JoinedRow row = join_row(part + r * Shape::kPartRow + c, ctl.statistics[r], splits, P.scale_log2);
      const float f = row.sum == 0.0f ? 0.0f : 1.0f / row.sum;
      const float x[4] = {row.o.x * f, row.o.y * f, row.o.z * f, row.o.w * f};
      if (c < P.dim) {
        const int64_t at = P.os.at(b, h, i0 + r) + c;
        const uint2 hi = make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.o) + at) = hi;
        if (P.o_low != nullptr) {
          const float2 v = unpack2<DT>(hi.x), w = unpack2<DT>(hi.y);
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.o_low) + at) =
              make_uint2(pack2<DT>(x[0] - v.x, x[1] - v.y), pack2<DT>(x[2] - w.x, x[3] - w.y));
        }
      }
      if (c == 0 && P.lse != nullptr)
        P.lse[((int64_t)b * P.heads + h) * P.queries + i0 + r] =
            row.sum == 0.0f ? -INFINITY : fmaf(row.top, P.scale, log2f(row.sum) * kLn2F);
    }
    cluster_sync_all();   // a block's shared memory stays until every block has read it
  }
}

// ---- backward ------------------------------------------------------------------------
// One block keeps 128 rows x1, x2 and walks rows y1, y2 128 (heads of up to 64: 64) at a time:
//   s = x1 y1^T, dp = x2 y2^T (TMEM, float32);  P = exp(scale s - lse), dS = P (dp - delta)
//   out1 += dS y1, and with DKV out2 += P y2, with P and dS over s and dp in TMEM as the
//   products' first operand.
// DKV = false: rows are queries (x1 = q, x2 = g; y1 = k, y2 = v): out1 = dq. DKV = true: rows are keys
// (x1 = k, x2 = v; y1 = q, y2 = g): out1 = dk, out2 = dv, over the heads of the group. Both kinds of
// blocks are one launch, the key blocks (the longer ones) first, so that the other kind fills the
// SMs that the last of them leave idle. delta = sum(g o) comes from a kernel before it, whose end
// only the warps that read delta wait for.
// With DKV s, dp and the two outputs fill TMEM, so nothing has a second buffer; the order of the
// products hides the exponentials instead: dp(t) runs while P(t) is computed, out2(t) and s(t + 1)
// while dS(t) is, out1(t) and dp(t + 1) while P(t + 1) is. Without it dp has two buffers and
// dp(t + 1) does not wait for out1(t). Groups of four warps take 32 columns each.
// Bound in long rows by the shared memory that the products of two tiles from there read (85 cycles
// each instead of 64), then by the power cap: 16 heads of 128, 4096 causal tokens, 203 us, 1.18 PFLOP/s
// of the seven products; in short windows by a block's start and end (2 x 2048 tokens, window 512: 103).
// Heads of up to 64 leave room for two blocks on an SM, with half of TMEM and steps of 64 rows each: one
// begins and ends, or waits for its products, while the other computes (8 x 1024 tokens of 12 heads of
// 64, window 256: 97 us with one block and steps of 128, 70 with two; 2 x 4096 of 16, causal: 317, 267).
constexpr int kColumns = 32;           // of a computing thread

// The copying warp also fetches lse and delta of the rows that are walked. Shared memory: x1, x2, the
// ring of y1 (three: s of the next step starts before out1 of this one has ended), the ring of y2 (two)
// and the control block.
template <int DP> struct BwdShared {
  static constexpr int kResident = DP <= 64 ? 2 : 1;   // blocks on an SM
  static constexpr int kStep = tc_query_step(DP), kGroups = kStep / kColumns;
  static constexpr int kWarps = 4 * kGroups, kCopyWarp = kWarps, kMmaWarp = kWarps + 1, kThreads = (kWarps + 2) * 32;
  static constexpr int kTmem = kTmemColumns / kResident;
  static constexpr int kTile = kTcRows * DP * 2, kPiece = kStep * DP * 2;
  static constexpr int kRing1 = 3, kRing2 = 2;
  static constexpr int kY1 = 2 * kTile, kY2 = kY1 + kRing1 * kPiece, kControl = kY2 + kRing2 * kPiece;
  struct Control {
    float stats[2][2][kStep];          // ring of two; lse (times log2 e) and delta, both negative
    uint64_t x_full, y1_full[kRing1], y1_free[kRing1], y2_full[kRing2], y2_free[kRing2], s_full, p_full,
        dp_full[2], ds_full[2],            // by the step's parity: dp(t + 1) may be there before dp(t) was waited for
        stat_full[2], stat_free[2], out_full;
    uint32_t tmem;
    int power;                         // float16, gradients of keys: of the two that scales dS
  };
  static constexpr int kBytes = kControl + (int)sizeof(Control);
};
static_assert(BwdShared<128>::kBytes <= 227 * 1024 && BwdShared<64>::kBytes <= 113 * 1024, "blocks on an SM");

// This lane's share of delta of a query, and of the square of its row of g (NORM).
template <int DT, bool NORM>
__device__ __forceinline__ void delta_share(const AttnParams& P, int b, int h, int64_t row, int c, float& d, float& squares) {
  float x[8], y[8], z[8];
  const int64_t o = P.os.at(b, h, row) + c;
  unpack16<DT>(__ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.g) + P.gs.at(b, h, row) + c)), x);
  unpack16<DT>(__ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.o) + o)), y);
  if (P.o_low != nullptr) {
    unpack16<DT>(__ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.o_low) + o)), z);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += z[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    d = fmaf(x[e], y[e], d);
    if constexpr (NORM) squares = fmaf(x[e], x[e], squares);
  }
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int w = LPR / 2; w > 0; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
  return v;
}

// delta of every query: as many lanes to a row as it has 16-byte vectors. Bound by HBM (g, o and what
// rounding took from o, once: 50 MB of 2 x 2048 tokens of 16 heads of 128 in 7.7 us, 6.5 TB/s).
template <int DT, int DP>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ AttnParams P) {
  constexpr int LPR = DP / 8, ROWS = 256 / LPR;
  grid_dependents_go();
  const int b = blockIdx.z, h = blockIdx.y, c = threadIdx.x % LPR * 8;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  float d = 0.0f, unused = 0.0f;
  if (row < P.queries && c < P.dim) delta_share<DT, false>(P, b, h, row, c, d, unused);
  d = row_sum<LPR>(d);
  if (threadIdx.x % LPR == 0 && row < P.queries) P.delta[((int64_t)b * P.heads + h) * P.queries + row] = d;
}

// The same for float16, with what the scale of dS is taken from: the norm of every row of g, and the
// largest norm of the block's rows of g, or of v among the keys that some query sees (what others hold
// may be anything). A norm that is not finite counts as 0: the gradients of its row are lost, but not
// those of its neighbours. Blocks of queries of a head come first, then those of keys. (67 MB of 2 x
// 2048 tokens of 16 heads of 128: 15.4 us, 4.4 TB/s, for the block's join of its rows; entries of 128
// rows took 17.6 to 25, an entry to a warp with its loads in flight together 19.)
template <int DP>
__global__ void __launch_bounds__(256) attention_delta_norms_kernel(const __grid_constant__ AttnParams P) {
  constexpr int LPR = DP / 8, ROWS = 256 / LPR;
  static_assert(ROWS == norm_rows(DP), "rows of an entry");
  __shared__ float tops[8];
  grid_dependents_go();
  const int b = blockIdx.z, h = blockIdx.y, c = threadIdx.x % LPR * 8;
  const int query_tiles = norm_tiles(P.queries, DP);
  const bool queries = (int)blockIdx.x < query_tiles;
  const int tile = queries ? blockIdx.x : blockIdx.x - query_tiles;
  if (!queries && h >= P.kv_heads) return;
  const int64_t row = (int64_t)tile * ROWS + threadIdx.x / LPR;
  float d = 0.0f, squares = 0.0f;
  if (queries) {
    if (row < P.queries && c < P.dim) delta_share<NT_F16, true>(P, b, h, row, c, d, squares);
  } else {
    const AttnKeys seen(P, attn_length(P, b), 0, P.queries);
    if (row < seen.hi && (row >= seen.lo || row < seen.sink_end) && c < P.dim) {
      float x[8];
      unpack16<NT_F16>(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.v) + P.vs.at(b, h, row) + c)), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = fmaf(x[e], x[e], squares);
    }
  }
  squares = row_sum<LPR>(squares);
  float top = squares < INFINITY ? sqrtf(squares) : 0.0f;
  if (queries) {
    d = row_sum<LPR>(d);
    if (threadIdx.x % LPR == 0 && row < P.queries) {
      const int64_t at = ((int64_t)b * P.heads + h) * P.queries + row;
      P.delta[at] = d;
      P.g_norm[at] = top;
    }
  }
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // (not negative)
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x > 0) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) top = fmaxf(top, tops[w]);
  if (queries) P.g_top[((int64_t)b * P.heads + h) * query_tiles + tile] = top;
  else P.v_top[((int64_t)b * P.kv_heads + h) * norm_tiles(P.keys, DP) + tile] = top;
}

template <int DT, int DP, bool DKV, bool FINE>
__device__ __forceinline__ void backward_block(const AttnParams& P, uint32_t block, const CUtensorMap& map_x1,
                                               const CUtensorMap& map_x2, const CUtensorMap& map_y1,
                                               const CUtensorMap& map_y2) {
  using Shape = BwdShared<DP>;
  constexpr int TILE = Shape::kTile, PIECE = Shape::kPiece, RING1 = Shape::kRing1, RING2 = Shape::kRing2;
  constexpr int kStep = Shape::kStep, kCopyWarp = Shape::kCopyWarp, kMmaWarp = Shape::kMmaWarp;
  // No static shared memory: the dynamic block starts where shared memory does, 1024 bytes in.
  extern __shared__ __align__(1024) uint8_t aligned[];
  typename Shape::Control& ctl = *reinterpret_cast<typename Shape::Control*>(aligned + Shape::kControl);
  const uint32_t base = smem_u32(aligned);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Blocks in the order of their work: the last queries, or the first keys, of every head first.
  const uint32_t heads = DKV ? P.kv_heads : P.heads, pairs = heads * P.batch;
  const int b = block % pairs / heads, h0 = block % heads;   // query head of dq, key head of dk and dv
  const int index = block / pairs;
  const int length = attn_length(P, b);

  // The block's rows [r0, r1) and the steps it walks.
  int r0, r1, part = 0, parts = 1, steps, per_head = 1;
  uint32_t from = 0;
  if constexpr (!DKV) {
    r0 = ((P.queries + kTcRows - 1) / kTcRows - 1 - index) * kTcRows;
    r1 = min(P.queries, r0 + kTcRows);
  } else {
    const AttnPiece piece(P, index);
    part = piece.part;
    parts = piece.parts;
    r0 = piece.tile * kTcRows;
    r1 = min(P.keys, r0 + kTcRows);
  }
  const AttnKeys key_range(P, length, r0, r1);
  const AttnQueries query_range(P, length, r0, r1);
  if constexpr (!DKV) {
    steps = key_range.blocks(kStep);
  } else {
    per_head = (query_range.hi - query_range.lo + kStep - 1) / kStep;
    const int64_t total = (int64_t)per_head * P.group;   // below 2^31, checked on the host
    from = (uint32_t)(total * part / parts);
    steps = (int)(total * (part + 1) / parts - from);
  }
  // Rows [begin, end) of `head` that step t streams; for the gradients of keys, counted on.
  struct Step {
    int begin, end, head, at;
  };
  auto start = [&](Step& s) {
    if constexpr (DKV) {
      s.head = h0 * P.group + (int)(from / (uint32_t)max(per_head, 1));
      s.at = (int)(from % (uint32_t)max(per_head, 1));
      s.begin = query_range.lo + s.at * kStep;
      s.end = min(query_range.hi, s.begin + kStep);
    } else {
      s.head = h0 / P.group;
      s.at = 0;
      key_range.block(0, kStep, s.begin, s.end);
    }
  };
  auto advance = [&](Step& s) {
    ++s.at;
    if constexpr (DKV) {
      if (s.at == per_head) {
        s.at = 0;
        ++s.head;
      }
      s.begin = query_range.lo + s.at * kStep;
      s.end = min(query_range.hi, s.begin + kStep);
    } else {
      key_range.block(s.at, kStep, s.begin, s.end);
    }
  };
  // FINE: whether a query of step s may see few keys, so that dS goes in as two values.
  auto fine = [&](const Step& s) {
    if constexpr (!FINE) return false;
    return DKV ? attn_few_keys(P, length, s.begin, s.end) : attn_few_keys(P, length, r0, r1);
  };

  // The copying warp sets up the barriers and issues the first copies while the rest is set up.
  auto load = [&](const CUtensorMap& map, int at, int token, int head, int rows, uint64_t* bar) {
#pragma unroll
    for (int half = 0; half < DP / 64; ++half)
#pragma unroll
      for (int row = 0; row < rows; row += kStep)
        tma_load(aligned + at + (half * rows + row) * 128, &map, half * 64, token + row, head, b, bar);
  };
  auto fill1 = [&](int t, const Step& s) {
    mbar_arrive_expect_tx(&ctl.y1_full[t % RING1], PIECE);
    load(map_y1, Shape::kY1 + t % RING1 * PIECE, s.begin, s.head, kStep, &ctl.y1_full[t % RING1]);
  };
  auto fill2 = [&](int t, const Step& s) {
    mbar_arrive_expect_tx(&ctl.y2_full[t % RING2], PIECE);
    load(map_y2, Shape::kY2 + t % RING2 * PIECE, s.begin, s.head, kStep, &ctl.y2_full[t % RING2]);
  };
  if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, Shape::kTmem);
  if (warp == kCopyWarp && lane == 0) {
    mbar_init(&ctl.x_full, 1); mbar_init(&ctl.out_full, 1);
#pragma unroll
    for (int i = 0; i < RING1; ++i) { mbar_init(&ctl.y1_full[i], 1); mbar_init(&ctl.y1_free[i], 1); }
#pragma unroll
    for (int i = 0; i < RING2; ++i) {
      mbar_init(&ctl.y2_full[i], 1); mbar_init(&ctl.y2_free[i], 1);
      mbar_init(&ctl.stat_full[i], 1); mbar_init(&ctl.stat_free[i], Shape::kWarps);
    }
    mbar_init(&ctl.s_full, 1); mbar_init(&ctl.p_full, Shape::kWarps);
#pragma unroll
    for (int i = 0; i < 2; ++i) { mbar_init(&ctl.dp_full[i], 1); mbar_init(&ctl.ds_full[i], Shape::kWarps); }
    fence_mbar_init();
    if (steps > 0) {
      Step s;
      start(s);
      mbar_arrive_expect_tx(&ctl.x_full, 2 * TILE);
      load(map_x1, 0, r0, h0, kTcRows, &ctl.x_full);
      fill1(0, s);
      load(map_x2, TILE, r0, h0, kTcRows, &ctl.x_full);
      fill2(0, s);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  // Columns: s, dp, out1 and, with DKV, out2, else the second buffer of dp.
  const uint32_t t_s = tmem, t_dp = tmem + kStep, t_out1 = tmem + 2 * kStep, t_out2 = t_out1 + DP;
  auto t_dp_of = [&](int t) { return DKV || (t & 1) == 0 ? t_dp : t_out1 + DP; };
  bool ok = true;

  if (warp == kCopyWarp) {
    Step copied{}, read{};
    if (steps > 0) {
      start(copied);
      read = copied;
    }
    int n1 = min(steps, 1), n2 = n1;
    float delta_scale = -1.0f;
    auto copies = [&](int t) {
      advance(copied);
      if (t >= RING1) ok = wait_warp(&ctl.y1_free[t % RING1], ring_phase(t - RING1, RING1));
      if (!ok) return;
      if (lane == 0) fill1(t, copied);
      n1 = t + 1;
      if (t >= RING2) ok = wait_warp(&ctl.y2_free[t % RING2], ring_phase(t - RING2, RING2));
      if (!ok) return;
      if (lane == 0) fill2(t, copied);
      n2 = t + 1;
    };
    auto statistics = [&](int t) {
      const int64_t stat = ((int64_t)b * P.heads + read.head) * P.queries + read.begin;
      float lse[kStep / 32], delta[kStep / 32];
#pragma unroll
      for (int i = 0; i < kStep / 32; ++i) {
        const int c = i * 32 + lane;
        const bool in = read.begin + c < read.end;
        lse[i] = in ? fmaf(-P.lse[stat + c], kLog2eF, DT == NT_F16 ? kWeightPower : 0) : 0.0f;
        delta[i] = in ? delta_scale * P.delta[stat + c] : 0.0f;
      }
      advance(read);
      if (t >= 2) ok = wait_warp(&ctl.stat_free[t & 1], ring_phase(t - 2, 2));
      if (!ok) return;
#pragma unroll
      for (int i = 0; i < kStep / 32; ++i) {
        ctl.stats[t & 1][0][i * 32 + lane] = lse[i];
        ctl.stats[t & 1][1][i * 32 + lane] = delta[i];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.stat_full[t & 1]);
    };
    // Both rings hold two steps and more; statistics(t + 1) wait for dS(t - 1), copies(t + 2) for
    // out1(t - 1) and out2(t): the order in which these end.
    if (steps > 1) copies(1);
    if constexpr (DKV) {
      grid_dependency_wait();
      if (DT == NT_F16 && steps > 0) {
        // One power of two for the block: the sum over the queries is one accumulator.
        float g = 0.0f;
        for (int h = h0 * P.group; h < (h0 + 1) * P.group; ++h)
          g = fmaxf(g, largest_norm(P.g_top + ((int64_t)b * P.heads + h) * norm_tiles(P.queries, P.dim), P.dim,
                                    query_range.lo, query_range.hi, lane));
        const int power = gradient_power(g, largest_value_norm(P, length, b, h0, query_range.lo, query_range.hi, lane));
        delta_scale = -power_of_two(power - kWeightPower);
        if (lane == 0) ctl.power = power;
        __syncwarp();
      }
      if (steps > 0) statistics(0);
    }
    for (int t = 0; t < steps && ok; ++t) {
      if (DKV && t + 1 < steps) statistics(t + 1);
      if (ok && t + 2 < steps) copies(t + 2);
    }
    if (!ok && lane == 0) {   // the copies in flight land before the block may end
      wait_bar(&ctl.x_full, 0);
      for (int i = max(0, n1 - RING1); i < n1; ++i) wait_bar(&ctl.y1_full[i % RING1], ring_phase(i, RING1));
      for (int i = max(0, n2 - RING2); i < n2; ++i) wait_bar(&ctl.y2_full[i % RING2], ring_phase(i, RING2));
    }
  } else if (warp == kMmaWarp) {
    const int width16 = (P.dim + 15) / 16;
    const uint32_t accumulate = tc_instruction<DT>(width16 * 16, true);
    const uint64_t x1 = tc_columns(base), x2 = tc_columns(base + TILE);
    // acc = x y^T of one step
    auto product = [&](uint32_t acc, uint64_t x, int at, int rows, uint64_t* done) {
      if (elect_one()) {
        const uint32_t instruction = tc_instruction<DT>((rows + 15) / 16 * 16, false);
        const uint64_t y = tc_columns(base + at);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          if (k < width16) tc_mma(acc, x + tc_column_step(kTcRows, k), y + tc_column_step(kStep, k), instruction, k > 0);
        tc_commit(done);
      }
      __syncwarp();
    };
    // acc += w y of one step, which ends its use of y; w lies in pieces of 32 columns, each over its
    // scores, with its low parts, where there are any, beside it
    auto sum = [&](uint32_t acc, uint32_t w, int at, int rows, bool add, bool low, uint64_t* done) {
      if (elect_one()) {
        const uint64_t y = tc_rows(base + at, kStep);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          if (k * 16 < rows)
            tc_mma_tmem(acc, w + (k >> 1) * kColumns + (k & 1) * 8, y + tc_row_step(k), accumulate, add || k > 0);
        if (low) {
#pragma unroll 1
          for (int k = 0; k * 16 < rows; ++k)
            tc_mma_tmem(acc, w + (k >> 1) * kColumns + kColumns / 2 + (k & 1) * 8, y + tc_row_step(k), accumulate, true);
        }
        tc_commit(done);
      }
      __syncwarp();
    };
    auto arrive = [&](uint64_t* bar, uint32_t phase, int at, int rows) {
      if (!wait_warp(bar, phase)) return false;
      clear_tail<DP>(aligned + at, rows, lane);
      return true;
    };
    int rows = 0;
    Step s;
    if (steps > 0) {
      start(s);
      rows = s.end - s.begin;
      ok = wait_warp(&ctl.x_full, 0) && arrive(&ctl.y1_full[0], 0, Shape::kY1, rows);
      if (ok) product(t_s, x1, Shape::kY1, rows, &ctl.s_full);
    }
    auto second = [&](int t, int rows) {   // dp(t)
      const int y2 = Shape::kY2 + t % RING2 * PIECE;
      if (!arrive(&ctl.y2_full[t % RING2], ring_phase(t, RING2), y2, rows)) return false;
      product(t_dp_of(t), x2, y2, rows, &ctl.dp_full[t & 1]);
      if constexpr (!DKV) {   // nothing else reads y2
        if (elect_one()) tc_commit(&ctl.y2_free[t % RING2]);
        __syncwarp();
      }
      return true;
    };
    if (!DKV && steps > 0 && ok) ok = second(0, rows);
    for (int t = 0; t < steps && ok; ++t) {
      if constexpr (DKV) ok = second(t, rows);
      ok = ok && wait_warp(&ctl.p_full, t & 1);
      if (!ok) break;
      tc_fence_after();
      if constexpr (DKV) sum(t_out2, t_s, Shape::kY2 + t % RING2 * PIECE, rows, t > 0, false, &ctl.y2_free[t % RING2]);
      const int now = rows;
      const bool low = fine(s);
      if (t + 1 < steps) {
        advance(s);
        rows = s.end - s.begin;
        const int next = Shape::kY1 + (t + 1) % RING1 * PIECE;
        ok = arrive(&ctl.y1_full[(t + 1) % RING1], ring_phase(t + 1, RING1), next, rows);
        if (!ok) break;
        product(t_s, x1, next, rows, &ctl.s_full);
        if constexpr (!DKV) ok = second(t + 1, rows);
      }
      ok = ok && wait_warp(&ctl.ds_full[t & 1], ring_phase(t, 2));
      if (!ok) break;
      tc_fence_after();
      sum(t_out1, t_dp_of(t), Shape::kY1 + t % RING1 * PIECE, now, t > 0, low, &ctl.y1_free[t % RING1]);
    }
    if (steps > 0) {   // (as in the forward)
      if (elect_one()) tc_commit(&ctl.out_full);
      __syncwarp();
      if (!ok) wait_bar(&ctl.out_full, 0);
    }
  } else {
    const int group = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t at_s = t_s + lanes + group * kColumns;
    float lse = 0.0f, delta = 0.0f;
    // float16: the power of two that dS carries; for dq one of each row, which the weights bring in, with
    // DKV one of the block, 2^kWeightPower of it from the weights and the rest from dP - delta.
    float carried = 1.0f;
    if constexpr (!DKV) {
      grid_dependency_wait();
      float g = 0.0f;
      if (r0 + row < r1) {
        const int64_t stat = ((int64_t)b * P.heads + h0) * P.queries + r0 + row;
        lse = -P.lse[stat] * kLog2eF;
        delta = -P.delta[stat];
        if constexpr (DT == NT_F16) g = P.g_norm[stat];
      }
      if constexpr (DT == NT_F16) {
        const int power = gradient_power(g, largest_value_norm(P, length, b, h0 / P.group, r0, r1, lane));
        lse += power;
        carried = power_of_two(power);
      }
    }
    // Steps without a masked pair: those whose rows are all there and lie within these bounds.
    int full_lo, full_hi;
    if constexpr (!DKV) {
      full_lo = P.window == 0 ? 0 : P.offset + r1 - P.window;   // first key the last query sees
      full_hi = P.offset + r0;                                   // last key the first query sees
    } else {
      // (a window is at most 2^31 - 1 and positions stay below it, hence the 64-bit sum)
      const int64_t last = P.window == 0 || r0 + kTcRows <= P.sinks ? INT32_MAX : (int64_t)r0 + P.window - 1 - P.offset;
      full_lo = r0 + kTcRows - 1 - P.offset;                     // first query that sees the last key
      full_hi = r0 + kTcRows > length ? -1 : (int)(last < INT32_MAX ? last : INT32_MAX);
    }
    const bool one_key = !DKV && attn_key_count(P, length, r0 + row) == 1;
    Step step;
    if (steps > 0) start(step);
    for (int t = 0; t < steps; ++t, advance(step)) {
      const int begin = step.begin, end = step.end;
      const bool full = end - begin == kStep && end - 1 <= full_hi && (begin >= full_lo || (!DKV && end <= P.sinks));
      // A wait that ran out is remembered and not waited for again (as in the forward).
      if (ok && DKV) ok = wait_bar(&ctl.stat_full[t & 1], ring_phase(t, 2));
      if (ok) ok = wait_bar(&ctl.s_full, t & 1);
      __syncwarp();
      tc_fence_after();
      float p[kColumns];
      tmem_load32(at_s, reinterpret_cast<uint32_t(&)[32]>(p));
      tmem_wait_load();
      if constexpr (!DKV) {   // s may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full);
      }
      const Pair scale2(P.scale_log2, P.scale_log2);
#pragma unroll
      for (int c = 0; c < kColumns; c += 4) {
        float4 ls = make_float4(lse, lse, lse, lse);   // negative
        if constexpr (DKV) ls = *reinterpret_cast<const float4*>(&ctl.stats[t & 1][0][group * kColumns + c]);
        fma2(Pair(p[c], p[c + 1]), scale2, Pair(ls.x, ls.y)).get(p[c], p[c + 1]);
        fma2(Pair(p[c + 2], p[c + 3]), scale2, Pair(ls.z, ls.w)).get(p[c + 2], p[c + 3]);
      }
      exponentials(p, std::make_integer_sequence<int, kColumns / 2>{});
      uint32_t seen = 0xffffffffu, moved = 0xffffffffu;   // moved: those with a dS (a full step has no other)
      if (!full) {
        ColumnMask mask;
        if constexpr (!DKV) {
          const int pos = P.offset + r0 + row;
          mask = {P.window == 0 ? 0 : pos - P.window + 1 - begin, min(end, pos + 1) - begin, P.sinks - begin};
        } else {
          const int key = r0 + row, first = P.offset + begin;
          const int64_t last = P.window == 0 || key < P.sinks ? (int64_t)kStep : (int64_t)key + P.window - first;
          mask = {key - first, key >= length ? 0 : (int)(last < end - begin ? last : end - begin), 0};
        }
        seen = mask.word(group * kColumns);
        if constexpr (DKV) moved = seen & ~__ballot_sync(0xffffffffu, attn_key_count(P, length, begin + group * kColumns + lane) == 1);
        else moved = one_key ? 0u : seen;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) p[c] = seen >> c & 1 ? p[c] : 0.0f;
      }
      uint32_t w[kColumns / 2];
      if constexpr (DKV) {
#pragma unroll
        for (int e = 0; e < kColumns / 2; ++e) w[e] = pack2<DT>(p[2 * e], p[2 * e + 1]);
        tmem_store16(at_s, w);
        tmem_wait_store();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full);
      }
      if (ok) ok = wait_bar(&ctl.dp_full[t & 1], ring_phase(t, 2));
      __syncwarp();
      tc_fence_after();
      const uint32_t at_dp = t_dp_of(t) + lanes + group * kColumns;
      if constexpr (DT == NT_F16 && DKV) carried = power_of_two(ctl.power - kWeightPower);
      uint32_t d[kColumns];
      tmem_load32(at_dp, d);
      tmem_wait_load();
      auto difference = [&](Pair x, Pair y) {
        if constexpr (DT == NT_F16 && DKV) return fma2(x, Pair(carried, carried), y);   // (delta comes scaled)
        else return add2(x, y);
      };
      // dp of a key that is not there may be NaN: 0 * NaN is cleared.
      auto there = [&](int c) { return (moved >> c & 1 ? 0xffffu : 0u) | (moved >> (c + 1) & 1 ? 0xffff0000u : 0u); };
      if (FINE && fine(step)) {
        uint32_t rest[kColumns / 2];   // what rounding takes away
#pragma unroll
        for (int c = 0; c < kColumns; c += 2) {
          float2 de = make_float2(delta, delta);   // negative
          if constexpr (DKV) de = *reinterpret_cast<const float2*>(&ctl.stats[t & 1][1][group * kColumns + c]);
          float a, e;
          mul2(Pair(p[c], p[c + 1]), difference(Pair(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), Pair(de.x, de.y))).get(a, e);
          w[c / 2] = pack2<DT>(a, e);
          const float2 hi = unpack2<DT>(w[c / 2]);
          rest[c / 2] = pack2<DT>(a - hi.x, e - hi.y);
          if (!full) {
            w[c / 2] &= there(c);
            rest[c / 2] &= there(c);
          }
        }
        tmem_store16(at_dp, w);
        tmem_store16(at_dp + kColumns / 2, rest);
      } else {
#pragma unroll
        for (int c = 0; c < kColumns; c += 4) {
          float4 de = make_float4(delta, delta, delta, delta);   // negative
          if constexpr (DKV) de = *reinterpret_cast<const float4*>(&ctl.stats[t & 1][1][group * kColumns + c]);
          float a, e;
          mul2(Pair(p[c], p[c + 1]), difference(Pair(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), Pair(de.x, de.y))).get(a, e);
          w[c / 2] = pack2<DT>(a, e);
          mul2(Pair(p[c + 2], p[c + 3]), difference(Pair(__uint_as_float(d[c + 2]), __uint_as_float(d[c + 3])), Pair(de.z, de.w))).get(a, e);
          w[c / 2 + 1] = pack2<DT>(a, e);
        }
        if (!full) {
#pragma unroll
          for (int c = 0; c < kColumns; c += 2) w[c / 2] &= there(c);
        }
        tmem_store16(at_dp, w);
      }
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ctl.ds_full[t & 1]);
        if constexpr (DKV) mbar_arrive(&ctl.stat_free[t & 1]);
      }
    }
    if (ok && steps > 0) ok = wait_bar(&ctl.out_full, 0);
    __syncwarp();
    tc_fence_after();
    // DKV: the first half of the groups store dk, the others dv; else all store dq: an equal share of the
    // columns each.
    constexpr int SHARERS = DKV ? Shape::kGroups / 2 : Shape::kGroups, WIDTH = DP / SHARERS, CHUNK = WIDTH < 32 ? WIDTH : 32;
    const int which = group / SHARERS, c_first = group % SHARERS * WIDTH;
    const uint32_t t_out = (which ? t_out2 : t_out1) + lanes + c_first;
    const float weights = DT == NT_F16 && DKV ? power_of_two(-kWeightPower) : 1.0f;
    const float f = which ? weights : DT == NT_F16 ? P.scale / carried * weights : P.scale;
    const int row0 = r0 + (warp & 3) * 32;
    // The tiles of x1 and x2 are free now.
    uint8_t* stage = aligned + warp * 4096;
    if (parts == 1) {
      constexpr int CH = WIDTH / 8;
#pragma unroll
      for (int c = 0; c < WIDTH; c += CHUNK) {
        uint32_t v[CHUNK];
        if (steps > 0) {
          tmem_load(t_out + c, v);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int e = 0; e < CHUNK; ++e) v[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < CHUNK; e += 8) {
          uint32_t q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            q[k] = pack2<DT>(__uint_as_float(v[e + 2 * k]) * f, __uint_as_float(v[e + 2 * k + 1]) * f);
          stage_vector<CH>(stage, lane, (c + e) / 8, make_uint4(q[0], q[1], q[2], q[3]));
        }
      }
      char* dst = static_cast<char*>(DKV ? (which ? P.dv : P.dk) : P.dq);
      const AttnStrides& st = DKV ? (which ? P.dvs : P.dks) : P.dqs;
      store_staged<CH>(stage, lane, dst + (st.at(b, h0, row0) + c_first) * 2, st.t * 2, r1 - row0, (P.dim - c_first + 7) / 8);
    } else {
      // float32 [batch, key head, split block, part, 2, 128, dim]
      char* dst = reinterpret_cast<char*>(
          P.partial + (((((int64_t)b * P.kv_heads + h0) * attn_joined(P, (P.keys + kTcKeyRows - 1) / kTcKeyRows) + index) * 2 + which) * kTcRows +
                       (warp & 3) * 32) * P.dim + c_first);
      constexpr int CH = CHUNK / 4;
#pragma unroll
      for (int c = 0; c < WIDTH; c += CHUNK) {
        uint32_t v[CHUNK];
        if (steps > 0) {
          tmem_load(t_out + c, v);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int e = 0; e < CHUNK; ++e) v[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < CHUNK; e += 4)
          stage_vector<CH>(stage, lane, e / 4,
                           make_uint4(__float_as_uint(__uint_as_float(v[e]) * f), __float_as_uint(__uint_as_float(v[e + 1]) * f),
                                      __float_as_uint(__uint_as_float(v[e + 2]) * f), __float_as_uint(__uint_as_float(v[e + 3]) * f)));
        store_staged<CH>(stage, lane, dst + c * 4, (int64_t)P.dim * 4, 32, (P.dim - c_first - c + 3) / 4);
      }
    }
  }
  if (!ok && P.error != nullptr) atomicOr(P.error, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_free(tmem, Shape::kTmem);
}

// `key_blocks` blocks own keys, the others queries. The longer kind comes first: the key blocks, unless
// all of them are cut (4 heads on one key head, 6508 tokens of 64: 138 us with the cut ones first, 103
// with the query blocks). FINE is a variant of its own: see the top of this file.
template <int DT, int DP, bool FINE>
__global__ void __launch_bounds__(BwdShared<DP>::kThreads, BwdShared<DP>::kResident)
attention_tc_backward(const __grid_constant__ AttnParams P, uint32_t key_blocks, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v) {
  const bool keys_first = P.rest == 1;
  const uint32_t split = keys_first ? key_blocks : gridDim.x - key_blocks;
  const uint32_t index = blockIdx.x < split ? blockIdx.x : blockIdx.x - split;
  if ((blockIdx.x < split) == keys_first) backward_block<DT, DP, true, FINE>(P, index, map_k, map_v, map_q, map_g);
  else backward_block<DT, DP, false, FINE>(P, index, map_q, map_g, map_k, map_v);
}

// ---- host ------------------------------------------------------------------------------

template <int DT, int DP, bool SPLIT>
static int launch_tc_forward(const AttnParams& P, unsigned blocks, cudaStream_t s) {
  const char* who = "nt_attention_forward";
  CUtensorMap q, k, v;
  int rc = large_smem<attention_tc_forward<DT, DP, SPLIT>>(FwdShared<DP>::kBytes, who);
  if (!rc) rc = make_map(&q, DT, P.q, P.qs, P.dim, P.queries, P.heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&k, DT, P.k, P.ks, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&v, DT, P.v, P.vs, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (rc) return rc;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks * (SPLIT ? P.splits : 1));
  config.blockDim = dim3(FwdShared<DP>::kThreads);
  config.dynamicSmemBytes = FwdShared<DP>::kBytes;
  config.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = SPLIT ? P.splits : 1;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = SPLIT ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&config, attention_tc_forward<DT, DP, SPLIT>, P, q, k, v);
  if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, who); }
  return launch_status("nt_attention_forward launch");
}

// Blocks of a cluster that share the tiles of one block of queries: more of them while the longest
// block is more than 1.5 times an SM's share of all tiles (1.25 times where a second block on the SM slows
// it: 6508 tokens, 4 heads of 64 on one, 68 us at 1.5, 58 at 1.25), with two tiles at least to each (512
// queries of 16 heads after 7680 keys, window 2048: 39 us in 32 blocks, 23 in clusters of 4). Clusters
// of 8 only where they all run at once: a second wave of them waits for 8 free SMs side by side (58 us).
template <int DT, int DP>
static int dispatch_tc_forward(AttnParams P, cudaStream_t s) {
  constexpr int rows = FwdShared<DP>::kRows;
  const unsigned blocks = (unsigned)((P.queries + rows - 1) / rows) * P.heads * P.batch;
  const int64_t end = (int64_t)P.offset + P.queries;
  int64_t longest = end < P.keys ? end : P.keys, mean = longest;
  if (P.window > 0 && (int64_t)P.window + rows + P.sinks < longest) longest = mean = (int64_t)P.window + rows + P.sinks;
  else if (P.offset + P.queries / 2 < mean) mean = P.offset + P.queries / 2;
  const int sms = current_sm_count(), quarters = FwdShared<DP>::kResident == 2 ? 5 : 6;
  P.splits = 1;
  while (P.splits < kMaxSplits && longest >= (int64_t)4 * P.splits * kTcRows &&
         longest * sms * 4 > quarters * (int64_t)blocks * mean * P.splits &&
         (P.splits < 4 || (int64_t)blocks * P.splits * 2 <= sms))
    P.splits *= 2;
  return P.splits > 1 ? launch_tc_forward<DT, DP, true>(P, blocks, s) : launch_tc_forward<DT, DP, false>(P, blocks, s);
}

template <int DT, int DP, bool FINE>
static int launch_tc_backward(const AttnParams& P, cudaStream_t s) {
  const char* who = "nt_attention_backward";
  CUtensorMap q, g, k, v;
  const int bytes = BwdShared<DP>::kBytes;
  int rc = large_smem<attention_tc_backward<DT, DP, FINE>>(bytes, who);
  if (!rc) rc = make_map(&q, DT, P.q, P.qs, P.dim, P.queries, P.heads, P.batch, BwdShared<DP>::kStep, who);
  if (!rc) rc = make_map(&g, DT, P.g, P.gs, P.dim, P.queries, P.heads, P.batch, BwdShared<DP>::kStep, who);
  if (!rc) rc = make_map(&k, DT, P.k, P.ks, P.dim, P.keys, P.kv_heads, P.batch, BwdShared<DP>::kStep, who);
  if (!rc) rc = make_map(&v, DT, P.v, P.vs, P.dim, P.keys, P.kv_heads, P.batch, BwdShared<DP>::kStep, who);
  if (rc) return rc;
  if constexpr (DT == NT_F16) {
    const int entries = norm_tiles(P.queries, DP) + norm_tiles(P.keys, DP);
    attention_delta_norms_kernel<DP><<<dim3(entries, P.heads, P.batch), 256, 0, s>>>(P);
  } else {
    constexpr int ROWS = 256 / (DP / 8);
    attention_delta_kernel<DT, DP><<<dim3((P.queries + ROWS - 1) / ROWS, P.heads, P.batch), 256, 0, s>>>(P);
  }
  rc = launch_status("nt_attention_backward launch");
  if (rc) return rc;
  const uint32_t query_blocks = (uint32_t)((P.queries + kTcRows - 1) / kTcRows) * P.heads * P.batch;
  const uint32_t key_blocks =
      (uint32_t)attn_pieces(P, (P.keys + kTcKeyRows - 1) / kTcKeyRows) * P.kv_heads * P.batch;
  // Its blocks may start while the kernel before it ends.
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(key_blocks + query_blocks);
  config.blockDim = dim3(BwdShared<DP>::kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&config, attention_tc_backward<DT, DP, FINE>, P, key_blocks, q, g, k, v);
  if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, "nt_attention_backward launch"); }
  return launch_status("nt_attention_backward launch");
}

int attention_tc_forward_launch(const AttnParams& P, int dtype, cudaStream_t s) {
  if (dtype == NT_BF16) return P.dim <= 64 ? dispatch_tc_forward<NT_BF16, 64>(P, s) : dispatch_tc_forward<NT_BF16, 128>(P, s);
  return P.dim <= 64 ? dispatch_tc_forward<NT_F16, 64>(P, s) : dispatch_tc_forward<NT_F16, 128>(P, s);
}

template <int DT, int DP>
static int dispatch_tc_backward(const AttnParams& P, cudaStream_t s) {
  const bool fine = P.lengths != nullptr || P.queries <= kShortQueries || P.keys <= kFineKeys || (P.window > 0 && (int64_t)P.window + P.sinks <= kFineKeys);
  return fine ? launch_tc_backward<DT, DP, true>(P, s) : launch_tc_backward<DT, DP, false>(P, s);
}

int attention_tc_backward_launch(const AttnParams& P, int dtype, cudaStream_t s) {
  if (dtype == NT_BF16) return P.dim <= 64 ? dispatch_tc_backward<NT_BF16, 64>(P, s) : dispatch_tc_backward<NT_BF16, 128>(P, s);
  return P.dim <= 64 ? dispatch_tc_backward<NT_F16, 64>(P, s) : dispatch_tc_backward<NT_F16, 128>(P, s);
}

}  // namespace nt
