// Sliding-window attention on the fifth-generation tensor cores, for float16 and bfloat16 rows
// that are whole 16-byte vectors. The mathematics and the masks are those of nt_attention.cu.
//
// Forward: a block owns 128 queries of one head and walks its visible keys 128 at a time. One
// warp copies tiles, one issues the products, eight do the softmax: two threads share a query's
// row, 64 columns each. S = q k^T accumulates in TMEM; the weights go back to TMEM over S as
// 16-bit values and are the first operand of o += w v. Two blocks share an SM, so one's products
// run under the other's exponentials.
//
// Backward: two passes of one kernel (see attention_tc_backward), each with S and dP computed
// again. Sums that cross blocks exist only for the sink keys and are added in order afterwards.
//
// Roundings below 32 bits: the weights and dS are rounded to the inputs' type because the second
// products take their operand in it; every sum, maximum and statistic is float32.
#include <cmath>

#include "nt_attention.cuh"
#include "nt_tc.cuh"

namespace nt {

constexpr int kTcRows = 128;
constexpr int kTcThreads = 320;        // 8 computing warps, 1 copying, 1 issuing products
constexpr int kCopyWarp = 8, kMmaWarp = 9;
constexpr uint32_t kFwdColumns = 256;  // TMEM: S (and the weights over it) 128, output up to 128
constexpr float kRescaleLog2 = 8.0f;

// A wait of a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity));
}

template <int DP> struct FwdShared {
  static constexpr int kTile = kTcRows * DP * 2;
  static constexpr int kBytes = 3 * kTile + 1024;
};

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

template <int DT, int DP>
__global__ void __launch_bounds__(kTcThreads, 2)
attention_tc_forward(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t q_full, k_full, k_free, v_full, v_free, s_full, w_full, o_full;
  __shared__ uint32_t tmem_slot;
  __shared__ float exchange[2][2][kTcRows];
  constexpr int TILE = FwdShared<DP>::kTile;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* aligned = raw + (base - smem_u32(raw));
  const uint32_t sq = base, sk = base + TILE, sv = base + 2 * TILE;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Blocks in the order of their work: the last queries of every head first.
  const uint32_t pairs = (uint32_t)P.heads * P.batch, tiles = gridDim.x / pairs;
  const int b = blockIdx.x % pairs / P.heads, h = blockIdx.x % P.heads, hk = h / P.group;
  const int i0 = (tiles - 1 - blockIdx.x / pairs) * kTcRows, i1 = min(P.queries, i0 + kTcRows);
  const int length = attn_length(P, b);
  const AttnKeys range(P, length, i0, i1);
  const int blocks = range.blocks(kTcRows);

  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, kFwdColumns);
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1); mbar_init(&k_full, 1); mbar_init(&k_free, 1); mbar_init(&v_full, 1); mbar_init(&v_free, 1);
    mbar_init(&s_full, 1); mbar_init(&w_full, 8); mbar_init(&o_full, 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t t_s = tmem, t_o = tmem + kTcRows;
  bool ok = true;

  if (warp == kCopyWarp) {
    if (lane == 0 && blocks > 0) {
      auto load = [&](const CUtensorMap* map, int offset, int token, int head, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
        for (int half = 0; half < DP / 64; ++half)
          tma_load(aligned + offset + half * kTcRows * 128, map, half * 64, token, head, b, bar);
      };
      load(&map_q, 0, i0, h, &q_full);
      int issued = 0;
      for (int j = 0; j < blocks && ok; ++j) {
        int begin, end;
        range.block(j, kTcRows, begin, end);
        if (j > 0) ok = wait_bar(&k_free, (j - 1) & 1);
        if (!ok) break;
        load(&map_k, TILE, begin, hk, &k_full);
        if (j > 0) ok = wait_bar(&v_free, (j - 1) & 1);
        if (!ok) { wait_bar(&k_full, j & 1); break; }
        load(&map_v, 2 * TILE, begin, hk, &v_full);
        issued = j + 1;
      }
      if (!ok) {   // the copies in flight land before the block may end
        wait_bar(&q_full, 0);
        if (issued > 0) { wait_bar(&k_full, (issued - 1) & 1); wait_bar(&v_full, (issued - 1) & 1); }
      }
    }
  } else if (warp == kMmaWarp) {
    const int width16 = (P.dim + 15) / 16;
    const uint32_t pv = tc_instruction<DT>(width16 * 16, true);
    const uint64_t dq = tc_columns(sq), dk = tc_columns(sk), dv = tc_rows(sv, kTcRows);
    if (blocks > 0) ok = wait_warp(&q_full, 0);
    for (int j = 0; j < blocks && ok; ++j) {
      int begin, end;
      range.block(j, kTcRows, begin, end);
      const int keys16 = (end - begin + 15) / 16;
      ok = wait_warp(&k_full, j & 1);
      if (!ok) break;
      if (elect_one()) {
        const uint32_t qk = tc_instruction<DT>(keys16 * 16, false);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          if (s < width16) tc_mma(t_s, dq + tc_column_step(kTcRows, s), dk + tc_column_step(kTcRows, s), qk, s > 0);
        tc_commit(&s_full);
        tc_commit(&k_free);
      }
      __syncwarp();
      ok = wait_warp(&v_full, j & 1);
      if (!ok) break;
      // Rows between the last visible key and the end of its group of 16 have weight 0 but may
      // hold anything: 0 * NaN must not reach the sum.
      const int tail = keys16 * 16 - (end - begin);
      if (tail > 0) {
        for (int i = lane; i < tail * (DP / 8); i += 32) {
          const int row = end - begin + i / (DP / 8), c = i % (DP / 8);
          *reinterpret_cast<uint4*>(aligned + 2 * TILE + (c / 8) * kTcRows * 128 + row * 128 + (c % 8) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      }
      ok = wait_warp(&w_full, j & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < kTcRows / 16; ++s)
          if (s < keys16) tc_mma_tmem(t_o, t_s + s * 8, dv + tc_row_step(s), pv, j > 0 || s > 0);
        tc_commit(&v_free);
      }
      __syncwarp();
    }
    if (elect_one()) tc_commit(&o_full);
    __syncwarp();
    if (!ok) wait_bar(&o_full, 0);   // no product is in flight when TMEM is given back
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // lane 32 (w % 4) in the address's upper half
    const int p = P.offset + i0 + row;
    const int p_first = P.offset + i0, p_last = P.offset + i1 - 1;
    const int sinks = range.sink_blocks(kTcRows);
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < blocks; ++j) {
      int begin, end;
      range.block(j, kTcRows, begin, end);
      // A wait that ran out is remembered and not waited for again; the warp still takes part in
      // every barrier, so that no other warp is left waiting for it.
      if (ok) ok = wait_bar(&s_full, j & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t r0[32], r1[32];
      tmem_load32(t_s + lanes + half * 64, r0);
      tmem_load32(t_s + lanes + half * 64 + 32, r1);
      tmem_wait_load();
      float s[64];
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        s[c] = __uint_as_float(r0[c]);
        s[32 + c] = __uint_as_float(r1[c]);
      }
      const bool full = end - begin == kTcRows && end - 1 <= p_first &&
                        (P.window == 0 || j < sinks || p_last - begin < P.window);
      if (!full) {
        const ColumnMask mask{P.window == 0 ? 0 : p - P.window + 1 - begin - half * 64, min(end, p + 1) - begin - half * 64,
                              P.sinks - begin - half * 64};
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          const uint32_t seen = mask.word(c0);
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c0 + c] = seen >> c & 1 ? s[c0 + c] : -INFINITY;
        }
      }
      float top = s[0], top1 = s[1];
#pragma unroll
      for (int c = 2; c < 64; c += 2) {
        top = fmaxf(top, s[c]);
        top1 = fmaxf(top1, s[c + 1]);
      }
      top = fmaxf(top, top1);
      exchange[j & 1][half][row] = top;
      named_barrier(1 + (warp & 3), 64);
      top = fmaxf(top, exchange[j & 1][half ^ 1][row]);
      // The maximum only has to keep the weights in range, so the old one stays until the new is
      // 2^8 above it: the output is then rescaled for a few of the first tiles of a row only.
      const bool raise = top > m && !((top - m) * P.scale_log2 <= kRescaleLog2);
      if (__any_sync(0xffffffffu, raise)) {
        const float f = raise ? ex2_approx((m - top) * P.scale_log2) : 1.0f;
        if (raise) m = top;
        l *= f;
        if (j > 0) {
          // Products complete in order: S of this tile is there, so o of the last one is too.
#pragma unroll
          for (int c = 0; c < DP / 2; c += 32) {
            uint32_t o[32];
            tmem_load32(t_o + lanes + half * (DP / 2) + c, o);
            tmem_wait_load();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_store32(t_o + lanes + half * (DP / 2) + c, o);
          }
        }
      }
      float shift = m == -INFINITY ? 0.0f : m;
      if (__any_sync(0xffffffffu, isinf(shift * P.scale_log2))) {
        // Scores near the ends of float32: subtract before scaling.
#pragma unroll
        for (int c = 0; c < 64; ++c) s[c] -= shift;
        shift = 0.0f;
      }
      const float minus = -shift * P.scale_log2;
      float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = ex2_approx(fmaf(s[c + 2 * e], P.scale_log2, minus));
          const float y = ex2_approx(fmaf(s[c + 2 * e + 1], P.scale_log2, minus));
          sum0 += x;
          sum1 += y;
          w[e] = pack2<DT>(x, y);
        }
        tmem_store16(t_s + lanes + half * 32 + c / 2, w);
      }
      l += sum0 + sum1;
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w_full);
    }
    if (ok && blocks > 0) ok = wait_bar(&o_full, 0);
    __syncwarp();
    tc_fence_after();
    exchange[blocks & 1][half][row] = l;
    named_barrier(1 + (warp & 3), 64);
    // Halves in a fixed order, so that both threads of a row have the same sum.
    l = exchange[blocks & 1][0][row] + exchange[blocks & 1][1][row];
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    const bool live = i0 + row < i1;
    uint16_t* out = static_cast<uint16_t*>(P.o) + P.os.at(b, h, i0 + row) + half * (DP / 2);
    uint16_t* low = P.o_low == nullptr ? nullptr
                                       : static_cast<uint16_t*>(P.o_low) + P.os.at(b, h, i0 + row) + half * (DP / 2);
#pragma unroll
    for (int c = 0; c < DP / 2; c += 32) {
      uint32_t o[32];
      if (blocks > 0) {
        tmem_load32(t_o + lanes + half * (DP / 2) + c, o);
        tmem_wait_load();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        if (!live || half * (DP / 2) + c + e >= P.dim) continue;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // A row without keys is 0 whatever the accumulator holds.
          const float x = f == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * k]) * f;
          const float y = f == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * k + 1]) * f;
          hi[k] = pack2<DT>(x, y);
          const float2 r = unpack2<DT>(hi[k]);
          lo[k] = pack2<DT>(x - r.x, y - r.y);
        }
        *reinterpret_cast<uint4*>(out + c + e) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (low != nullptr) *reinterpret_cast<uint4*>(low + c + e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    if (live && half == 0 && P.lse != nullptr)
      P.lse[((int64_t)b * P.heads + h) * P.queries + i0 + row] =
          l == 0.0f ? -INFINITY : fmaf(m, P.scale, log2f(l) * kLn2F);
  }
  if (!ok && P.error != nullptr) atomicOr(P.error, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_free(tmem, kFwdColumns);
}

// ---- backward ------------------------------------------------------------------------
// One block keeps 128 rows x1, x2 and walks rows y1, y2 128 at a time:
//   s = x1 y1^T, dp = x2 y2^T (TMEM, float32);  P = exp(scale s - lse), dS = P (dp - delta)
//   out1 += dS y1, and with DKV out2 += P y2, with P and dS over s and dp in TMEM as the
//   products' first operand.
// DKV = false: rows are queries (x1 = q, x2 = g; y1 = k, y2 = v): out1 = dq; delta = sum(g o) is
// computed on the way in and stored. DKV = true: rows are keys (x1 = k, x2 = v; y1 = q, y2 = g):
// out1 = dk, out2 = dv, over the heads of the group.
// s, dp and the two outputs fill TMEM, so nothing has a second buffer; the order of the products
// hides the exponentials instead: dp(t) runs while P(t) is computed, out2(t) and s(t + 1) while
// dS(t) is, out1(t) and dp(t + 1) while P(t + 1) is. Two groups of four warps take 64 columns each.
constexpr int kStep = kTcQueryStep;
constexpr uint32_t kBwdColumns = 512;

constexpr int kBwdThreads = 352;       // 8 computing warps, 1 copying, 1 issuing products, 1 for lse and delta
constexpr int kStatWarp = 10;

// Shared memory: x1, x2, the ring of y1 (three: s of the next step starts before out1 of this one
// has ended), the ring of y2 (two) and the control block.
template <int DP> struct BwdShared {
  static constexpr int kTile = kTcRows * DP * 2;
  static constexpr int kRing1 = 3, kRing2 = 2;
  static constexpr int kY1 = 2 * kTile, kY2 = (2 + kRing1) * kTile, kControl = (2 + kRing1 + kRing2) * kTile;
  struct Control {
    float stats[2][2][kStep];          // ring of two; lse (times log2 e), delta
    uint64_t x_full, y1_full[kRing1], y1_free[kRing1], y2_full[kRing2], y2_free[kRing2], s_full, dp_full, p_full, ds_full,
        stat_full[2], stat_free[2], out_full;
    uint32_t tmem;
  };
  static constexpr int kBytes = kControl + (int)sizeof(Control);
};
static_assert(kStep == kTcRows, "rows kept and rows streamed have one shape");
static_assert(BwdShared<128>::kBytes <= 227 * 1024, "one block per SM");

// Phase of slot use n of a ring of `size`.
__device__ __forceinline__ uint32_t ring_phase(int n, int size) { return (uint32_t)(n / size) & 1u; }

template <int DT, int DP, bool DKV>
__global__ void __launch_bounds__(kBwdThreads, 1)
attention_tc_backward(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap map_x1,
                      const __grid_constant__ CUtensorMap map_x2, const __grid_constant__ CUtensorMap map_y1,
                      const __grid_constant__ CUtensorMap map_y2) {
  using Shape = BwdShared<DP>;
  constexpr int TILE = Shape::kTile, RING1 = Shape::kRing1, RING2 = Shape::kRing2;
  // No static shared memory: the dynamic block starts where shared memory does, 1024 bytes in.
  extern __shared__ __align__(1024) uint8_t aligned[];
  typename Shape::Control& ctl = *reinterpret_cast<typename Shape::Control*>(aligned + Shape::kControl);
  const uint32_t base = smem_u32(aligned);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Blocks in the order of their work: the last queries, or the first keys, of every head first.
  const uint32_t heads = DKV ? P.kv_heads : P.heads, pairs = heads * P.batch, tiles = gridDim.x / pairs;
  const int b = blockIdx.x % pairs / heads, h0 = blockIdx.x % heads;   // query head of dq, key head of dk and dv
  const int index = blockIdx.x / pairs;
  const int length = attn_length(P, b);

  // The block's rows [r0, r1) and the steps it walks.
  int r0, r1, part = 0, parts = 1, tile = 0, steps, per_head = 1;
  uint32_t from = 0;
  if constexpr (!DKV) {
    r0 = (tiles - 1 - index) * kTcRows;
    r1 = min(P.queries, r0 + kTcRows);
  } else {
    const int split = P.sink_tiles * P.parts;
    tile = index < split ? index / P.parts : index - split + P.sink_tiles;
    part = index < split ? index % P.parts : 0;
    parts = index < split ? P.parts : 1;
    r0 = tile * kTcRows;
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

  if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, kBwdColumns);
  if (threadIdx.x == 0) {
    mbar_init(&ctl.x_full, 1); mbar_init(&ctl.out_full, 1);
#pragma unroll
    for (int i = 0; i < RING1; ++i) { mbar_init(&ctl.y1_full[i], 1); mbar_init(&ctl.y1_free[i], 1); }
#pragma unroll
    for (int i = 0; i < RING2; ++i) {
      mbar_init(&ctl.y2_full[i], 1); mbar_init(&ctl.y2_free[i], 1);
      mbar_init(&ctl.stat_full[i], 1); mbar_init(&ctl.stat_free[i], 8);
    }
    mbar_init(&ctl.s_full, 1); mbar_init(&ctl.dp_full, 1); mbar_init(&ctl.p_full, 8); mbar_init(&ctl.ds_full, 8);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  const uint32_t t_s = tmem, t_dp = tmem + kStep, t_out1 = tmem + 2 * kStep, t_out2 = t_out1 + DP;
  bool ok = true;

  if (warp == kCopyWarp) {
    if (lane == 0 && steps > 0) {
      auto load = [&](const CUtensorMap* map, int at, int token, int head, uint64_t* bar) {
#pragma unroll
        for (int half = 0; half < DP / 64; ++half)
          tma_load(aligned + at + half * kTcRows * 128, map, half * 64, token, head, b, bar);
      };
      mbar_arrive_expect_tx(&ctl.x_full, 2 * TILE);
      load(&map_x1, 0, r0, h0, &ctl.x_full);
      load(&map_x2, TILE, r0, h0, &ctl.x_full);
      Step s;
      start(s);
      int n1 = 0, n2 = 0;
      for (int t = 0; t < steps; ++t, advance(s)) {
        if (t >= RING1) ok = wait_bar(&ctl.y1_free[t % RING1], ring_phase(t - RING1, RING1));
        if (!ok) break;
        mbar_arrive_expect_tx(&ctl.y1_full[t % RING1], TILE);
        load(&map_y1, Shape::kY1 + t % RING1 * TILE, s.begin, s.head, &ctl.y1_full[t % RING1]);
        n1 = t + 1;
        if (t >= RING2) ok = wait_bar(&ctl.y2_free[t % RING2], ring_phase(t - RING2, RING2));
        if (!ok) break;
        mbar_arrive_expect_tx(&ctl.y2_full[t % RING2], TILE);
        load(&map_y2, Shape::kY2 + t % RING2 * TILE, s.begin, s.head, &ctl.y2_full[t % RING2]);
        n2 = t + 1;
      }
      if (!ok) {   // the copies in flight land before the block may end
        wait_bar(&ctl.x_full, 0);
        for (int i = max(0, n1 - RING1); i < n1; ++i) wait_bar(&ctl.y1_full[i % RING1], ring_phase(i, RING1));
        for (int i = max(0, n2 - RING2); i < n2; ++i) wait_bar(&ctl.y2_full[i % RING2], ring_phase(i, RING2));
      }
    }
  } else if (warp == kStatWarp) {
    if constexpr (DKV) {
      Step s;
      start(s);
      for (int t = 0; t < steps; ++t, advance(s)) {
        const int64_t stat = ((int64_t)b * P.heads + s.head) * P.queries + s.begin;
        float lse[kStep / 32], delta[kStep / 32];
#pragma unroll
        for (int i = 0; i < kStep / 32; ++i) {
          const int c = i * 32 + lane;
          const bool in = s.begin + c < s.end;
          lse[i] = in ? P.lse[stat + c] * kLog2eF : 0.0f;
          delta[i] = in ? P.delta[stat + c] : 0.0f;
        }
        if (t >= 2) ok = wait_warp(&ctl.stat_free[t & 1], ring_phase(t - 2, 2));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kStep / 32; ++i) {
          ctl.stats[t & 1][0][i * 32 + lane] = lse[i];
          ctl.stats[t & 1][1][i * 32 + lane] = delta[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.stat_full[t & 1]);
      }
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
    // acc += w y of one step, which ends its use of y; w lies in two halves of 64 columns
    auto sum = [&](uint32_t acc, uint32_t w, int at, int rows, bool add, uint64_t* done) {
      if (elect_one()) {
        const uint64_t y = tc_rows(base + at, kStep);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          if (k * 16 < rows)
            tc_mma_tmem(acc, w + (k >> 2) * 64 + (k & 3) * 8, y + tc_row_step(k), accumulate, add || k > 0);
        tc_commit(done);
      }
      __syncwarp();
    };
    // Waits for a tile and clears its rows between the step's end and the end of its group of 16:
    // their weights are 0, but 0 * NaN must not reach a sum.
    auto arrive = [&](uint64_t* bar, uint32_t phase, int at, int rows) {
      if (!wait_warp(bar, phase)) return false;
      const int tail = (rows + 15) / 16 * 16 - rows;
      if (tail > 0) {
        for (int i = lane; i < tail * (DP / 8); i += 32) {
          const int row = rows + i / (DP / 8), c = i % (DP / 8);
          *reinterpret_cast<uint4*>(aligned + at + (c / 8) * kStep * 128 + row * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      }
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
    for (int t = 0; t < steps && ok; ++t) {
      const int y1 = Shape::kY1 + t % RING1 * TILE, y2 = Shape::kY2 + t % RING2 * TILE;
      ok = arrive(&ctl.y2_full[t % RING2], ring_phase(t, RING2), y2, rows);
      if (!ok) break;
      product(t_dp, x2, y2, rows, &ctl.dp_full);
      if constexpr (!DKV) {   // nothing else reads y2
        if (elect_one()) tc_commit(&ctl.y2_free[t % RING2]);
        __syncwarp();
      }
      ok = wait_warp(&ctl.p_full, t & 1);
      if (!ok) break;
      tc_fence_after();
      if constexpr (DKV) sum(t_out2, t_s, y2, rows, t > 0, &ctl.y2_free[t % RING2]);
      const int now = rows;
      if (t + 1 < steps) {
        advance(s);
        rows = s.end - s.begin;
        const int next = Shape::kY1 + (t + 1) % RING1 * TILE;
        ok = arrive(&ctl.y1_full[(t + 1) % RING1], ring_phase(t + 1, RING1), next, rows);
        if (!ok) break;
        product(t_s, x1, next, rows, &ctl.s_full);
      }
      ok = wait_warp(&ctl.ds_full, t & 1);
      if (!ok) break;
      tc_fence_after();
      sum(t_out1, t_dp, y1, now, t > 0, &ctl.y1_free[t % RING1]);
    }
    if (elect_one()) tc_commit(&ctl.out_full);
    __syncwarp();
    if (!ok) wait_bar(&ctl.out_full, 0);
  } else {
    const int group = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    float lse = 0.0f, delta = 0.0f;
    if constexpr (!DKV) {
      // delta of the row: each of its two threads sums half of the columns.
      const int64_t stat = ((int64_t)b * P.heads + h0) * P.queries + r0 + row;
      const bool live = r0 + row < r1;
      float d = 0.0f;
      if (live) {
        const uint16_t* g = static_cast<const uint16_t*>(P.g) + P.gs.at(b, h0, r0 + row);
        const uint16_t* o = static_cast<const uint16_t*>(P.o) + P.os.at(b, h0, r0 + row);
        const uint16_t* low = P.o_low == nullptr ? nullptr : static_cast<const uint16_t*>(P.o_low) + P.os.at(b, h0, r0 + row);
#pragma unroll
        for (int c = 0; c < DP / 2; c += 8) {
          const int at = group * (DP / 2) + c;
          if (at >= P.dim) break;
          float x[8], y[8], z[8];
          unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(g + at)), x);
          unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(o + at)), y);
          if (low != nullptr) unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(low + at)), z);
#pragma unroll
          for (int e = 0; e < 8; ++e) d = fmaf(x[e], low != nullptr ? y[e] + z[e] : y[e], d);
        }
        lse = P.lse[stat] * kLog2eF;
      }
      float* halves = &ctl.stats[0][0][0];
      halves[group * kTcRows + row] = d;
      named_barrier(1, 256);
      delta = halves[row] + halves[kTcRows + row];
      if (live && group == 0) P.delta[stat] = delta;
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
      float p[64];
      {
        uint32_t s0[32], s1[32];
        tmem_load32(t_s + lanes + group * 64, s0);
        tmem_load32(t_s + lanes + group * 64 + 32, s1);
        tmem_wait_load();
        if constexpr (!DKV) {   // s may be overwritten
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.p_full);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          p[c] = __uint_as_float(s0[c]);
          p[32 + c] = __uint_as_float(s1[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        float4 ls = make_float4(lse, lse, lse, lse);
        if constexpr (DKV) ls = *reinterpret_cast<const float4*>(&ctl.stats[t & 1][0][group * 64 + c]);
        p[c] = ex2_approx(fmaf(p[c], P.scale_log2, -ls.x));
        p[c + 1] = ex2_approx(fmaf(p[c + 1], P.scale_log2, -ls.y));
        p[c + 2] = ex2_approx(fmaf(p[c + 2], P.scale_log2, -ls.z));
        p[c + 3] = ex2_approx(fmaf(p[c + 3], P.scale_log2, -ls.w));
      }
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
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
        seen[0] = mask.word(group * 64);
        seen[1] = mask.word(group * 64 + 32);
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
#pragma unroll
          for (int c = 0; c < 32; ++c) p[c0 + c] = seen[c0 / 32] >> c & 1 ? p[c0 + c] : 0.0f;
        }
      }
      if constexpr (DKV) {
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack2<DT>(p[c0 + 2 * e], p[c0 + 2 * e + 1]);
          tmem_store16(t_s + lanes + group * 64 + c0 / 2, w);
        }
        tmem_wait_store();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full);
      }
      if (ok) ok = wait_bar(&ctl.dp_full, t & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t w[32];
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 32) {
        uint32_t d[32];
        tmem_load32(t_dp + lanes + group * 64 + c0, d);
        tmem_wait_load();
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          float4 de = make_float4(delta, delta, delta, delta);
          if constexpr (DKV) de = *reinterpret_cast<const float4*>(&ctl.stats[t & 1][1][group * 64 + c0 + c]);
          const float a = p[c0 + c] * (__uint_as_float(d[c]) - de.x), e = p[c0 + c + 1] * (__uint_as_float(d[c + 1]) - de.y);
          const float f = p[c0 + c + 2] * (__uint_as_float(d[c + 2]) - de.z),
                      g = p[c0 + c + 3] * (__uint_as_float(d[c + 3]) - de.w);
          w[(c0 + c) / 2] = pack2<DT>(a, e);
          w[(c0 + c) / 2 + 1] = pack2<DT>(f, g);
        }
        if (!full) {
          // dp of a key that is not there may be NaN: 0 * NaN is cleared here.
#pragma unroll
          for (int c = 0; c < 32; c += 2)
            w[(c0 + c) / 2] &= (seen[c0 / 32] >> c & 1 ? 0xffffu : 0u) | (seen[c0 / 32] >> (c + 1) & 1 ? 0xffff0000u : 0u);
        }
      }
      tmem_store32(t_dp + lanes + group * 64, w);
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ctl.ds_full);
        if constexpr (DKV) mbar_arrive(&ctl.stat_free[t & 1]);
      }
    }
    if (ok && steps > 0) ok = wait_bar(&ctl.out_full, 0);
    __syncwarp();
    tc_fence_after();
    // DKV: the first group stores dk, the second dv; else half of dq's columns each.
    const bool live = r0 + row < r1;
    constexpr int WIDTH = DKV ? DP : DP / 2;
    const int c_first = DKV ? 0 : group * WIDTH;
    const uint32_t t_out = (DKV && group == 1 ? t_out2 : t_out1) + lanes + c_first;
    const float f = DKV && group == 1 ? 1.0f : P.scale;
#pragma unroll
    for (int c = 0; c < WIDTH; c += 32) {
      uint32_t v[32];
      if (steps > 0) {
        tmem_load32(t_out + c, v);
        tmem_wait_load();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
      }
      if (parts == 1) {
        void* dst = DKV ? (group == 0 ? P.dk : P.dv) : P.dq;
        const AttnStrides& st = DKV ? (group == 0 ? P.dks : P.dvs) : P.dqs;
        uint16_t* out = static_cast<uint16_t*>(dst) + st.at(b, h0, r0 + row) + c_first + c;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (!live || c_first + c + e >= P.dim) continue;
          uint32_t q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            q[k] = pack2<DT>(__uint_as_float(v[e + 2 * k]) * f, __uint_as_float(v[e + 2 * k + 1]) * f);
          *reinterpret_cast<uint4*>(out + e) = make_uint4(q[0], q[1], q[2], q[3]);
        }
      } else {
        // [batch, key head, sink block, part, 2, 128, dim]
        float* out = P.partial + (((((int64_t)b * P.kv_heads + h0) * P.sink_tiles + tile) * parts + part) * 2 + group) *
                                     kTcRows * P.dim + (int64_t)row * P.dim + c;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          if (c + e >= P.dim) continue;
          *reinterpret_cast<float4*>(out + e) =
              make_float4(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f, __uint_as_float(v[e + 2]) * f,
                          __uint_as_float(v[e + 3]) * f);
        }
      }
    }
  }
  if (!ok && P.error != nullptr) atomicOr(P.error, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_free(tmem, kBwdColumns);
}

// ---- host ------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// (column, token, head, batch) of one tensor, boxes of 64 columns x `rows` tokens, zeros outside.
static int make_map(CUtensorMap* map, int dtype, const void* ptr, const AttnStrides& st, int dim, int tokens, int heads,
                    int batch, int rows, const char* who) {
  EncodeTiled encode = encode_tiled();
  if (!encode) { set_error("%s: the driver has no cuTensorMapEncodeTiled", who); return NT_ECUDA; }
  const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
  // The stride of a dimension of one element is never used, but has to be a valid one.
  const cuuint64_t row_bytes = ((cuuint64_t)dim * 2 + 15) / 16 * 16;
  const cuuint64_t strides[3] = {tokens > 1 ? (cuuint64_t)st.t * 2 : row_bytes, heads > 1 ? (cuuint64_t)st.h * 2 : row_bytes,
                                 batch > 1 ? (cuuint64_t)st.b * 2 : row_bytes};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult rc = encode(map, dtype == NT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                             const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) { set_error("%s: cuTensorMapEncodeTiled failed (%d)", who, (int)rc); return NT_ECUDA; }
  return NT_OK;
}

template <typename K>
static int large_smem(K kernel, int bytes, const char* who) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? NT_OK : cuda_fail(e, who);
}

template <int DT, int DP>
static int launch_tc_forward(const AttnParams& P, cudaStream_t s) {
  const char* who = "nt_attention_forward";
  CUtensorMap q, k, v;
  // A runtime call first: the map encoder is a driver call and needs a context on this thread.
  int rc = large_smem(attention_tc_forward<DT, DP>, FwdShared<DP>::kBytes, who);
  if (!rc) rc = make_map(&q, DT, P.q, P.qs, P.dim, P.queries, P.heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&k, DT, P.k, P.ks, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&v, DT, P.v, P.vs, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (rc) return rc;
  const unsigned grid = (unsigned)((P.queries + kTcRows - 1) / kTcRows) * P.heads * P.batch;
  attention_tc_forward<DT, DP><<<grid, kTcThreads, FwdShared<DP>::kBytes, s>>>(P, q, k, v);
  return launch_status("nt_attention_forward launch");
}

template <int DT, int DP>
static int launch_tc_backward(const AttnParams& P, cudaStream_t s) {
  const char* who = "nt_attention_backward";
  CUtensorMap q, g, k, v;
  const int bytes = BwdShared<DP>::kBytes;
  int rc = large_smem(attention_tc_backward<DT, DP, false>, bytes, who);
  if (!rc) rc = large_smem(attention_tc_backward<DT, DP, true>, bytes, who);
  if (!rc) rc = make_map(&q, DT, P.q, P.qs, P.dim, P.queries, P.heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&g, DT, P.g, P.gs, P.dim, P.queries, P.heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&k, DT, P.k, P.ks, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (!rc) rc = make_map(&v, DT, P.v, P.vs, P.dim, P.keys, P.kv_heads, P.batch, kTcRows, who);
  if (rc) return rc;
  const unsigned rows = (unsigned)((P.queries + kTcRows - 1) / kTcRows) * P.heads * P.batch;
  attention_tc_backward<DT, DP, false><<<rows, kBwdThreads, bytes, s>>>(P, q, g, k, v);
  rc = launch_status("nt_attention_backward launch");
  if (rc) return rc;
  const int tiles = (P.keys + kTcKeyRows - 1) / kTcKeyRows + P.sink_tiles * (P.parts - 1);
  attention_tc_backward<DT, DP, true><<<(unsigned)tiles * P.kv_heads * P.batch, kBwdThreads, bytes, s>>>(P, k, v, q, g);
  return launch_status("nt_attention_backward launch");
}

int attention_tc_forward_launch(const AttnParams& P, int dtype, cudaStream_t s) {
  if (dtype == NT_BF16) return P.dim <= 64 ? launch_tc_forward<NT_BF16, 64>(P, s) : launch_tc_forward<NT_BF16, 128>(P, s);
  return P.dim <= 64 ? launch_tc_forward<NT_F16, 64>(P, s) : launch_tc_forward<NT_F16, 128>(P, s);
}

int attention_tc_backward_launch(const AttnParams& P, int dtype, cudaStream_t s) {
  if (dtype == NT_BF16) return P.dim <= 64 ? launch_tc_backward<NT_BF16, 64>(P, s) : launch_tc_backward<NT_BF16, 128>(P, s);
  return P.dim <= 64 ? launch_tc_backward<NT_F16, 64>(P, s) : launch_tc_backward<NT_F16, 128>(P, s);
}

}  // namespace nt
