// Sliding-window attention of one new token per sequence over a cache of keys and values.
//
// Bound: HBM, one read of the visible keys and values (2 head_dim elements a key and key head
// against 4 head_dim products per query head) for every 8 query heads of a key head, on the FP32 pipe
// for every 4, 2 or 1 (what divides their number). The visible keys are the sinks [0, sink_end) and the
// window [lo, length); number n of them is row n or n + skip. Blocks of a cluster share one
// (sequence, key head, up to 8 query heads): each block takes a contiguous piece of the visible
// keys, each warp pieces of that, with a running maximum, sum and output of its own; they are
// joined over the block in shared memory and over the cluster in distributed shared memory, always
// in the same order.
#include <cmath>

#include "nt_attention.cuh"
#include "nt_tc.cuh"

namespace nt {

// The block's piece [from, to) of the visible keys of its sequence.
struct StepKeys {
  int sink_end, skip, from, to;
  __device__ __forceinline__ StepKeys(const AttnParams& P, int length, int rank, int splits) {
    const int lo = P.window == 0 ? 0 : max(0, length - P.window);
    sink_end = min(P.sinks, lo);
    const int visible = sink_end + length - lo;
    const int chunk = (visible + splits - 1) / splits;
    from = min(visible, rank * chunk);
    to = min(visible, from + chunk);
    skip = lo - sink_end;
  }
  __device__ __forceinline__ int64_t row(int n) const { return n < sink_end ? n : (int64_t)n + skip; }
};

// Joins the partial results of the block's warps (maximum and sum in ml[warp][head][2], output in
// acc[warp][head][DP], unnormalised) and of the `splits` blocks from block `base` of the cluster on,
// of which this one is number `rank`, and stores the output. `acc` is in shared memory at the same
// place in every block.
template <int DT, int DP, int WARPS, int HEADS>
__device__ __forceinline__ void join_step(const AttnParams& P, float* acc, const float* ml, int heads, int b, int h0, int splits,
                                          int rank, int base = 0) {
  constexpr int THREADS = WARPS * 32, STRIDE = HEADS * DP;
  __syncthreads();
  for (int i = threadIdx.x; i < heads * DP; i += THREADS) {
    const int g = i / DP, c = i % DP;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[(w * HEADS + g) * 2]);
    float sum = 0.0f, a = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = top == -INFINITY ? 0.0f : exp2f((ml[(w * HEADS + g) * 2] - top) * P.scale_log2);
      sum = fmaf(ml[(w * HEADS + g) * 2 + 1], f, sum);
      a = fmaf(acc[w * STRIDE + i], f, a);
    }
    if (splits == 1) {
      if (c < P.dim) store1<DT>(P.o, P.os.at(b, h0 + g, 0) + c, sum == 0.0f ? 0.0f : a / sum);
    } else {
      acc[i] = a;                             // only this thread reads column i of the partial outputs
      acc[STRIDE + i] = c == 0 ? top : sum;   // statistics of the block: columns 0 and 1
    }
  }
  if (gridDim.x == 1) return;
  __syncthreads();
  cluster_sync_all();
  for (int i = (rank * THREADS + threadIdx.x) * 4; splits > 1 && i < heads * DP; i += splits * THREADS * 4) {
    const int g = i / DP, c = i % DP;
    const JoinedRow row = join_row(acc + i, acc + STRIDE + g * DP, splits, P.scale_log2, base);
    const float x[4] = {row.o.x, row.o.y, row.o.z, row.o.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < P.dim) store1<DT>(P.o, P.os.at(b, h0 + g, 0) + c + e, row.sum == 0.0f ? 0.0f : x[e] / row.sum);
  }
  cluster_sync_all();   // a block's shared memory stays until every block has read it
}

// ---- 16-bit rows of whole 16-byte vectors ------------------------------------------------
// A warp owns a ring of 16-key stages that tiled copies fill, 2 KB each (copies of single rows, 256
// bytes, came at one per 30 cycles and SM, a third of the bandwidth); the 128-byte swizzle spreads
// the eight rows that an ldmatrix reads over the banks. The products are the small matrix
// instructions, with the keys as their 16 rows and the query heads as their 8 columns: S^T = K q^T,
// O^T += V^T P^T. (A tcgen05 product has 128 rows; a group of query heads has one to eight.) P^T is
// the accumulator of the first as the second operand of the other, transposed between the lanes in
// registers. The weights are rounded to the type of the values for the second product. (197 MB of 32
// sequences of 16 heads of 128 on 4, window 4096: 40 us, 75 % of the measured copy rate; 8 full caches
// of 32768, as pairs in clusters of 16: 88 us, 92 %.)
constexpr int kRingWarps = 4;
constexpr int kRingKeys = 16;

template <int DP> struct StepShared {
  static constexpr int kTile = kRingKeys * DP * 2;      // keys or values
  // (More in flight is slower: the DRAM sees as many streams as there are warps. 8 sequences up to 32768
  // keys took 64.5 us with 2 stages, 67 with 3, 109 with 6; all apart, before two shared a cluster.)
  static constexpr int kStages = DP == 128 ? 2 : 4;
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kBytes = kRingWarps * kRing + 1024;
  static_assert(kRingWarps * 8 * DP * 4 <= kBytes - 1024, "the partial outputs take the rings' place");
};

// The sequence of number z, and with BOTH the one of number batch - 1 - z, the longest first: the last
// blocks to start are short and the blocks that share an SM differ (the lengths are known on the device
// alone). Every block ranks them for itself, in `scratch`; more than kRankedBatch of them stay in
// their order.
constexpr int kRankedBatch = 256;
template <bool BOTH>
__device__ __forceinline__ int ranked_sequence(const AttnParams& P, int z, int* scratch, int* found) {
  if (!BOTH && (P.batch == 1 || P.batch > kRankedBatch)) return z;   // (a pair is one of a few sequences)
  for (int i = threadIdx.x; i < P.batch; i += blockDim.x) {
    const int n = attn_length(P, i);
    scratch[i] = P.window == 0 ? n : min(n, P.window + P.sinks);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < P.batch; i += blockDim.x) {
    const int n = scratch[i];
    int rank = 0;
    for (int j = 0; j < P.batch; ++j) rank += scratch[j] > n || (scratch[j] == n && j < i);
    if (rank == z) found[0] = i;
    if (BOTH && rank == P.batch - 1 - z) found[1] = i;
  }
  __syncthreads();
  return found[0];
}

// The pieces of 16 visible keys of a sequence: those of the sinks, then those of the window; the block's
// share of them is [from, to).
struct StepPieces {
  int sink_end, lo, length, sinks, from, to;
  __device__ __forceinline__ StepPieces(const AttnParams& P, int n, int rank, int splits) : length(n) {
    lo = P.window == 0 ? 0 : max(0, n - P.window);
    sink_end = min(P.sinks, lo);
    sinks = (sink_end + kRingKeys - 1) / kRingKeys;
    const int pieces = sinks + (n - lo + kRingKeys - 1) / kRingKeys;
    const int chunk = (pieces + splits - 1) / splits;
    from = min(pieces, rank * chunk);
    to = min(pieces, from + chunk);
  }
  __device__ __forceinline__ void piece(int i, int& row, int& rows) const {
    row = i < sinks ? i * kRingKeys : lo + (i - sinks) * kRingKeys;
    rows = min(kRingKeys, (i < sinks ? sink_end : length) - row);
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_transposed(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int DT>
__device__ __forceinline__ void mma16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == NT_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// PAIRED: a cluster serves two sequences, the longest with the shortest and so on, and deals its
// blocks to them by their lengths.
template <int DT, int DP, bool PAIRED>
__global__ void __launch_bounds__(kRingWarps * 32)
attention_step_ring_kernel(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v) {
  using Shape = StepShared<DP>;
  constexpr int STAGES = Shape::kStages, TILE = Shape::kTile;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kRingWarps][STAGES];
  __shared__ float ml[kRingWarps][8][2];
  __shared__ int sequences[2];
  // The same place in every block of the cluster.
  uint8_t* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int passes = (P.group + 7) / 8;
  const int hk = blockIdx.y / passes, first = blockIdx.y % passes * 8;
  const int h0 = hk * P.group + first, heads = min(8, P.group - first);
  int b = ranked_sequence<PAIRED>(P, blockIdx.z, reinterpret_cast<int*>(ring), sequences), splits = gridDim.x, rank = blockIdx.x, base = 0;
  if (PAIRED && sequences[1] != b) {
    auto visible = [&](int b) {
      const int n = attn_length(P, b);
      return P.window == 0 ? n : min(n, P.window + P.sinks);
    };
    const int64_t one = visible(b), both = max((int64_t)1, one + visible(sequences[1]));
    const int share = min(splits - 1, max(1, (int)((2 * one * splits + both) / (2 * both))));
    if (rank >= share) {
      b = sequences[1];
      base = share;
      rank -= share;
      splits -= share;
    } else {
      splits = share;
    }
  }
  const StepPieces pieces(P, attn_length(P, b), rank, splits);
  uint8_t* mine = ring + warp * Shape::kRing;

  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
    fence_proxy_async();   // the ranking used the ring's place
  }
  __syncwarp();

  const int blocks = pieces.to - pieces.from;
  const int count = blocks > warp ? (blocks - warp + kRingWarps - 1) / kRingWarps : 0;   // of this warp
  auto fill = [&](int i) {
    if (lane == 0) {
      int row, rows;
      pieces.piece(pieces.from + warp + i * kRingWarps, row, rows);
      uint64_t* bar = &full[warp][i % STAGES];
      uint8_t* dst = mine + i % STAGES * 2 * TILE;
      mbar_arrive_expect_tx(bar, 2 * TILE);
#pragma unroll
      for (int half = 0; half < DP / 64; ++half) {
        tma_load(dst + half * kRingKeys * 128, &map_k, half * 64, row, hk, b, bar);
        tma_load(dst + TILE + half * kRingKeys * 128, &map_v, half * 64, row, hk, b, bar);
      }
    }
  };
  for (int i = 0; i < min(count, STAGES); ++i) fill(i);

  const int steps = (P.dim + 15) / 16;
  uint32_t q[DP / 16][2];
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = k * 16 + e * 8 + 2 * t;
      uint32_t v = 0;
      if (g < heads) {
        const uint16_t* src = static_cast<const uint16_t*>(P.q) + P.qs.at(b, h0 + g, 0);
        v = (c < P.dim ? src[c] : 0u) | (uint32_t)(c + 1 < P.dim ? src[c + 1] : 0u) << 16;
      }
      q[k][e] = v;
    }
  float acc[DP / 16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[k][e] = 0.0f;

  bool ok = true;
  int i = 0;
  for (; i < count; ++i) {
    ok = __all_sync(0xffffffffu, wait_bar(&full[warp][i % STAGES], (i / STAGES) & 1));
    if (!ok) break;
    uint8_t* stage = mine + i % STAGES * 2 * TILE;
    int row, rows;
    pieces.piece(pieces.from + warp + i * kRingWarps, row, rows);
    if (rows < kRingKeys) {
      // What lies past the last visible key may be anything; its weight is 0, but 0 * NaN must not
      // reach the sum.
      for (int n = lane; n < (kRingKeys - rows) * (DP / 8); n += 32)
        *reinterpret_cast<uint4*>(stage + TILE + n % (DP / 64) * kRingKeys * 128 + (rows + n / (DP / 8)) * 128 +
                                  n / (DP / 64) % 8 * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();   // the next copy into this stage comes after it
      __syncwarp();
    }
    // Lane's row of the four 8 x 8 matrices of a 16 x 16 tile, and the 16-byte vector of its columns,
    // where the swizzle put it.
    const uint32_t at_k = smem_u32(stage) + (lane & 15) * 128;
    const uint32_t at_v = smem_u32(stage) + TILE + ((lane >> 4) * 8 + (lane & 7)) * 128;
    const int vec_k = lane >> 4, vec_v = lane >> 3 & 1, swap = lane & 7;
    auto column = [&](int k, int vec) {
      return (uint32_t)((k >> 2) * kRingKeys * 128 + ((((k & 3) * 2 + vec) ^ swap) << 4));
    };
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      if (k < steps) {
        uint32_t a[4];
        ldmatrix4(at_k + column(k, vec_k), a);
        mma16x8x16<DT>(s, a, q[k][0], q[k][1]);
      }
    // s: keys g and g + 8, heads 2 t and 2 t + 1.
    if (g >= rows) s[0] = s[1] = -INFINITY;
    if (g + 8 >= rows) s[2] = s[3] = -INFINITY;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = fmaxf(s[e], s[e + 2]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(top, m[e]);
      const float shift = top == -INFINITY ? 0.0f : top;
      const float old = ex2_approx((m[e] - shift) * P.scale_log2);
      m[e] = top;
      s[e] = ex2_approx((s[e] - shift) * P.scale_log2);
      s[e + 2] = ex2_approx((s[e + 2] - shift) * P.scale_log2);
      l[e] = fmaf(l[e], old, s[e] + s[e + 2]);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        acc[k][e] *= old;
        acc[k][e + 2] *= old;
      }
    }
    const uint32_t p0 = transpose8x8(pack2<DT>(s[0], s[1])), p1 = transpose8x8(pack2<DT>(s[2], s[3]));
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      if (k < steps) {
        uint32_t a[4];
        ldmatrix4_transposed(at_v + column(k, vec_v), a);
        mma16x8x16<DT>(acc[k], a, p0, p1);
      }
    __syncwarp();
    if (i + STAGES < count) fill(i + STAGES);
  }
  if (!ok) {   // the copies in flight land before the block may end
    for (int n = i; n < min(count, i + STAGES); ++n) wait_bar(&full[warp][n % STAGES], (n / STAGES) & 1);
    if (lane == 0 && P.error != nullptr) atomicOr(P.error, 1);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], o);
  __syncthreads();   // every warp is done with its ring
  float* part = reinterpret_cast<float*>(ring) + warp * 8 * DP;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[(2 * t + (e & 1)) * DP + k * 16 + g + (e >> 1) * 8] = acc[k][e];
  if (g == 0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      ml[warp][2 * t + e][0] = m[e];
      ml[warp][2 * t + e][1] = l[e];
    }
  }
  join_step<DT, DP, kRingWarps, 8>(P, reinterpret_cast<float*>(ring), &ml[0][0][0], heads, b, h0, splits, rank, base);
}

// ---- float32, and 16-bit rows of any layout ------------------------------------------------
// Lanes of 16 bytes share a row (LPR of them); every lane group keeps its own running maximum, sum
// and output for HG query heads, joined over the warp by shuffles. (394 MB of float32, 32
// sequences of 16 heads of 128 on 4, window 4096: 136 us, 44 % of the measured copy rate, 190 with a sum
// over the lanes for each row and head; what costs is the instructions of a row beside its loads.)
constexpr int kStepThreads = 256;
constexpr int kStepWarps = kStepThreads / 32;
constexpr int kStepRows = 4;   // rows in flight per lane group

// Sums of N values (the rows and heads at hand) over a group of 2 O lanes: each step adds half of the
// values that are left to the lanes on one side and the rest to the other, N - 1 shuffles in place of
// log2(2 O) a value. Lane by lane the values then lie in their order, N / (2 O) to a lane or one to
// every 2 O / N lanes.
template <int O, int N, int ALL>
__device__ __forceinline__ void group_scatter(float (&v)[ALL], int lane) {
  if constexpr (O >= 1) {
    if constexpr (N > 1) {
      const bool up = lane & O;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float give = up ? v[i] : v[i + N / 2], keep = up ? v[i + N / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, O);
      }
      group_scatter<O / 2, N / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
      group_scatter<O / 2, 1>(v, lane);
    }
  }
}
template <int LPR, int N>
__device__ __forceinline__ float group_value(const float (&v)[N], int lane, int i) {
  constexpr int EACH = N > LPR ? N / LPR : 1, APART = LPR > N ? LPR / N : 1;
  return __shfl_sync(0xffffffffu, v[i % EACH], (lane & ~(LPR - 1)) + i / EACH * APART);
}

template <int DT, int LPR, int HG>
__global__ void __launch_bounds__(kStepThreads) attention_step_kernel(const __grid_constant__ AttnParams P) {
  using T = typename Elem<DT>::T;
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int DP = LPR * EPV;
  constexpr int RPL = 32 / LPR;
  __shared__ float part_ml[kStepWarps][HG][2];
  __shared__ __align__(16) float part_acc[kStepWarps][HG][DP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / LPR, col = lane % LPR * EPV;
  const int splits = gridDim.x, rank = blockIdx.x;
  const int passes = P.group / HG;
  const int hk = blockIdx.y / passes, h0 = hk * P.group + blockIdx.y % passes * HG;
  const int b = blockIdx.z;
  const StepKeys keys(P, attn_length(P, b), rank, splits);
  const int from = keys.from, to = keys.to;

  float q[HG][EPV], acc[HG][EPV], m[HG], l[HG];
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      acc[g][e] = 0.0f;
      q[g][e] = col + e < P.dim ? load1<DT>(P.q, P.qs.at(b, h0 + g, 0) + col + e) : 0.0f;
    }
  }
  const T* kb = static_cast<const T*>(P.k) + P.ks.at(b, hk, 0) + col;
  const T* vb = static_cast<const T*>(P.v) + P.vs.at(b, hk, 0) + col;
  auto load = [&](const T* base, int64_t stride, int n, uint4& raw) {
    raw = make_uint4(0, 0, 0, 0);
    if (n < to && col < P.dim) {
      const T* src = base + keys.row(n) * stride;
      if (P.vec) {
        raw = __ldcs(reinterpret_cast<const uint4*>(src));
      } else {
        T* out = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int e = 0; e < EPV; ++e)
          if (col + e < P.dim) out[e] = src[e];
      }
    }
  };
  constexpr int STRIDE = kStepWarps * RPL;
  for (int n0 = from + warp * RPL + sub; n0 - sub < to; n0 += STRIDE * kStepRows) {
    uint4 kr[kStepRows], vr[kStepRows];
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) load(kb, P.ks.t, n0 + r * STRIDE, kr[r]);
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) load(vb, P.vs.t, n0 + r * STRIDE, vr[r]);
    float part[kStepRows * HG], s[kStepRows][HG];
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      float kf[EPV];
      unpack16<DT>(kr[r], kf);
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < EPV; ++e) d = fmaf(q[g][e], kf[e], d);
        part[r * HG + g] = d;
      }
    }
    group_scatter<LPR / 2, kStepRows * HG>(part, lane);
#pragma unroll
    for (int r = 0; r < kStepRows; ++r)
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        const float d = group_value<LPR, kStepRows * HG>(part, lane, r * HG + g);
        s[r][g] = n0 + r * STRIDE < to ? d : -INFINITY;
      }
#pragma unroll
    for (int g = 0; g < HG; ++g) {
      float top = m[g];
#pragma unroll
      for (int r = 0; r < kStepRows; ++r) top = fmaxf(top, s[r][g]);
      const float shift = top == -INFINITY ? 0.0f : top;
      const float old = exp2f((m[g] - shift) * P.scale_log2);
      m[g] = top;
      l[g] *= old;
#pragma unroll
      for (int e = 0; e < EPV; ++e) acc[g][e] *= old;
#pragma unroll
      for (int r = 0; r < kStepRows; ++r) {
        s[r][g] = exp2f((s[r][g] - shift) * P.scale_log2);
        l[g] += s[r][g];
      }
    }
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      float vf[EPV];
      unpack16<DT>(vr[r], vf);
#pragma unroll
      for (int g = 0; g < HG; ++g)
#pragma unroll
        for (int e = 0; e < EPV; ++e) acc[g][e] = fmaf(s[r][g], vf[e], acc[g][e]);
    }
  }
  // Join the lane groups of a warp, then the warps.
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    float top = m[g];
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = top == -INFINITY ? 0.0f : exp2f((m[g] - top) * P.scale_log2);
    l[g] *= f;
#pragma unroll
    for (int e = 0; e < EPV; ++e) acc[g][e] *= f;
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
#pragma unroll
      for (int e = 0; e < EPV; ++e) acc[g][e] += __shfl_xor_sync(0xffffffffu, acc[g][e], o);
    }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < EPV; ++e) part_acc[warp][g][col + e] = acc[g][e];
      if (lane == 0) {
        part_ml[warp][g][0] = top;
        part_ml[warp][g][1] = l[g];
      }
    }
  }
  join_step<DT, DP, kStepWarps, HG>(P, &part_acc[0][0][0], &part_ml[0][0][0], HG, b, h0, splits, rank);
}

// Blocks of one cluster share the visible keys: as many as the device runs at once (`most_blocks`:
// a second wave of short pieces costs more than the idle SMs of one; 32 sequences with 4 key heads
// and a 4096-key window take 39 us in clusters of 2 and 47 in clusters of 4), with at least `least`
// keys to a block. Clusters of 16 are past what every device promises; where this one runs none of
// that size the launch falls back to 8.
constexpr int kStepMaxSplits = 16;
static int step_splits(const AttnParams& P, int64_t units, int most_blocks, int least) {
  const int64_t most = P.window == 0 ? P.keys : (int64_t)P.window + P.sinks < P.keys ? (int64_t)P.window + P.sinks : P.keys;
  int splits = 1;
  while (splits < kStepMaxSplits && units * splits * 2 <= most_blocks && most > (int64_t)least * splits) splits *= 2;
  return splits;
}

template <typename K, typename... Maps>
static int launch_step(K kernel, const AttnParams& P, int splits, int heads, int sequences, int threads, size_t bytes,
                       cudaStream_t s, const Maps&... maps) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(splits, heads, sequences);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = bytes;
  config.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = splits > 1 ? 1 : 0;
  if (splits > kMaxSplits) {
    int clusters = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess || clusters < 1) {
      cudaGetLastError();
      config.gridDim.x = attr.val.clusterDim.x = kMaxSplits;
    }
  }
  cudaError_t e = cudaLaunchKernelEx(&config, kernel, P, maps...);
  if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, "nt_attention_step launch"); }
  return launch_status("nt_attention_step launch");
}

template <int DT, int DP, bool PAIRED>
static int launch_ring(const AttnParams& P, int splits, int heads, cudaStream_t s) {
  const char* who = "nt_attention_step";
  CUtensorMap k, v;
  int rc = large_smem<attention_step_ring_kernel<DT, DP, PAIRED>>(StepShared<DP>::kBytes, who);
  if (!rc) rc = make_map(&k, DT, P.k, P.ks, P.dim, P.keys, P.kv_heads, P.batch, kRingKeys, who);
  if (!rc) rc = make_map(&v, DT, P.v, P.vs, P.dim, P.keys, P.kv_heads, P.batch, kRingKeys, who);
  if (rc) return rc;
  return launch_step(attention_step_ring_kernel<DT, DP, PAIRED>, P, splits, heads, PAIRED ? (P.batch + 1) / 2 : P.batch,
                     kRingWarps * 32, StepShared<DP>::kBytes, s, k, v);
}

template <int DT, int DP>
static int dispatch_ring(const AttnParams& P, cudaStream_t s) {
  const int heads = P.kv_heads * ((P.group + 7) / 8);
  const int splits = step_splits(P, (int64_t)P.batch * heads, 3 * current_sm_count(), kRingWarps * kRingKeys);
  // Clusters of 8 become clusters of 16 for two sequences, whose lengths differ as a rule: 8 sequences of 16
  // heads on 4, up to 32768 keys, 63 us apart and 56.5 paired (all of 32768: 84, 87); 4 of 32 on 8, up to
  // 16384, 37 and 35. Smaller ones gain nothing: 32 sequences in clusters of 4 for two take 44, in
  // clusters of 2 39.
  return P.batch > 1 && splits == kStepMaxSplits / 2 ? launch_ring<DT, DP, true>(P, kStepMaxSplits, heads, s)
                                                     : launch_ring<DT, DP, false>(P, splits, heads, s);
}

template <int DT, int LPR, int HG>
static int launch_simt(const AttnParams& P, cudaStream_t s) {
  const int heads = P.kv_heads * (P.group / HG);
  const int splits = step_splits(P, (int64_t)P.batch * heads, 2 * current_sm_count(), 64);
  return launch_step(attention_step_kernel<DT, LPR, HG>, P, splits, heads, P.batch, kStepThreads, 0, s);
}

template <int DT, int LPR>
static int dispatch_heads(const AttnParams& P, cudaStream_t s) {
  if (P.group % 4 == 0) return launch_simt<DT, LPR, 4>(P, s);
  if (P.group % 2 == 0) return launch_simt<DT, LPR, 2>(P, s);
  return launch_simt<DT, LPR, 1>(P, s);
}

template <int DT>
static int dispatch_step(const AttnParams& P, cudaStream_t s) {
  if constexpr (DT != NT_F32) {
    if (P.vec && P.keys > 0) return P.dim <= 64 ? dispatch_ring<DT, 64>(P, s) : dispatch_ring<DT, 128>(P, s);
  }
  constexpr int EPV = DT == NT_F32 ? 4 : 8;
  return P.dim <= 64 ? dispatch_heads<DT, 64 / EPV>(P, s) : dispatch_heads<DT, 128 / EPV>(P, s);
}

int attention_step_launch(const AttnParams& P, int dtype, cudaStream_t s) {
  switch (dtype) {
    case NT_F32: return dispatch_step<NT_F32>(P, s);
    case NT_F16: return dispatch_step<NT_F16>(P, s);
    default: return dispatch_step<NT_BF16>(P, s);
  }
}

}  // namespace nt
