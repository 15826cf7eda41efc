// Sliding-window attention with sinks: the C entry points and the kernels for float32 (and for
// 16-bit rows that are no whole 16-byte vectors).
//
//   S = scale q k^T over the visible keys,  m = max S,  l = sum exp(S - m),
//   o = sum exp(S - m) v / l,  lse = m + ln l
//   P = exp(S - lse),  dv = P^T g,  dP = g v^T,  delta = sum(g o),  dS = P (dP - delta),
//   dq = scale dS k,  dk = scale dS^T q, dk and dv summed over the query heads of a group
//
// Nothing of size queries x keys is stored: the forward keeps the running maximum and sum, the
// backward computes S again from lse. All sums are float32. The gradients of queries and of
// keys are two passes over the pairs (each computes S and dP), so that every sum has one owner
// and a fixed order: no atomics.
#include <cmath>
#include <climits>

#include "nt_attention.cuh"
#include "nt_tc.cuh"

namespace nt {

// ---- float32 kernels: 64 x 64 blocks on the FP32 pipe ---------------------------------
// 256 threads as 16 x 16; a thread holds rows 4 ty .. 4 ty + 3 and columns tx + 16 j. Rows in
// shared memory are DP + 4 floats apart, so the eight threads of a 16-byte wavefront that read
// eight consecutive rows touch different banks. A product step reads 8 vectors of 16 bytes for
// 64 fused multiply-adds, which keeps the FP32 pipe and not shared memory the limit.
constexpr int kRows = 64;
constexpr int kSimtThreads = 256;
constexpr int kWeightStride = kRows + 4;

// rows [first, first + 64) of one head into shared memory as float32; zero past `end` and past
// the head's width.
template <int DT, int DP>
__device__ __forceinline__ void load_tile(float* dst, const void* base, int64_t row_stride, int64_t first, int64_t end,
                                          int dim, int vec) {
  using T = typename Elem<DT>::T;
  constexpr int EPV = 16 / (int)sizeof(T);
  const T* src = static_cast<const T*>(base);
  if (vec) {
#pragma unroll 4
    for (int i = threadIdx.x; i < kRows * (DP / EPV); i += kSimtThreads) {
      const int r = i / (DP / EPV), c = i % (DP / EPV) * EPV;
      float v[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) v[e] = 0.0f;
      if (first + r < end && c < dim)
        unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(src + (first + r) * row_stride + c)), v);
#pragma unroll
      for (int e = 0; e < EPV; e += 4)
        *reinterpret_cast<float4*>(dst + r * (DP + 4) + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
  } else {
    for (int i = threadIdx.x; i < kRows * DP; i += kSimtThreads) {
      const int r = i / DP, c = i % DP;
      dst[r * (DP + 4) + c] = first + r < end && c < dim ? Elem<DT>::to_f32(src[(first + r) * row_stride + c]) : 0.0f;
    }
  }
}

// s[i][j] = sum over the width of a[4 ty + i] . b[tx + 16 j], even and odd columns apart: two
// multiply-adds to an instruction, which leaves the loads more of the issue slots (here and in
// tile_accumulate: 4 x 1024 causal tokens of 4 heads of 128, backward 481 -> 459 us).
template <int DP>
__device__ __forceinline__ void tile_product(const float* a, const float* b, int tx, int ty, float (&s)[4][4]) {
  Pair sum[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = Pair(0.0f, 0.0f);
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * (DP + 4) + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * (DP + 4) + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sum[i][j] = fma2(Pair(x[i].z, x[i].w), Pair(y[j].z, y[j].w), fma2(Pair(x[i].x, x[i].y), Pair(y[j].x, y[j].y), sum[i][j]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float even, odd;
      sum[i][j].get(even, odd);
      s[i][j] = even + odd;
    }
}

// acc[i][u] += sum over the 64 columns c of w[4 ty + i][c] * b[c][4 tx + 64 u ..]
template <int DP>
__device__ __forceinline__ void tile_accumulate(const float* w, const float* b, int tx, int ty, float4 (&acc)[4][DP / 64]) {
#pragma unroll 2
  for (int c = 0; c < kRows; c += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(w + (4 * ty + i) * kWeightStride + c);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int u = 0; u < DP / 64; ++u) {
        const float4 y = *reinterpret_cast<const float4*>(b + (c + k) * (DP + 4) + 4 * tx + 64 * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = k == 0 ? x[i].x : k == 1 ? x[i].y : k == 2 ? x[i].z : x[i].w;
          fma2(Pair(f, f), Pair(y.x, y.y), Pair(acc[i][u].x, acc[i][u].y)).get(acc[i][u].x, acc[i][u].y);
          fma2(Pair(f, f), Pair(y.z, y.w), Pair(acc[i][u].z, acc[i][u].w)).get(acc[i][u].z, acc[i][u].w);
        }
      }
  }
}

template <int DT, int DP>
__device__ __forceinline__ void store_row4(void* base, int64_t at, int tx, int dim, const float4 (&acc)[DP / 64], float f) {
#pragma unroll
  for (int u = 0; u < DP / 64; ++u) {
    const float v[4] = {acc[u].x, acc[u].y, acc[u].z, acc[u].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 4 * tx + 64 * u + e;
      if (c < dim) store1<DT>(base, at + c, v[e] * f);
    }
  }
}

__device__ __forceinline__ float lanes16_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float lanes16_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The maximum is kept of the scores before the scale: a difference of scores is formed before it
// is scaled, so that scores near the ends of float32 do not overflow on the way. 4 x 1024 causal tokens of
// 4 heads of 128: 200 us, 23 TFLOP/s of the tiles' products, with shared memory busy for 42 % of the
// cycles, instructions issued in 26 % and 18 % of the warps there: a block waits for its operands from
// shared memory, then at its barriers for one tile after another, and 256 blocks on 148 SMs do not
// cover that. 4 x 256 tokens of 4 heads of 64 are 64 blocks and 23 us of their latency.
template <int DT, int DP>
__global__ void __launch_bounds__(kSimtThreads) attention_forward_kernel(const __grid_constant__ AttnParams P) {
  extern __shared__ __align__(16) float smem[];
  float* q = smem;
  float* kv = q + kRows * (DP + 4);
  float* w = kv + kRows * (DP + 4);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  // Blocks in the order of their work: the last queries of every head first.
  const uint32_t pairs = (uint32_t)P.heads * P.batch, tiles = gridDim.x / pairs;
  const int b = blockIdx.x % pairs / P.heads, h = blockIdx.x % P.heads, hk = h / P.group;
  const int i0 = (tiles - 1 - blockIdx.x / pairs) * kRows, i1 = min(P.queries, i0 + kRows);
  const int length = attn_length(P, b);
  const AttnKeys range(P, length, i0, i1);
  const int es = sizeof(typename Elem<DT>::T);
  load_tile<DT, DP>(q, static_cast<const char*>(P.q) + P.qs.at(b, h, 0) * es, P.qs.t, i0, i1, P.dim, P.vec);
  float m[4], l[4];
  float4 acc[4][DP / 64];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < DP / 64; ++u) acc[i][u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  const int blocks = range.blocks(kRows);
  for (int t = 0; t < blocks; ++t) {
    int begin, end;
    range.block(t, kRows, begin, end);
    __syncthreads();
    load_tile<DT, DP>(kv, static_cast<const char*>(P.k) + P.ks.at(b, hk, 0) * es, P.ks.t, begin, end, P.dim, P.vec);
    __syncthreads();
    float s[4][4];
    tile_product<DP>(q, kv, tx, ty, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = P.offset + i0 + 4 * ty + i;
      float top = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = begin + tx + 16 * j;
        s[i][j] = key < end && attn_visible(P, length, p, key) ? s[i][j] : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      top = lanes16_max(top);
      const float shift = top == -INFINITY ? 0.0f : top;
      const float old = exp2f((m[i] - shift) * P.scale_log2);
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f((s[i][j] - shift) * P.scale_log2);
        sum += e;
        w[(4 * ty + i) * kWeightStride + tx + 16 * j] = e;
      }
      l[i] = l[i] * old + lanes16_sum(sum);
#pragma unroll
      for (int u = 0; u < DP / 64; ++u) {
        acc[i][u].x *= old; acc[i][u].y *= old; acc[i][u].z *= old; acc[i][u].w *= old;
      }
    }
    __syncthreads();
    load_tile<DT, DP>(kv, static_cast<const char*>(P.v) + P.vs.at(b, hk, 0) * es, P.vs.t, begin, end, P.dim, P.vec);
    __syncthreads();
    tile_accumulate<DP>(w, kv, tx, ty, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i0 + 4 * ty + i;
    if (row >= i1) continue;
    const float f = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
    store_row4<DT, DP>(P.o, P.os.at(b, h, row), tx, P.dim, acc[i], f);
    if (DT != NT_F32 && P.o_low != nullptr) {
#pragma unroll
      for (int u = 0; u < DP / 64; ++u) {
        float* a = &acc[i][u].x;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = a[e] * f - Elem<DT>::to_f32(Elem<DT>::from_f32(a[e] * f));
      }
      store_row4<DT, DP>(P.o_low, P.os.at(b, h, row), tx, P.dim, acc[i], 1.0f);
    }
    if (P.lse != nullptr && tx == 0)
      P.lse[((int64_t)b * P.heads + h) * P.queries + row] = l[i] == 0.0f ? -INFINITY : fmaf(m[i], P.scale, log2f(l[i]) * kLn2F);
  }
}

// delta = sum over the width of g o of every query, 16 lanes to a row (2 us of latency at 4 x 256 tokens
// of 4 heads of 64, 4 at 4 x 1024 of 128).
template <int DT>
__global__ void __launch_bounds__(256) attention_rows_delta_kernel(const __grid_constant__ AttnParams P) {
  grid_dependents_go();
  const int b = blockIdx.z, h = blockIdx.y;
  const int64_t row = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  float d = 0.0f;
  if (row < P.queries) {
    const int64_t g = P.gs.at(b, h, row), o = P.os.at(b, h, row);
    for (int c = threadIdx.x % 16; c < P.dim; c += 16) {
      float x = load1<DT>(P.o, o + c);
      if (DT != NT_F32 && P.o_low != nullptr) x += load1<DT>(P.o_low, o + c);
      d = fmaf(load1<DT>(P.g, g + c), x, d);
    }
  }
  d = lanes16_sum(d);
  if (threadIdx.x % 16 == 0 && row < P.queries) P.delta[((int64_t)b * P.heads + h) * P.queries + row] = d;
}

// A block of the backward. DKV = false: it owns 64 queries and walks the keys (x1 = q, x2 = g; y1 = k,
// y2 = v), giving dq. DKV = true: it owns 64 keys and walks the queries of its group's heads (x1 = k,
// x2 = v; y1 = q, y2 = g), giving dk and dv. In both, s = x1 y1^T and dp = x2 y2^T, out1 = dS y1, and
// with DKV out2 = P y2.
template <int DT, int DP, bool DKV>
__device__ __forceinline__ void backward_block(const AttnParams& P, uint32_t block) {
  extern __shared__ __align__(16) float smem[];
  constexpr int TILE = kRows * (DP + 4);
  float *x1 = smem, *x2 = x1 + TILE, *y1 = x2 + TILE, *y2 = y1 + TILE;
  float *wds = y2 + TILE, *wp = wds + kRows * kWeightStride;
  __shared__ float row_lse[kRows], row_delta[kRows];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int es = sizeof(typename Elem<DT>::T);
  // Blocks in the order of their work: the last queries, or the first keys, of every head first.
  const uint32_t heads = DKV ? P.kv_heads : P.heads, pairs = heads * P.batch;
  const int b = block % pairs / heads, index = block / pairs;
  const int length = attn_length(P, b);
  const char *qb = static_cast<const char*>(P.q), *kb = static_cast<const char*>(P.k), *vb = static_cast<const char*>(P.v),
             *gb = static_cast<const char*>(P.g);
  float4 out1[4][DP / 64], out2[4][DP / 64];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int u = 0; u < DP / 64; ++u) out1[i][u] = out2[i][u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

  if constexpr (!DKV) {
    const int h = block % heads, hk = h / P.group;
    const int i0 = ((P.queries + kRows - 1) / kRows - 1 - index) * kRows, i1 = min(P.queries, i0 + kRows);
    const AttnKeys range(P, length, i0, i1);
    load_tile<DT, DP>(x1, qb + P.qs.at(b, h, 0) * es, P.qs.t, i0, i1, P.dim, P.vec);
    load_tile<DT, DP>(x2, gb + P.gs.at(b, h, 0) * es, P.gs.t, i0, i1, P.dim, P.vec);
    grid_dependency_wait();
    const int64_t stat = ((int64_t)b * P.heads + h) * P.queries;
    float lse[4], delta[4];
    bool one_key[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i0 + 4 * ty + i;
      one_key[i] = attn_key_count(P, length, r) == 1;
      lse[i] = r < i1 ? P.lse[stat + r] * kLog2eF : 0.0f;
      delta[i] = r < i1 ? P.delta[stat + r] : 0.0f;
    }
    const int blocks = range.blocks(kRows);
    for (int t = 0; t < blocks; ++t) {
      int begin, end;
      range.block(t, kRows, begin, end);
      __syncthreads();
      load_tile<DT, DP>(y1, kb + P.ks.at(b, hk, 0) * es, P.ks.t, begin, end, P.dim, P.vec);
      load_tile<DT, DP>(y2, vb + P.vs.at(b, hk, 0) * es, P.vs.t, begin, end, P.dim, P.vec);
      __syncthreads();
      float s[4][4], dp[4][4];
      tile_product<DP>(x1, y1, tx, ty, s);
      tile_product<DP>(x2, y2, tx, ty, dp);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = begin + tx + 16 * j;
          const bool seen = key < end && attn_visible(P, length, P.offset + i0 + 4 * ty + i, key);
          const float pr = exp2f(fmaf(s[i][j], P.scale_log2, -lse[i]));
          wds[(4 * ty + i) * kWeightStride + tx + 16 * j] = seen && !one_key[i] ? pr * (dp[i][j] - delta[i]) : 0.0f;
        }
      __syncthreads();
      tile_accumulate<DP>(wds, y1, tx, ty, out1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + 4 * ty + i < i1) store_row4<DT, DP>(P.dq, P.dqs.at(b, h, i0 + 4 * ty + i), tx, P.dim, out1[i], P.scale);
  } else {
    const int hk = block % heads;
    const AttnPiece piece(P, index);
    const int tile = piece.tile, part = piece.part, parts = piece.parts;
    const int k0 = tile * kRows, k1 = min(P.keys, k0 + kRows);
    const AttnQueries range(P, length, k0, k1);
    load_tile<DT, DP>(x1, kb + P.ks.at(b, hk, 0) * es, P.ks.t, k0, k1, P.dim, P.vec);
    load_tile<DT, DP>(x2, vb + P.vs.at(b, hk, 0) * es, P.vs.t, k0, k1, P.dim, P.vec);
    grid_dependency_wait();
    const int steps = (range.hi - range.lo + kRows - 1) / kRows;
    const int64_t total = (int64_t)steps * P.group;
    const int64_t from = total * part / parts, to = total * (part + 1) / parts;
    for (int64_t t = from; t < to; ++t) {
      const int h = hk * P.group + (int)(t / steps);
      const int begin = range.lo + (int)(t % steps) * kRows, end = min(range.hi, begin + kRows);
      __syncthreads();
      load_tile<DT, DP>(y1, qb + P.qs.at(b, h, 0) * es, P.qs.t, begin, end, P.dim, P.vec);
      load_tile<DT, DP>(y2, gb + P.gs.at(b, h, 0) * es, P.gs.t, begin, end, P.dim, P.vec);
      const int64_t stat = ((int64_t)b * P.heads + h) * P.queries;
      if (threadIdx.x < kRows) {
        const bool in = begin + (int)threadIdx.x < end;
        row_lse[threadIdx.x] = in ? P.lse[stat + begin + threadIdx.x] * kLog2eF : 0.0f;
        row_delta[threadIdx.x] = in ? P.delta[stat + begin + threadIdx.x] : 0.0f;
      }
      __syncthreads();
      float s[4][4], dp[4][4];
      tile_product<DP>(x1, y1, tx, ty, s);
      tile_product<DP>(x2, y2, tx, ty, dp);
      bool one_key[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) one_key[j] = attn_key_count(P, length, begin + tx + 16 * j) == 1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = tx + 16 * j, key = k0 + 4 * ty + i;
          const bool seen = begin + c < end && attn_visible(P, length, P.offset + begin + c, key);
          const float pr = seen ? exp2f(fmaf(s[i][j], P.scale_log2, -row_lse[c])) : 0.0f;
          wp[(4 * ty + i) * kWeightStride + c] = pr;
          wds[(4 * ty + i) * kWeightStride + c] = seen && !one_key[j] ? pr * (dp[i][j] - row_delta[c]) : 0.0f;
        }
      __syncthreads();
      tile_accumulate<DP>(wds, y1, tx, ty, out1);
      tile_accumulate<DP>(wp, y2, tx, ty, out2);
    }
    if (parts == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = k0 + 4 * ty + i;
        if (row >= k1) continue;
        store_row4<DT, DP>(P.dk, P.dks.at(b, hk, row), tx, P.dim, out1[i], P.scale);
        store_row4<DT, DP>(P.dv, P.dvs.at(b, hk, row), tx, P.dim, out2[i], 1.0f);
      }
    } else {
      // [batch, kv head, split block, part, 2, 64, dim]
      const int64_t at = (((int64_t)b * P.kv_heads + hk) * attn_joined(P, (P.keys + kRows - 1) / kRows) + index) * 2 * kRows * P.dim;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t r = 4 * ty + i;
        store_row4<NT_F32, DP>(P.partial, at + r * P.dim, tx, P.dim, out1[i], P.scale);
        store_row4<NT_F32, DP>(P.partial, at + (kRows + r) * P.dim, tx, P.dim, out2[i], 1.0f);
      }
    }
  }
}

// Both kinds of blocks in one launch, so that one fills the SMs that the other leaves idle: `key_blocks`
// own keys, the others queries; the longer kind comes first, the key blocks unless all of them are cut.
// Bound by the operands' reads of shared memory where there are blocks enough (4 x 1024 causal tokens of 4
// heads of 128: 457 us, 35 TFLOP/s of the tiles' products, shared memory busy for 67 % of the cycles,
// the FP32 pipe for about half), else by the copies and products of one block after another.
template <int DT, int DP>
__global__ void __launch_bounds__(kSimtThreads, DP <= 64 ? 2 : 1)
attention_backward_kernel(const __grid_constant__ AttnParams P, uint32_t key_blocks) {
  const bool keys_first = P.rest == 1;
  const uint32_t split = keys_first ? key_blocks : gridDim.x - key_blocks;
  const uint32_t index = blockIdx.x < split ? blockIdx.x : blockIdx.x - split;
  if ((blockIdx.x < split) == keys_first) backward_block<DT, DP, true>(P, index);
  else backward_block<DT, DP, false>(P, index);
}

// dk and dv of the key blocks (of `tile_rows` keys) that were cut: the parts added in order, four
// elements a thread. Grid: runs of 1024 elements of dk or dv of a block, in that order; then blocks,
// then batch x key head. Bound by latency: the parts were just written to the L2 (3.7 MB of 8192 tokens of 4
// key heads: 5 us).
template <int DT>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnParams P, int tile_rows) {
  const int size = tile_rows * P.dim, runs = (size + 1023) / 1024;   // (size is a multiple of 64)
  const int e = (blockIdx.x % runs * 256 + threadIdx.x) * 4, which = blockIdx.x / runs % 2;
  const int tiles = (P.keys + tile_rows - 1) / tile_rows, cut = P.rest > 1 ? tiles : P.sink_tiles;
  const int block = blockIdx.x / runs / 2, tile = block % cut, pair = block / cut;
  const bool sink = tile < P.sink_tiles;
  const int first = sink ? tile * P.parts : P.sink_tiles * P.parts + (tile - P.sink_tiles) * P.rest;
  const int b = pair / P.kv_heads, hk = pair % P.kv_heads;
  if (e >= size || tile * tile_rows + e / P.dim >= P.keys) return;
  const float* src = P.partial + (((int64_t)pair * attn_joined(P, tiles) + first) * 2 + which) * size + e;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = 0; k < (sink ? P.parts : P.rest); ++k) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)k * 2 * size));
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  const float out[4] = {s.x, s.y, s.z, s.w};
  void* dst = which == 0 ? P.dk : P.dv;
  const AttnStrides& st = which == 0 ? P.dks : P.dvs;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = tile * tile_rows + (e + i) / P.dim;
    if (key < P.keys) store1<DT>(dst, st.at(b, hk, key) + (e + i) % P.dim, out[i]);
  }
}

// ---- launches ------------------------------------------------------------------------

template <int DT, int DP>
static int launch_forward(const AttnParams& P, cudaStream_t s) {
  const size_t bytes = (size_t)(2 * kRows * (DP + 4) + kRows * kWeightStride) * 4;
  const int rc = large_smem<attention_forward_kernel<DT, DP>>(bytes, "nt_attention_forward");
  if (rc) return rc;
  const unsigned grid = (unsigned)((P.queries + kRows - 1) / kRows) * P.heads * P.batch;
  attention_forward_kernel<DT, DP><<<grid, kSimtThreads, bytes, s>>>(P);
  return launch_status("nt_attention_forward launch");
}

template <int DT, int DP>
static int launch_backward(const AttnParams& P, cudaStream_t s) {
  const char* who = "nt_attention_backward launch";
  const size_t bytes = (size_t)(4 * kRows * (DP + 4) + 2 * kRows * kWeightStride) * 4;
  int rc = large_smem<attention_backward_kernel<DT, DP>>(bytes, "nt_attention_backward");
  if (rc) return rc;
  if (P.queries > 0) {
    attention_rows_delta_kernel<DT><<<dim3((P.queries + 15) / 16, P.heads, P.batch), 256, 0, s>>>(P);
    rc = launch_status(who);
    if (rc) return rc;
  }
  const uint32_t key_blocks = (uint32_t)attn_pieces(P, (P.keys + kRows - 1) / kRows) * P.kv_heads * P.batch;
  const uint32_t query_blocks = (uint32_t)((P.queries + kRows - 1) / kRows) * P.heads * P.batch;
  if (key_blocks + query_blocks == 0) return NT_OK;
  // Its blocks may start while the kernel before it ends.
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(key_blocks + query_blocks);
  config.blockDim = dim3(kSimtThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = P.queries > 0 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, attention_backward_kernel<DT, DP>, P, key_blocks);
  if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, who); }
  return launch_status(who);
}

template <int DT>
static int dispatch_forward(const AttnParams& P, cudaStream_t s) {
  return P.dim <= 64 ? launch_forward<DT, 64>(P, s) : launch_forward<DT, 128>(P, s);
}
template <int DT>
static int launch_join(const AttnParams& P, int tile_rows, cudaStream_t s) {
  const unsigned runs = (tile_rows * P.dim + 1023) / 1024;
  const unsigned cut = P.rest > 1 ? (P.keys + tile_rows - 1) / tile_rows : P.sink_tiles;
  if (cut == 0) return NT_OK;
  attention_join_kernel<DT><<<runs * 2 * cut * P.batch * P.kv_heads, 256, 0, s>>>(P, tile_rows);
  return launch_status("nt_attention_backward (join) launch");
}
template <int DT>
static int dispatch_backward(const AttnParams& P, cudaStream_t s) {
  const int rc = P.dim <= 64 ? launch_backward<DT, 64>(P, s) : launch_backward<DT, 128>(P, s);
  return rc ? rc : launch_join<DT>(P, kRows, s);
}

// The window where it hides a key: 0 where it covers every position (below `positions`) or every key
// is a sink.
static int64_t effective_window(const nt_attention_args& a, int64_t positions) {
  return a.window >= positions || a.sinks >= a.keys ? 0 : a.window;
}

// Into how many pieces the backward cuts the queries of its key blocks; the pieces' sums are joined by
// a kernel of their own. Counted in steps of one block of queries:
// - where the longest ordinary block is more than an SM's share of all steps (few key heads, many
//   query heads to each, long rows), every key block is cut, to half of that share (4 query heads of
//   64 on one key head, 1000 tokens, window 100, 2 sequences, backward: 38 us uncut, 21 cut);
// - a sink block sees every later query, an ordinary one those of its own width and one window: a
//   sink block's piece is no longer than an ordinary block or piece (3000 tokens, window 200, 4 sinks, 8
//   heads on 2: all cut alike 40 us, so 31), or half of an SM's share (it starts first: long rows
//   take the same time with fewer parts to keep and join).
// The share counts the sink blocks' steps too: many sinks are most of the work, fill the SMs uncut and
// would fill the workspace cut. So the pieces of all heads together stay below some 600.
// A join costs some 4 us and a step 1 on the tensor cores but 10 on the FP32 pipe, so whole blocks are
// those of up to 16 steps there and 2 here (float32, 2 x 1024 tokens of 8 heads, window 256, backward: 294
// us with 16, 174 with 2; 300 tokens of 2 heads: 148, 62; both with the passes in one launch).
constexpr int kTcLeastPiece = 16, kLeastPiece = 2;
struct KeySplit {
  int sink_tiles, parts, rest;
};
static KeySplit key_split(const nt_attention_args& a, int tile_rows, int step_rows, int least) {
  auto up = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
  const int64_t window = effective_window(a, a.query_offset + a.queries), group = a.query_heads / a.kv_heads;
  const int64_t tiles = up(a.keys, tile_rows), steps = up(a.queries, step_rows);
  if (tiles == 0 || steps == 0) return {0, 1, 1};
  int64_t ordinary = window == 0 ? steps : up(tile_rows + window - 1, step_rows) + 1;
  if (ordinary > steps) ordinary = steps;
  const int64_t sinks = window > 0 ? up(a.sinks, tile_rows) : 0;   // (fewer than tiles)
  // Both passes; without a window about half of the blocks' pairs lie past the diagonal.
  const int64_t share = (sinks * steps + (tiles - sinks) * ordinary) * a.query_heads * a.batch * (window == 0 ? 1 : 2) /
                        current_sm_count();
  const int64_t longest = ordinary * group;
  int64_t piece = longest > least ? longest : least, rest = 1;
  if (piece < share / 2) piece = share / 2;
  if (longest >= least && longest > share) {
    piece = share > least ? share / 2 : least / 2;
    rest = up(longest, piece) < 32 ? up(longest, piece) : 32;
  }
  const int64_t parts = sinks > 0 ? up(steps * group, piece) : 1;
  return {parts > 1 ? (int)sinks : 0, (int)parts, (int)rest};
}

// The statistics of the backward at the start of its workspace: delta, and for float16 the norms.
struct StatisticsPlaces {
  size_t g_norm, g_top, v_top, end;   // bytes from delta on
  explicit StatisticsPlaces(const nt_attention_args& a) {
    auto bytes = [](int64_t n) { return ((size_t)n * 4 + 255) / 256 * 256; };
    auto tops = [&](int64_t rows) { return (int64_t)norm_tiles((int)rows, a.head_dim); };
    const bool norms = a.dtype == NT_F16;
    g_norm = bytes(a.batch * a.query_heads * a.queries);
    g_top = g_norm + (norms ? bytes(a.batch * a.query_heads * a.queries) : 0);
    v_top = g_top + (norms ? bytes(a.batch * a.query_heads * tops(a.queries)) : 0);
    end = v_top + (norms ? bytes(a.batch * a.kv_heads * tops(a.keys)) : 0);
  }
};

static void set_split(AttnParams& P, const KeySplit& split) {
  P.sink_tiles = split.sink_tiles;
  P.parts = split.parts;
  P.rest = split.rest;
}

static size_t partial_bytes(const nt_attention_args& a, int tile_rows, int step_rows, int least) {
  AttnParams P{};
  set_split(P, key_split(a, tile_rows, step_rows, least));
  return (size_t)a.batch * a.kv_heads * attn_joined(P, (int)((a.keys + tile_rows - 1) / tile_rows)) * 2 * tile_rows * a.head_dim * 4;
}

static int check_attention(const nt_attention_args& a, const char* who) {
  if (dtype_size(a.dtype) == 0) { set_error("%s: unsupported dtype %d", who, a.dtype); return NT_EUNSUPPORTED; }
  if (a.head_dim < 1 || a.head_dim > NT_ATTENTION_MAX_HEAD_DIM) {
    set_error("%s: head_dim must be in [1, %d]", who, NT_ATTENTION_MAX_HEAD_DIM);
    return NT_EINVAL;
  }
  if (a.batch < 0 || a.queries < 0 || a.keys < 0 || a.kv_heads < 1 || a.query_heads < 1 || a.query_heads % a.kv_heads) {
    set_error("%s: sizes must be nonnegative and query_heads a positive multiple of kv_heads", who);
    return NT_EINVAL;
  }
  if (a.batch > 65535 || a.query_heads > 65535 || a.keys >= INT_MAX / 2 || a.queries >= INT_MAX / 2) {
    set_error("%s: batch and heads must be below 65536, queries and keys below 2^30", who);
    return NT_EINVAL;
  }
  if ((a.queries + kRows - 1) / kRows * (a.query_heads / a.kv_heads) > INT_MAX) {
    set_error("%s: too many queries for one key head", who);
    return NT_EINVAL;
  }
  if (a.batch * a.query_heads * ((a.queries + kRows - 1) / kRows + 1) > INT_MAX ||
      a.batch * a.kv_heads * (((a.keys > a.queries ? a.keys : a.queries) + kRows - 1) / kRows + 1) > INT_MAX) {
    set_error("%s: too many blocks of queries or keys", who);
    return NT_EINVAL;
  }
  if (a.window < 0 || a.sinks < 0 || a.query_offset < 0 || a.query_offset >= INT_MAX / 2) {
    set_error("%s: window, sinks and query_offset must be nonnegative, query_offset below 2^30", who);
    return NT_EINVAL;
  }
  if (!(a.scale > 0.0f) || !std::isfinite(a.scale)) { set_error("%s: scale must be positive and finite", who); return NT_EINVAL; }
  return NT_OK;
}

// Zero from the moment the library is there: a word that were allocated and cleared on a stream could be
// cleared again by every replay of a graph, or after a kernel of another stream has set it.
static __device__ int32_t attention_error_word;

static AttnStrides strides(const int64_t* s) { return {s[0], s[1], s[2]}; }

// Rows are whole 16-byte vectors at 16-byte aligned addresses (the stride of a dimension of
// one element does not matter); strides are those a tiled copy takes.
static bool vector_rows(const nt_attention_args& a, const void* p, const int64_t* s, int64_t heads, int64_t tokens) {
  const int es = dtype_size(a.dtype);
  const int64_t sizes[3] = {a.batch, heads, tokens};
  if (!p) return true;
  if (!aligned16(p) || a.head_dim * es % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && (s[i] * es % 16 || s[i] <= 0 || s[i] > ((int64_t)1 << 38) / es)) return false;
  return true;
}
static bool vector_query(const nt_attention_args& a, const void* p, const int64_t* s) {
  return vector_rows(a, p, s, a.query_heads, a.queries);
}
static bool vector_key(const nt_attention_args& a, const void* p, const int64_t* s) {
  return vector_rows(a, p, s, a.kv_heads, a.keys);
}

// `positions`: every query stands below it.
static AttnParams attention_params(const nt_attention_args& a, int64_t positions) {
  AttnParams P{};
  P.q = a.query; P.k = a.key; P.v = a.value; P.g = a.gradient; P.o = a.output;
  P.dq = a.grad_query; P.dk = a.grad_key; P.dv = a.grad_value;
  P.qs = strides(a.query_strides); P.ks = strides(a.key_strides); P.vs = strides(a.value_strides);
  P.gs = strides(a.gradient_strides); P.os = strides(a.output_strides); P.dqs = strides(a.grad_query_strides);
  P.dks = strides(a.grad_key_strides); P.dvs = strides(a.grad_value_strides);
  P.o_low = a.output_low; P.lse = a.lse; P.lengths = a.lengths; P.error = a.error;
  P.batch = (int)a.batch; P.heads = (int)a.query_heads; P.kv_heads = (int)a.kv_heads;
  P.group = (int)(a.query_heads / a.kv_heads); P.queries = (int)a.queries; P.keys = (int)a.keys; P.dim = a.head_dim;
  P.window = (int)effective_window(a, positions);
  P.sinks = P.window == 0 ? 0 : (int)a.sinks;
  P.offset = (int)a.query_offset;
  P.scale = a.scale;
  P.scale_log2 = a.scale * kLog2eF;
  P.parts = P.rest = 1;
  return P;
}

}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_attention_workspace_size(const nt_attention_args* args) {
  if (!args || check_attention(*args, "nt_attention_workspace_size")) return 0;
  const size_t a = partial_bytes(*args, kRows, kRows, kLeastPiece);
  const size_t b = args->dtype == NT_F32 ? 0 : partial_bytes(*args, kTcKeyRows, tc_query_step(args->head_dim), kTcLeastPiece);
  return StatisticsPlaces(*args).end + (a > b ? a : b);
}

int nt_attention_forward(const nt_attention_args* args, void* stream) {
  nt::TraceRange trace("nt_attention_forward");
  if (!args) { set_error("nt_attention_forward: args is NULL"); return NT_EINVAL; }
  const nt_attention_args& a = *args;
  int rc = check_attention(a, "nt_attention_forward");
  if (rc) return rc;
  if (a.batch == 0 || a.queries == 0) return NT_OK;
  if (!a.query || !a.output || (a.keys > 0 && (!a.key || !a.value))) {
    set_error("nt_attention_forward: NULL query/key/value/output");
    return NT_EINVAL;
  }
  AttnParams P = attention_params(a, a.query_offset + a.queries);
  P.vec = vector_query(a, a.query, a.query_strides) && vector_key(a, a.key, a.key_strides) &&
          vector_key(a, a.value, a.value_strides);
  cudaStream_t s = as_stream(stream);
  if (a.dtype != NT_F32 && a.keys > 0 && P.vec && vector_query(a, a.output, a.output_strides) &&
      vector_query(a, a.output_low, a.output_strides))
    return attention_tc_forward_launch(P, a.dtype, s);
  switch (a.dtype) {
    case NT_F32: return dispatch_forward<NT_F32>(P, s);
    case NT_F16: return dispatch_forward<NT_F16>(P, s);
    default: return dispatch_forward<NT_BF16>(P, s);
  }
}

int nt_attention_backward(const nt_attention_args* args, void* stream) {
  nt::TraceRange trace("nt_attention_backward");
  if (!args) { set_error("nt_attention_backward: args is NULL"); return NT_EINVAL; }
  const nt_attention_args& a = *args;
  int rc = check_attention(a, "nt_attention_backward");
  if (rc) return rc;
  if (a.batch == 0 || (a.queries == 0 && a.keys == 0)) return NT_OK;
  if (a.queries > 0 && (!a.query || !a.output || !a.gradient || !a.grad_query || !a.lse)) {
    set_error("nt_attention_backward: NULL query/output/gradient/grad_query/lse");
    return NT_EINVAL;
  }
  if (a.keys > 0 && (!a.key || !a.value || !a.grad_key || !a.grad_value)) {
    set_error("nt_attention_backward: NULL key/value/grad_key/grad_value");
    return NT_EINVAL;
  }
  const size_t need = nt_attention_workspace_size(&a);
  if (need > 0 && (!a.workspace || a.workspace_bytes < need || !aligned16(a.workspace))) {
    set_error("nt_attention_backward: needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, a.workspace_bytes);
    return NT_EINVAL;
  }
  AttnParams P = attention_params(a, a.query_offset + a.queries);
  const StatisticsPlaces places(a);
  auto at = [&](size_t bytes) { return reinterpret_cast<float*>(static_cast<char*>(a.workspace) + bytes); };
  P.delta = at(0);
  P.g_norm = at(places.g_norm);
  P.g_top = at(places.g_top);
  P.v_top = at(places.v_top);
  P.partial = at(places.end);
  P.vec = vector_query(a, a.query, a.query_strides) && vector_key(a, a.key, a.key_strides) &&
          vector_key(a, a.value, a.value_strides) && vector_query(a, a.gradient, a.gradient_strides) &&
          vector_query(a, a.output, a.output_strides);
  const bool tc = a.dtype != NT_F32 && a.keys > 0 && a.queries > 0 && P.vec &&
                  vector_query(a, a.output_low, a.output_strides) && vector_query(a, a.grad_query, a.grad_query_strides) &&
                  vector_key(a, a.grad_key, a.grad_key_strides) && vector_key(a, a.grad_value, a.grad_value_strides);
  const int tile_rows = tc ? kTcKeyRows : kRows;
  set_split(P, tc ? key_split(a, kTcKeyRows, tc_query_step(a.head_dim), kTcLeastPiece) : key_split(a, kRows, kRows, kLeastPiece));
  cudaStream_t s = as_stream(stream);
  if (tc) {
    rc = attention_tc_backward_launch(P, a.dtype, s);
    if (rc) return rc;
    return a.dtype == NT_F16 ? launch_join<NT_F16>(P, tile_rows, s) : launch_join<NT_BF16>(P, tile_rows, s);
  }
  switch (a.dtype) {
    case NT_F32: return dispatch_backward<NT_F32>(P, s);
    case NT_F16: return dispatch_backward<NT_F16>(P, s);
    default: return dispatch_backward<NT_BF16>(P, s);
  }
}

int nt_attention_step(const nt_attention_args* args, void* stream) {
  nt::TraceRange trace("nt_attention_step");
  if (!args) { set_error("nt_attention_step: args is NULL"); return NT_EINVAL; }
  const nt_attention_args& a = *args;
  int rc = check_attention(a, "nt_attention_step");
  if (rc) return rc;
  if (a.queries != 1) { set_error("nt_attention_step: queries must be 1"); return NT_EINVAL; }
  if (a.batch == 0) return NT_OK;
  if (!a.query || !a.output || !a.lengths || (a.keys > 0 && (!a.key || !a.value))) {
    set_error("nt_attention_step: NULL query/key/value/lengths/output");
    return NT_EINVAL;
  }
  AttnParams P = attention_params(a, a.keys);
  P.vec = vector_key(a, a.key, a.key_strides) && vector_key(a, a.value, a.value_strides);
  return attention_step_launch(P, a.dtype, as_stream(stream));
}

int nt_attention_error_word(int32_t** word) {
  if (!word) { set_error("nt_attention_error_word: word is NULL"); return NT_EINVAL; }
  void* p = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&p, attention_error_word);
  if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, "nt_attention_error_word"); }
  *word = static_cast<int32_t*>(p);
  return NT_OK;
}

}  // extern "C"
