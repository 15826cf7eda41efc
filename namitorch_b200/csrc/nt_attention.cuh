// What the attention kernels share: the problem, which keys a query sees, and the ranges of
// keys (of a block of queries) and of queries (of a block of keys) that hold every visible pair.
#pragma once

#include <cuda.h>

#include "nt_common.cuh"

namespace nt {

// Element strides of the first three dimensions: batch, head, token.
struct AttnStrides {
  int64_t b, h, t;
  __host__ __device__ __forceinline__ int64_t at(int64_t batch, int64_t head, int64_t token) const {
    return batch * b + head * h + token * t;
  }
};

struct AttnParams {
  const void *q, *k, *v, *g;
  void *o, *dq, *dk, *dv;
  void* o_low;       // what rounding took from o, in o's type and strides, or NULL
  AttnStrides qs, ks, vs, gs, os, dqs, dks, dvs;
  float* lse;        // [batch, heads, queries]
  float* delta;      // [batch, heads, queries]: sum over head_dim of g * o
  // Tensor-core backward of float16: the row norms of g [batch, heads, queries], and the largest of
  // each norm_rows rows of g [batch, heads, ..] and of v [batch, kv_heads, ..] (attention_delta_norms_kernel).
  float *g_norm, *g_top, *v_top;
  float* partial;    // backward: partial gradients of the split key blocks
  const int32_t* lengths;
  int32_t* error;
  int batch, heads, kv_heads, group, queries, keys, dim;
  int window;        // 0: none
  int sinks;         // 0 without a window
  int offset;
  int vec;           // rows are 16-byte aligned runs of whole 16-byte vectors
  // Backward over key blocks: the queries of the first `sink_tiles` blocks are cut into `parts`
  // pieces, those of the others into `rest`. Pieces count on through the blocks of a key head; with
  // rest = 1 the others have none, they are whole.
  int sink_tiles, parts, rest;
  int splits;        // forward: blocks of a cluster that share a block of queries
  float scale, scale_log2;
};

constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kLn2F = 0.6931471805599453f;

__device__ __forceinline__ int attn_length(const AttnParams& P, int b) {
  return P.lengths == nullptr ? P.keys : min(max(P.lengths[b], 0), P.keys);
}

__device__ __forceinline__ bool attn_visible(const AttnParams& P, int length, int p, int j) {
  return j < length && j <= p && (P.window == 0 || p - j < P.window || j < P.sinks);
}

// How many keys query i sees. One key has the weight 1 whatever its score is, so dS of a query that sees
// one is 0: what is left of P (dP - delta) in float32 is not the gradient of anything.
__device__ __forceinline__ int attn_key_count(const AttnParams& P, int length, int i) {
  const int end = min(length, P.offset + i + 1);
  const int start = P.window == 0 ? 0 : min(max(P.offset + i + 1 - P.window, 0), end);
  return end - start + min(P.sinks, start);
}

// Keys that queries [i0, i1) see: [0, sink_end) and [lo, hi), disjoint. The window's range
// starts where the first query's window does, not at a multiple of the block.
struct AttnKeys {
  int sink_end, lo, hi;
  __device__ __forceinline__ AttnKeys(const AttnParams& P, int length, int i0, int i1) {
    hi = min(length, P.offset + i1);
    lo = P.window == 0 ? 0 : min(hi, max(0, P.offset + i0 - P.window + 1));
    sink_end = min(P.sinks, hi);
    if (lo <= sink_end) { lo = 0; sink_end = 0; }
  }
  __device__ __forceinline__ int sink_blocks(int width) const { return (sink_end + width - 1) / width; }
  __device__ __forceinline__ int blocks(int width) const { return sink_blocks(width) + (hi - lo + width - 1) / width; }
  // First key and end (exclusive) of block j.
  __device__ __forceinline__ void block(int j, int width, int& begin, int& end) const {
    const int s = sink_blocks(width);
    begin = j < s ? j * width : lo + (j - s) * width;
    end = min(begin + width, j < s ? sink_end : hi);
  }
};

// Queries [lo, hi) that see a key of [k0, k1).
struct AttnQueries {
  int lo, hi;
  __device__ __forceinline__ AttnQueries(const AttnParams& P, int length, int k0, int k1) {
    const int64_t last = P.window == 0 || k0 < P.sinks ? (int64_t)P.queries
                                                        : (int64_t)k1 - 1 + P.window - P.offset;
    lo = max(0, k0 - P.offset);
    hi = (int)(last < P.queries ? last : P.queries);
    if (k0 >= length || hi < lo) hi = lo;
  }
};

// Key block and piece of block `index` of a key head.
struct AttnPiece {
  int tile, part, parts;
  __device__ __forceinline__ AttnPiece(const AttnParams& P, int index) {
    const int first = P.sink_tiles * P.parts;
    parts = index < first ? P.parts : P.rest;
    tile = index < first ? index / P.parts : P.sink_tiles + (index - first) / P.rest;
    part = (index < first ? index : index - first) % parts;
  }
};
// Pieces of all `tiles` key blocks of a key head, and those among them whose sums are joined.
__host__ __device__ inline int attn_pieces(const AttnParams& P, int tiles) {
  return P.sink_tiles * P.parts + (tiles - P.sink_tiles) * P.rest;
}
__host__ __device__ inline int attn_joined(const AttnParams& P, int tiles) {
  return P.rest > 1 ? attn_pieces(P, tiles) : P.parts > 1 ? P.sink_tiles * P.parts : 0;
}

// nt_attention_map.cu: tensor map (column, token, head, batch) of a 16-bit tensor with boxes of 64
// columns x `rows` tokens, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, int dtype, const void* ptr, const AttnStrides& st, int dim, int tokens, int heads, int batch,
             int rows, const char* who);
// nt_attention_step.cu: one token per sequence.
int attention_step_launch(const AttnParams& P, int dtype, cudaStream_t s);
// nt_attention_tc.cu: the tensor-core forms (16-bit types, 16-byte aligned rows).
constexpr int kTcKeyRows = 128;    // keys of a block of the key / value gradients
// Rows that share an entry of g_top and v_top, and the entries of `rows` rows.
__host__ __device__ constexpr int norm_rows(int dim) { return dim <= 64 ? 32 : 16; }
__host__ __device__ constexpr int norm_tiles(int rows, int dim) { return (rows + norm_rows(dim) - 1) / norm_rows(dim); }
constexpr int tc_query_step(int dim) { return dim <= 64 ? 64 : 128; }   // queries it takes at a time
int attention_tc_forward_launch(const AttnParams& P, int dtype, cudaStream_t s);
int attention_tc_backward_launch(const AttnParams& P, int dtype, cudaStream_t s);

}  // namespace nt
