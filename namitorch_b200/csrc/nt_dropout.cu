// Dropout from a counter-based generator, with the bias before it and the residual after it:
//   y = residual + keep(e) (x + bias) / (1 - p),   dx = keep(e) g / (1 - p),   dbias = sum over rows of dx
// keep(e) is a function of (seed, offset, e) alone: word e % 4 of Philox4x32-7 at the counter
// (e / 4, offset). Forward and backward compute it where they need it, so no mask is written
// or read. Seven rounds are the fewest that pass the Crush batteries (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).
//
// Bound: HBM (x, residual in, y out; g in, dx out). One Philox call (7 rounds of two 32 x 32 ->
// 64 products) gives four elements. 16384 x 2048 bfloat16: forward 33 us, 93 % of the measured copy rate;
// backward with the bias gradient 31 and 4, 66 % in its first kernel: its warps, 39 % of those an SM
// holds, wait for the multiplier (2.3 of some 7 cycles between two instructions of a warp) and for the
// four rows they load (1.5), which no other row's work covers (the rows left over after fours, loaded
// ahead too, cost an eighth of the blocks: 33). float32: 64 and 51 us, 96 and 81 %. Widths that are no
// multiple of 8, and unaligned tensors, go element by element: 16384 x 2047 bfloat16 86 and 90 us.
#include <cmath>

#include "nt_rows.cuh"

namespace nt {

struct DropoutParams {
  const void* x;
  const void* bias;
  const void* residual;
  void* y;
  float* partial;
  int64_t rows;
  int64_t width;
  uint32_t threshold;
  float scale;
  uint32_t offset0, offset1;
  uint32_t keys[7][2];   // of the rounds: operands in constant memory, nothing to compute per call
};

__device__ __forceinline__ uint4 philox7(uint64_t counter, const DropoutParams& P) {
  uint32_t a = (uint32_t)counter, b = (uint32_t)(counter >> 32), c = P.offset0, d = P.offset1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t x = (uint64_t)a * 0xD2511F53u, y = (uint64_t)c * 0xCD9E8D57u;
    a = (uint32_t)(y >> 32) ^ b ^ P.keys[r][0];
    b = (uint32_t)y;
    c = (uint32_t)(x >> 32) ^ d ^ P.keys[r][1];
    d = (uint32_t)x;
  }
  return make_uint4(a, b, c, d);
}

// Columns one thread holds. A row of the tensor is dealt to CX threads of a block, V columns
// each; the block covers RY rows at a time and walks down the rows, so that a thread keeps its
// columns: the bias is loaded once and the bias gradient summed in registers.
constexpr int kDropoutColumns = 8;
constexpr int kDropoutThreads = 256;
constexpr int kAhead = 4;
// Partial rows of the bias gradient (row slots of the grid) at most.
constexpr int64_t kDropoutMaxSlots = 1024;

// Which of the V columns from flat element e0 are kept. On the vector path e0 is a multiple of 8;
// otherwise a thread's columns start anywhere in a counter's four words,
// and one more counter than V / 4 covers them.
template <bool VEC>
__device__ __forceinline__ void keep_columns(int64_t e0, const DropoutParams& P, bool (&keep)[kDropoutColumns]) {
  constexpr int V = kDropoutColumns;
  const uint64_t counter = (uint64_t)e0 >> 2;
  if constexpr (VEC) {
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
      const uint4 w = philox7(counter + c, P);
      keep[4 * c] = w.x >= P.threshold;
      keep[4 * c + 1] = w.y >= P.threshold;
      keep[4 * c + 2] = w.z >= P.threshold;
      keep[4 * c + 3] = w.w >= P.threshold;
    }
  } else {
    uint32_t w[V + 4];
#pragma unroll
    for (int c = 0; c < V / 4 + 1; ++c) {
      const uint4 r = philox7(counter + c, P);
      w[4 * c] = r.x; w[4 * c + 1] = r.y; w[4 * c + 2] = r.z; w[4 * c + 3] = r.w;
    }
    const int shift = (int)(e0 & 3);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const uint32_t lo = shift & 1 ? w[k + 1] : w[k], hi = shift & 1 ? w[k + 3] : w[k + 2];
      keep[k] = (shift & 2 ? hi : lo) >= P.threshold;
    }
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void load_columns(const void* base, int64_t e0, int live, float (&v)[kDropoutColumns]) {
  if constexpr (VEC) {
    load8<DT>(base, e0, v);
  } else {
#pragma unroll
    for (int k = 0; k < kDropoutColumns; ++k) v[k] = k < live ? load1<DT>(base, e0 + k) : 0.0f;
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_columns(void* base, int64_t e0, int live, const float (&v)[kDropoutColumns]) {
  if constexpr (VEC) {
    store8<DT>(base, e0, v);
  } else {
#pragma unroll
    for (int k = 0; k < kDropoutColumns; ++k)
      if (k < live) store1<DT>(base, e0 + k, v[k]);
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kDropoutThreads) dropout_forward_kernel(const __grid_constant__ DropoutParams P) {
  constexpr int V = kDropoutColumns;
  const int64_t c0 = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (c0 >= P.width) return;
  const int live = (int)min((int64_t)V, P.width - c0);
  float b[V];
#pragma unroll
  for (int k = 0; k < V; ++k) b[k] = P.bias != nullptr && k < live ? load1<DT>(P.bias, c0 + k) : 0.0f;
  const int64_t stride = (int64_t)gridDim.y * blockDim.y;
#pragma unroll 2
  for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < P.rows; row += stride) {
    const int64_t e0 = row * P.width + c0;
    float x[V], r[V];
    bool keep[V];
    load_columns<DT, VEC>(P.x, e0, live, x);
    if (P.residual != nullptr) load_columns<DT, VEC>(P.residual, e0, live, r);
    else {
#pragma unroll
      for (int k = 0; k < V; ++k) r[k] = 0.0f;
    }
    keep_columns<VEC>(e0, P, keep);
    // A dropped element contributes exactly 0, whatever x holds (0 * inf would be NaN).
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = keep[k] ? fmaf(x[k] + b[k], P.scale, r[k]) : r[k];
    store_columns<DT, VEC>(P.y, e0, live, r);
  }
}

// AFFINE: the block also sums its rows of dx per column (in 32 bits, in row order; the RY row
// groups are added in order in shared memory) and writes one partial row; the reduction kernel
// adds the partial rows in a fixed order.
template <int DT, bool VEC, bool AFFINE>
__global__ void __launch_bounds__(kDropoutThreads) dropout_backward_kernel(const __grid_constant__ DropoutParams P) {
  constexpr int V = kDropoutColumns;
  __shared__ float sums[AFFINE ? kDropoutThreads * V : 1];
  const int64_t c0 = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  const int live = (int)max((int64_t)0, min((int64_t)V, P.width - c0));
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  if (live > 0) {
    const int64_t stride = (int64_t)gridDim.y * blockDim.y;
    auto body = [&](int64_t e0, float (&g)[V]) {
      bool keep[V];
      keep_columns<VEC>(e0, P, keep);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        g[k] = keep[k] ? g[k] * P.scale : 0.0f;
        if constexpr (AFFINE) acc[k] += g[k];
      }
      if (P.y != nullptr) store_columns<DT, VEC>(P.y, e0, live, g);
    };
    int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y;
    if constexpr (VEC) {
      // kAhead rows in flight, packed as they came.
      constexpr int N = DT == NT_F32 ? 2 : 1;
      for (; row + (kAhead - 1) * stride < P.rows; row += kAhead * stride) {
        uint4 raw[kAhead][N];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
          for (int k = 0; k < N; ++k)
            raw[i][k] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const typename Elem<DT>::T*>(P.x) +
                                                              (row + i * stride) * P.width + c0) + k);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          float g[V];
#pragma unroll
          for (int k = 0; k < N; ++k) unpack16<DT>(raw[i][k], g + k * (V / N));
          body((row + i * stride) * P.width + c0, g);
        }
      }
    }
    for (; row < P.rows; row += stride) {
      const int64_t e0 = row * P.width + c0;
      float g[V];
      load_columns<DT, VEC>(P.x, e0, live, g);
      body(e0, g);
    }
  }
  if constexpr (AFFINE) {
    const int columns = blockDim.x * V;
#pragma unroll
    for (int k = 0; k < V; ++k) sums[threadIdx.y * columns + threadIdx.x * V + k] = acc[k];
    __syncthreads();
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < columns; c += blockDim.x * blockDim.y) {
      const int64_t column = (int64_t)blockIdx.x * columns + c;
      if (column >= P.width) break;
      float s = 0.0f;
      for (int j = 0; j < (int)blockDim.y; ++j) s += sums[j * columns + c];
      P.partial[(int64_t)blockIdx.y * P.width + column] = s;
    }
  }
}

// Column sums of the partial rows: lane j of a column adds partial rows j, j + 32, ... in order,
// then the lane sums are added in lane order. (592 partial rows of 2048: 4 us of loads one behind another.)
constexpr int kReduceLanes = 32;
template <int DT>
__global__ void __launch_bounds__(32 * kReduceLanes)
dropout_bias_reduce_kernel(const float* partial, int64_t slots, int64_t width, void* out) {
  __shared__ float lanes[kReduceLanes][32];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < width)
#pragma unroll 4
    for (int64_t k = threadIdx.y; k < slots; k += kReduceLanes) s += partial[k * width + c];
  lanes[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
#pragma unroll
    for (int j = 1; j < kReduceLanes; ++j) s += lanes[j][threadIdx.x];
    store1<DT>(out, c, s);
  }
}

struct DropoutGrid {
  dim3 grid, block;
};

// Blocks of CX x RY threads over [rows, width / 8]: rows wider than 256 threads are cut into
// equal parts, narrow ones share a block; the grid holds as many row slots as the device runs at
// once, at most `most`.
template <typename K>
static DropoutGrid dropout_grid(K kernel, int64_t rows, int64_t width, int64_t most) {
  const int64_t groups = (width + kDropoutColumns - 1) / kDropoutColumns;
  const int64_t parts = (groups + kDropoutThreads - 1) / kDropoutThreads;
  const int64_t cx = (groups + parts - 1) / parts;
  const int64_t ry = kDropoutThreads / cx;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, (int)(cx * ry), 0) != cudaSuccess || per_sm < 1) per_sm = 4;
  int64_t slots = (int64_t)current_sm_count() * per_sm / parts;
  if (slots > (rows + ry - 1) / ry) slots = (rows + ry - 1) / ry;
  if (slots > most) slots = most;
  if (slots < 1) slots = 1;
  return {dim3((unsigned)parts, (unsigned)slots), dim3((unsigned)cx, (unsigned)ry)};
}

template <int DT, bool VEC>
static int launch_dropout_forward(const DropoutParams& P, cudaStream_t s) {
  const DropoutGrid g = dropout_grid(dropout_forward_kernel<DT, VEC>, P.rows, P.width, 65535);
  dropout_forward_kernel<DT, VEC><<<g.grid, g.block, 0, s>>>(P);
  return launch_status("nt_dropout_forward launch");
}

template <int DT, bool VEC>
static int launch_dropout_backward(const DropoutParams& P, void* grad_bias, cudaStream_t s) {
  if (grad_bias == nullptr) {
    const DropoutGrid g = dropout_grid(dropout_backward_kernel<DT, VEC, false>, P.rows, P.width, 65535);
    dropout_backward_kernel<DT, VEC, false><<<g.grid, g.block, 0, s>>>(P);
    return launch_status("nt_dropout_backward launch");
  }
  const DropoutGrid g = dropout_grid(dropout_backward_kernel<DT, VEC, true>, P.rows, P.width, kDropoutMaxSlots);
  dropout_backward_kernel<DT, VEC, true><<<g.grid, g.block, 0, s>>>(P);
  int rc = launch_status("nt_dropout_backward launch");
  if (rc) return rc;
  dropout_bias_reduce_kernel<DT><<<(unsigned)((P.width + 31) / 32), dim3(32, kReduceLanes), 0, s>>>(
      P.partial, g.grid.y, P.width, grad_bias);
  return launch_status("nt_dropout_backward (reduce) launch");
}

template <bool VEC>
static int dispatch_dropout_forward(const DropoutParams& P, int dtype, cudaStream_t s) {
  switch (dtype) {
    case NT_F32: return launch_dropout_forward<NT_F32, VEC>(P, s);
    case NT_F16: return launch_dropout_forward<NT_F16, VEC>(P, s);
    default: return launch_dropout_forward<NT_BF16, VEC>(P, s);
  }
}

template <bool VEC>
static int dispatch_dropout_backward(const DropoutParams& P, int dtype, void* grad_bias, cudaStream_t s) {
  switch (dtype) {
    case NT_F32: return launch_dropout_backward<NT_F32, VEC>(P, grad_bias, s);
    case NT_F16: return launch_dropout_backward<NT_F16, VEC>(P, grad_bias, s);
    default: return launch_dropout_backward<NT_BF16, VEC>(P, grad_bias, s);
  }
}

static int check_dropout(const nt_dropout_args& a, const char* who, DropoutParams* P) {
  if (dtype_size(a.dtype) == 0) { set_error("%s: unsupported dtype %d", who, a.dtype); return NT_EUNSUPPORTED; }
  if (a.rows < 0 || a.width < 0 || (a.width > 0 && a.rows > INT64_MAX / 16 / a.width) || a.width > (int64_t)1 << 36) {
    set_error("%s: rows and width must be nonnegative and their product a valid size", who);
    return NT_EINVAL;
  }
  if (!(a.p >= 0.0 && a.p < 1.0)) { set_error("%s: p must be in [0, 1)", who); return NT_EINVAL; }
  P->rows = a.rows;
  P->width = a.width;
  P->threshold = (uint32_t)floor(a.p * 4294967296.0);
  P->scale = (float)(1.0 / (1.0 - a.p));
  for (uint32_t r = 0; r < 7; ++r) {
    P->keys[r][0] = (uint32_t)a.seed + r * 0x9E3779B9u;
    P->keys[r][1] = (uint32_t)(a.seed >> 32) + r * 0xBB67AE85u;
  }
  P->offset0 = (uint32_t)a.offset;
  P->offset1 = (uint32_t)(a.offset >> 32);
  return NT_OK;
}

}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_dropout_workspace_size(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1) return 0;
  return (size_t)(rows < kDropoutMaxSlots ? rows : kDropoutMaxSlots) * (size_t)width * sizeof(float);
}

int nt_dropout_forward(const nt_dropout_args* args, void* stream) {
  nt::TraceRange trace("nt_dropout_forward");
  if (!args) { set_error("nt_dropout_forward: args is NULL"); return NT_EINVAL; }
  const nt_dropout_args& a = *args;
  DropoutParams P{};
  int rc = check_dropout(a, "nt_dropout_forward", &P);
  if (rc) return rc;
  if (a.rows == 0 || a.width == 0) return NT_OK;
  if (!a.input || !a.output) { set_error("nt_dropout_forward: NULL input/output"); return NT_EINVAL; }
  P.x = a.input; P.bias = a.bias; P.residual = a.residual; P.y = a.output;
  const bool vec = a.width % kDropoutColumns == 0 && aligned16(a.input) && aligned16(a.output) &&
                   (!a.residual || aligned16(a.residual));
  cudaStream_t s = as_stream(stream);
  return vec ? dispatch_dropout_forward<true>(P, a.dtype, s) : dispatch_dropout_forward<false>(P, a.dtype, s);
}

int nt_dropout_backward(const nt_dropout_args* args, void* stream) {
  nt::TraceRange trace("nt_dropout_backward");
  if (!args) { set_error("nt_dropout_backward: args is NULL"); return NT_EINVAL; }
  const nt_dropout_args& a = *args;
  DropoutParams P{};
  int rc = check_dropout(a, "nt_dropout_backward", &P);
  if (rc) return rc;
  cudaStream_t s = as_stream(stream);
  if (a.width == 0 || (!a.output && !a.grad_bias)) return NT_OK;
  if (a.rows == 0) {
    if (!a.grad_bias) return NT_OK;
    cudaError_t e = cudaMemsetAsync(a.grad_bias, 0, (size_t)a.width * dtype_size(a.dtype), s);
    return e == cudaSuccess ? NT_OK : cuda_fail(e, "nt_dropout_backward");
  }
  if (!a.input) { set_error("nt_dropout_backward: NULL input"); return NT_EINVAL; }
  if (a.grad_bias) {
    const size_t need = nt_dropout_workspace_size(a.rows, a.width);
    if (!a.workspace || a.workspace_bytes < need) {
      set_error("nt_dropout_backward: the bias gradient needs a workspace of %zu bytes (got %zu)", need, a.workspace_bytes);
      return NT_EINVAL;
    }
  }
  P.x = a.input; P.y = a.output; P.partial = static_cast<float*>(a.workspace);
  const bool vec = a.width % kDropoutColumns == 0 && aligned16(a.input) && (!a.output || aligned16(a.output));
  return vec ? dispatch_dropout_backward<true>(P, a.dtype, a.grad_bias, s)
             : dispatch_dropout_backward<false>(P, a.dtype, a.grad_bias, s);
}

}  // extern "C"
