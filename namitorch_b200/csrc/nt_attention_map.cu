// Tensor maps of the attention kernels' tiled copies.
#include "nt_attention.cuh"

namespace nt {

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
int make_map(CUtensorMap* map, int dtype, const void* ptr, const AttnStrides& st, int dim, int tokens, int heads, int batch,
             int rows, const char* who) {
  EncodeTiled encode = encode_tiled();
  if (!encode) { set_error("%s: the driver has no cuTensorMapEncodeTiled", who); return NT_ECUDA; }
  const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
  // The stride of a dimension of one element is never used, but has to be a valid one.
  const cuuint64_t row_bytes = ((cuuint64_t)dim * 2 + 15) / 16 * 16;
  const cuuint64_t strides[3] = {tokens > 1 ? (cuuint64_t)st.t * 2 : row_bytes, heads > 1 ? (cuuint64_t)st.h * 2 : row_bytes,
                                 batch > 1 ? (cuuint64_t)st.b * 2 : row_bytes};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, ones[4] = {1, 1, 1, 1};
  auto run = [&] {
    return encode(map, dtype == NT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = run();
  if (rc == CUDA_ERROR_INVALID_CONTEXT || rc == CUDA_ERROR_NOT_INITIALIZED) {
    // The encoder is a driver call, and this thread (an autograd worker's first) may have made no
    // runtime call that binds the device's context: setting the current device again does.
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err == cudaSuccess) err = cudaSetDevice(device);
    if (err != cudaSuccess) return cuda_fail(err, who);
    rc = run();
  }
  if (rc != CUDA_SUCCESS) { set_error("%s: cuTensorMapEncodeTiled failed (%d)", who, (int)rc); return NT_ECUDA; }
  return NT_OK;
}

}  // namespace nt
