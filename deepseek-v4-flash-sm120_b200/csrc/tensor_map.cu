// TMA tensor maps for the kernels that load 16-bit rows in boxes of 64 values.
#include "tensor_map.h"

#include <mutex>

namespace dsv4 {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, looked up once (the library links no driver library).
cudaError_t encoder(EncodeTiled* out) {
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  static EncodeTiled fn = nullptr;
  if (fn == nullptr) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult st;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &st);
    if (e) return e;
    if (st != cudaDriverEntryPointSuccess || f == nullptr) return cudaErrorNotSupported;
    fn = reinterpret_cast<EncodeTiled>(f);
  }
  *out = fn;
  return cudaSuccess;
}

}  // namespace

cudaError_t make_map_16bit(CUtensorMap* m, bool bf16, const void* ptr, int tokens, int heads, int d, int64_t stride_t,
                           int64_t stride_h, int box_t, int box_h) {
  EncodeTiled enc;
  cudaError_t e = encoder(&enc);
  if (e) return e;
  // the stride of a dimension of one element is never used, but has to be a legal one
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? stride_h : d) * 2,
                                 static_cast<cuuint64_t>(tokens > 1 ? stride_t : d) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_h), static_cast<cuuint32_t>(box_t)};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace dsv4
