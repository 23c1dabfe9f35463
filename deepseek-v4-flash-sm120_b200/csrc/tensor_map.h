// TMA tensor maps of [tokens, heads, d] tensors of 16-bit values (tensor_map.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv4 {

// Boxes of `box_t` tokens, `box_h` heads and 64 values, 128-byte swizzle; strides in elements.
cudaError_t make_map_16bit(CUtensorMap* m, bool bf16, const void* ptr, int tokens, int heads, int d, int64_t stride_t,
                           int64_t stride_h, int box_t, int box_h);

}  // namespace dsv4
