// Launcher of the 8-bit quantisation kernels (fp8_quant.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

int launch_quantize_fp8(const void* x, int64_t rows, int64_t cols, int64_t x_stride, int32_t dtype,
                        int32_t block_rows, void* q, int64_t q_stride, float* scales,
                        int64_t scale_stride_row, int64_t scale_stride_block,
                        cudaStream_t stream);

}  // namespace b200
