// Launcher of the 8-bit block-scaled product (fp8_linear.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_paged_attn.h"

namespace b200 {

int launch_fp8_linear(const b200_fp8_linear_args* args, const void* x, const float* x_scales,
                      const void* w, const float* w_scales, const void* bias, void* out,
                      void* workspace, size_t workspace_bytes, uint32_t* error_word,
                      cudaStream_t stream);

}  // namespace b200
