// Launcher of the token sampling kernel (sample.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_paged_attn.h"

namespace b200 {

int launch_sample_tokens(const b200_sample_args* args, const void* logits, const float* uniforms,
                         const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, int64_t* tokens, float* logprobs,
                         float* sampling_logprobs, cudaStream_t stream);

}  // namespace b200
