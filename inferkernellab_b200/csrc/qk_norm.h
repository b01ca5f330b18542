// Launcher of the per-head norm + rotary + KV append kernel (qk_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_paged_attn.h"

namespace b200 {

int launch_qk_norm_rope_append(const b200_cache_desc* cache, const b200_qk_norm_args* args,
                               const void* query, const void* key, const void* value,
                               const void* q_weight, const void* k_weight, const void* cos,
                               const void* sin, const void* slots, void* query_out,
                               uint32_t* error_word, cudaStream_t stream);

}  // namespace b200
