// Launchers of the KV page kernels (pages.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_paged_attn.h"

namespace b200 {

int launch_copy_kv_pages(const b200_cache_desc* cache, const void* src, const void* dst,
                         const void* tokens, int32_t index_dtype, int64_t num_pairs,
                         uint32_t* error_word, cudaStream_t stream);

int launch_remap_block_tables(const void* tables, int32_t table_dtype, int64_t table_stride,
                              int64_t num_rows, int32_t table_width, const int32_t* page_map,
                              int32_t num_blocks, void* out, int64_t out_stride,
                              uint32_t* error_word, cudaStream_t stream);

}  // namespace b200
