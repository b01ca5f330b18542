// Physical pages of the paged KV cache: copied to other pages in every layer,
// and block tables rewritten to new page ids.
//
//   copy:   for every pair i, layer l and token j < tokens[i] (or block_size):
//             K[l, dst[i], j] = K[l, src[i], j],  V likewise -- the bytes as they are
//   remap:  out[r, c] = page_map[table[r, c]]
//
// A fork of a request copies its last, partly filled page; compacting a pool
// moves pages and then rewrites the tables.  Bound: bytes.  A page of one layer
// is contiguous in K and in V, so a copy is 2 * layers * pairs contiguous runs;
// a CTA takes 16 KB of one run, four vectors a thread, with all of its loads in
// flight before its first store.  Measured: 900 pages x 16 layers (0.94 GB copied) and
// 256 x 512 table entries in 287.5 us, 6.57 TB/s, the measured copy rate; one page of
// 4 layers and one table row in 2.7 us, two launches.
#include <algorithm>

#include "../../include/b200_paged_attn.h"
#include "common.cuh"
#include "host_common.h"
#include "pages.h"

namespace b200 {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;  // vectors of a thread
constexpr int kRemapThreads = 256;

struct CopyParams {
  uint8_t* k;
  uint8_t* v;
  const void* src;
  const void* dst;
  const void* tokens;  // may be null: whole pages
  uint32_t* err;
  long long page_bytes, layer_bytes, num_pairs;
  long long token_bytes;
  int num_blocks, block_size, index64, chunks;
};

// grid: x = pair * chunks + chunk, y = layer, z = 0: K, 1: V.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long pair = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x % p.chunks;
  const long long from = load_index(p.src, pair, p.index64);
  const long long to = load_index(p.dst, pair, p.index64);
  long long n = p.block_size;
  if (p.tokens) n = min(max(load_index(p.tokens, pair, p.index64), 0LL), n);
  if (from < 0 || to < 0) return;  // a negative id: nothing to copy
  if (from >= p.num_blocks || to >= p.num_blocks) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadBlock);
    return;
  }
  uint8_t* base = (blockIdx.z ? p.v : p.k) + blockIdx.y * p.layer_bytes;
  const V* a = reinterpret_cast<const V*>(base + from * p.page_bytes);
  V* b = reinterpret_cast<V*>(base + to * p.page_bytes);
  const long long vecs = n * p.token_bytes / static_cast<int>(sizeof(V));
  const long long first =
      static_cast<long long>(chunk) * (kCopyThreads * kCopyVecs) + threadIdx.x;
  V x[kCopyVecs];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (first + i * kCopyThreads < vecs) x[i] = a[first + i * kCopyThreads];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (first + i * kCopyThreads < vecs) b[first + i * kCopyThreads] = x[i];
}

struct RemapParams {
  const void* tables;
  const int* page_map;
  void* out;
  uint32_t* err;
  long long in_stride, out_stride;
  long long total;
  int width, num_blocks, table64;
};

__global__ void __launch_bounds__(kRemapThreads) remap_tables_kernel(const RemapParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long at = blockIdx.x * static_cast<long long>(kRemapThreads) + threadIdx.x;
  if (at >= p.total) return;
  const long long row = at / p.width;
  const long long col = at - row * p.width;
  long long id = load_index(p.tables, row * p.in_stride + col, p.table64);
  if (id >= 0 && id < p.num_blocks)
    id = p.page_map[id];
  else if (id >= p.num_blocks && p.err)
    atomicOr(p.err, kErrBadBlock);
  if (p.table64)
    reinterpret_cast<long long*>(p.out)[row * p.out_stride + col] = id;
  else
    reinterpret_cast<int*>(p.out)[row * p.out_stride + col] = static_cast<int>(id);
}

}  // namespace

int launch_copy_kv_pages(const b200_cache_desc* c, const void* src, const void* dst,
                         const void* tokens, int32_t index_dtype, int64_t num_pairs,
                         uint32_t* error_word, cudaStream_t stream) {
  if (c == nullptr) return set_error(B200_ERR_INVALID, "null descriptor");
  if (c->num_layers <= 0 || c->num_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 ||
      c->head_dim <= 0)
    return set_error(B200_ERR_INVALID, "cache dimensions must be positive");
  if (c->dtype != B200_F16 && c->dtype != B200_BF16)
    return set_error(B200_ERR_UNSUPPORTED, "cache dtype must be float16 or bfloat16");
  if (index_dtype != B200_I32 && index_dtype != B200_I64)
    return set_error(B200_ERR_INVALID, "index dtype must be int32 or int64");
  if (num_pairs < 0) return set_error(B200_ERR_INVALID, "the page count must be non-negative");
  if (num_pairs == 0) return B200_OK;
  if (!src || !dst || !c->k_cache || !c->v_cache)
    return set_error(B200_ERR_INVALID, "null tensor pointer");
  CopyParams p;
  p.k = static_cast<uint8_t*>(c->k_cache);
  p.v = static_cast<uint8_t*>(c->v_cache);
  p.src = src;
  p.dst = dst;
  p.tokens = tokens;
  p.err = error_word;
  p.num_pairs = num_pairs;
  p.token_bytes = 2LL * c->num_kv_heads * c->head_dim;
  p.page_bytes = p.token_bytes * c->block_size;
  p.layer_bytes = p.page_bytes * c->num_blocks;
  p.num_blocks = c->num_blocks;
  p.block_size = c->block_size;
  p.index64 = index_dtype == B200_I64;
  // 16-byte vectors where every token starts on a 16-byte boundary, else one
  // 16-bit element at a time.
  const bool vec = p.token_bytes % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(c->k_cache) |
                     reinterpret_cast<uintptr_t>(c->v_cache)) & 15u) == 0;
  const long long per_chunk = static_cast<long long>(kCopyThreads) * kCopyVecs * (vec ? 16 : 2);
  const long long chunks = ceil_div64(p.page_bytes, per_chunk);
  if (num_pairs * chunks > 0x7fffffffLL || c->num_layers > 65535)
    return set_error(B200_ERR_UNSUPPORTED, "too many pages or layers in one copy");
  p.chunks = static_cast<int>(chunks);
  const dim3 grid(static_cast<unsigned>(num_pairs * chunks), static_cast<unsigned>(c->num_layers),
                  2);
  return cuda_status(
      launch_dependent(vec ? copy_pages_kernel<uint4> : copy_pages_kernel<uint16_t>, grid,
                       dim3(kCopyThreads), 0, stream, p),
      "copy_pages_kernel launch");
}

int launch_remap_block_tables(const void* tables, int32_t table_dtype, int64_t table_stride,
                              int64_t num_rows, int32_t table_width, const int32_t* page_map,
                              int32_t num_blocks, void* out, int64_t out_stride,
                              uint32_t* error_word, cudaStream_t stream) {
  if (table_dtype != B200_I32 && table_dtype != B200_I64)
    return set_error(B200_ERR_INVALID, "block tables must use int32 or int64");
  if (num_rows < 0 || table_width < 0 || num_blocks <= 0)
    return set_error(B200_ERR_INVALID, "table or pool size out of range");
  if (num_rows == 0 || table_width == 0) return B200_OK;
  if (!tables || !page_map || !out) return set_error(B200_ERR_INVALID, "null tensor pointer");
  if (num_rows > 1 && out_stride < table_width)
    return set_error(B200_ERR_INVALID, "rows of out must not overlap");
  RemapParams p;
  p.tables = tables;
  p.page_map = page_map;
  p.out = out;
  p.err = error_word;
  p.in_stride = table_stride;
  p.out_stride = out_stride;
  p.total = num_rows * table_width;
  p.width = table_width;
  p.num_blocks = num_blocks;
  p.table64 = table_dtype == B200_I64;
  const long long blocks = ceil_div64(p.total, kRemapThreads);
  if (blocks > 0x7fffffffLL) return set_error(B200_ERR_UNSUPPORTED, "block tables too large");
  return cuda_status(launch_dependent(remap_tables_kernel, dim3(static_cast<unsigned>(blocks)),
                                      dim3(kRemapThreads), 0, stream, p),
                     "remap_tables_kernel launch");
}

}  // namespace b200
