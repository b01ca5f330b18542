// Per-head RMS norm of q and k, rotary embedding and KV append in one launch.
//
// For every token t and head h, with the rotary dimension R <= head_dim D:
//   n(x, w)[i] = x[i] * rsqrt(mean(x^2) + eps) * w[i]
//   q_out[t, h]                = turn(n(q[t, h], q_weight), cos[t], sin[t])
//   cache.K[layer, slot[t], h] = turn(n(k[t, h], k_weight), cos[t], sin[t])
//   cache.V[layer, slot[t], h] = v[t, h]
// where turn() rotates the first R dimensions, turn(y)[i] = y[i] * cos[i] +
// rotate_half(y)[i] * sin[i], rotate_half(y) = concat(-y[R/2:R], y[:R/2]), and
// leaves the other D - R as they are.  All arithmetic is in 32 bits with one
// rounding to the 16-bit type at the end: unlike rope_append_kv, which repeats
// the roundings of a chain of 16-bit torch operations bit for bit, there is no
// such chain to match here, and each extra rounding would cost up to half a
// unit in the last place.
//
// Bound: each of q, k, v is read once and written once, so DRAM bytes at a
// prefill batch and the launch at a decode step.  A row (one head of one token)
// belongs to D / 16 neighbouring lanes, each with the 8 pairs it rotates in two
// 16-byte vectors, so the sum of squares takes log2(D / 16) shuffles and no
// shared memory.
#include <algorithm>

#include "../../include/b200_paged_attn.h"
#include "common.cuh"
#include "host_common.h"
#include "qk_norm.h"

namespace b200 {

namespace {

struct QkNormParams {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* q_weight;
  const uint8_t* k_weight;
  const uint8_t* cos;
  const uint8_t* sin;
  uint8_t* q_out;
  uint8_t* k_cache;
  uint8_t* v_cache;
  const void* slots;
  uint32_t* err;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, cos_st, sin_st;  // elements
  long long num_slots, layer_slot_base;
  float eps;
  int num_q_heads, num_kv_heads, head_dim, rotary_dim, slots64;
};

// 8 x 16-bit elements = one 16-byte access.
struct alignas(16) Vec8 {
  uint16_t h[8];
};

template <typename E>
__device__ __forceinline__ float lane_f(const Vec8& v, int i) {
  typename E::T t;
  memcpy(&t, &v.h[i], 2);
  return to_float<E>(t);
}

template <typename E>
__device__ __forceinline__ void lane_set(Vec8& v, int i, float x) {
  typename E::T t = from_float<E>(x);
  memcpy(&v.h[i], &t, 2);
}

// Source and destination of row `row` of token t: q heads, then k heads, then v
// heads.  kind 0: q, 1: k, 2: v.
template <typename T>
__device__ __forceinline__ int row_pointers(const QkNormParams& p, long long t, int row,
                                            long long slot, const T** src, T** dst) {
  const int kv = p.num_kv_heads;
  if (row < p.num_q_heads) {
    *src = reinterpret_cast<const T*>(p.q) + t * p.q_st + row * p.q_sh;
    *dst = reinterpret_cast<T*>(p.q_out) + t * p.qo_st + row * p.qo_sh;
    return 0;
  }
  const bool is_k = row < p.num_q_heads + kv;
  const int h = row - p.num_q_heads - (is_k ? 0 : kv);
  *src = is_k ? reinterpret_cast<const T*>(p.k) + t * p.k_st + h * p.k_sh
              : reinterpret_cast<const T*>(p.v) + t * p.v_st + h * p.v_sh;
  *dst = reinterpret_cast<T*>(is_k ? p.k_cache : p.v_cache) +
         ((p.layer_slot_base + slot) * kv + h) * p.head_dim;
  return is_k ? 1 : 2;
}

// One CTA per token; LANES = D / 16 lanes per row, blockDim a multiple of 32.
template <typename E, int LANES>
__global__ void __launch_bounds__(512) qk_norm_vec_kernel(const QkNormParams p) {
  using T = typename E::T;
  const long long t = blockIdx.x;
  const int rows = p.num_q_heads + 2 * p.num_kv_heads;
  const int part = threadIdx.x % LANES;
  const int rot_half = p.rotary_dim / 2;
  // The 8 pairs of this lane: rotated ones first, then the dimensions past R
  // taken as pairs half of their count apart.
  const bool rotated = part * 8 < rot_half;
  const int past = part * 8 - rot_half;
  const int lo = rotated ? part * 8 : p.rotary_dim + past;
  const int hi = rotated ? lo + rot_half : lo + (p.head_dim - p.rotary_dim) / 2;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Vec8 c1, c2, s1, s2;
  if (rotated) {
    const T* c = reinterpret_cast<const T*>(p.cos) + t * p.cos_st;
    const T* s = reinterpret_cast<const T*>(p.sin) + t * p.sin_st;
    c1 = *reinterpret_cast<const Vec8*>(c + lo);
    c2 = *reinterpret_cast<const Vec8*>(c + hi);
    s1 = *reinterpret_cast<const Vec8*>(s + lo);
    s2 = *reinterpret_cast<const Vec8*>(s + hi);
  }
  const long long slot = load_index(p.slots, t, p.slots64);
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  if (slot >= p.num_slots && threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadSlot);
  const int per_pass = blockDim.x / LANES;
  const int lane_row = threadIdx.x / LANES;
  // Whole warps walk the rows together: the shuffles below need every lane.
  for (int base = 0; base < rows; base += per_pass) {
    if (base + (threadIdx.x & ~31) / LANES >= rows) break;  // warp-uniform
    const int row = base + lane_row;
    const bool live = row < rows && (row < p.num_q_heads || slot_ok);
    const T* src = nullptr;
    T* dst = nullptr;
    int kind = 2;
    Vec8 x1 = {}, x2 = {};
    if (live) {
      kind = row_pointers<T>(p, t, row, slot, &src, &dst);
      x1 = *reinterpret_cast<const Vec8*>(src + lo);
      x2 = *reinterpret_cast<const Vec8*>(src + hi);
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = lane_f<E>(x1, j), b = lane_f<E>(x2, j);
      ss = fmaf(a, a, fmaf(b, b, ss));
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live) continue;
    if (kind != 2) {
      const float inv = rsqrtf(ss / static_cast<float>(p.head_dim) + p.eps);
      const T* w = reinterpret_cast<const T*>(kind == 0 ? p.q_weight : p.k_weight);
      const Vec8 w1 = *reinterpret_cast<const Vec8*>(w + lo);
      const Vec8 w2 = *reinterpret_cast<const Vec8*>(w + hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = lane_f<E>(x1, j) * inv * lane_f<E>(w1, j);
        const float b = lane_f<E>(x2, j) * inv * lane_f<E>(w2, j);
        lane_set<E>(x1, j, rotated ? a * lane_f<E>(c1, j) - b * lane_f<E>(s1, j) : a);
        lane_set<E>(x2, j, rotated ? b * lane_f<E>(c2, j) + a * lane_f<E>(s2, j) : b);
      }
    }
    *reinterpret_cast<Vec8*>(dst + lo) = x1;
    *reinterpret_cast<Vec8*>(dst + hi) = x2;
  }
}

// Any head_dim, stride and alignment: a warp per row, one element at a time.
template <typename E>
__global__ void __launch_bounds__(1024) qk_norm_any_kernel(const QkNormParams p) {
  using T = typename E::T;
  const long long t = blockIdx.x;
  const int rows = p.num_q_heads + 2 * p.num_kv_heads;
  const int lane = threadIdx.x & 31;
  const int half = p.rotary_dim / 2;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const T* c = reinterpret_cast<const T*>(p.cos) + t * p.cos_st;
  const T* s = reinterpret_cast<const T*>(p.sin) + t * p.sin_st;
  const long long slot = load_index(p.slots, t, p.slots64);
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  if (slot >= p.num_slots && threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadSlot);
  for (int row = threadIdx.x >> 5; row < rows; row += blockDim.x >> 5) {
    if (row >= p.num_q_heads && !slot_ok) continue;
    const T* src;
    T* dst;
    const int kind = row_pointers<T>(p, t, row, slot, &src, &dst);
    if (kind == 2) {
      for (int i = lane; i < p.head_dim; i += 32) dst[i] = src[i];
      continue;
    }
    float ss = 0.f;
    for (int i = lane; i < p.head_dim; i += 32) {
      const float a = to_float<E>(src[i]);
      ss = fmaf(a, a, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / static_cast<float>(p.head_dim) + p.eps);
    const T* w = reinterpret_cast<const T*>(kind == 0 ? p.q_weight : p.k_weight);
    for (int i = lane; i < half; i += 32) {
      const float a = to_float<E>(src[i]) * inv * to_float<E>(w[i]);
      const float b = to_float<E>(src[i + half]) * inv * to_float<E>(w[i + half]);
      dst[i] = from_float<E>(a * to_float<E>(c[i]) - b * to_float<E>(s[i]));
      dst[i + half] = from_float<E>(b * to_float<E>(c[i + half]) + a * to_float<E>(s[i + half]));
    }
    for (int i = p.rotary_dim + lane; i < p.head_dim; i += 32)
      dst[i] = from_float<E>(to_float<E>(src[i]) * inv * to_float<E>(w[i]));
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename E>
cudaError_t launch(const QkNormParams& p, long long tokens, bool vec, cudaStream_t stream) {
  const long long rows = p.num_q_heads + 2LL * p.num_kv_heads;
  const int lanes = vec ? p.head_dim / 16 : 32;
  // Every row of a token at once where the threads allow.
  const dim3 block(static_cast<unsigned>(std::min<long long>(vec ? 512 : 1024, (rows * lanes + 31) / 32 * 32)));
  const dim3 grid(static_cast<unsigned>(tokens));
  void (*kern)(QkNormParams) = qk_norm_any_kernel<E>;
  if (vec) {
    switch (lanes) {
      case 1: kern = qk_norm_vec_kernel<E, 1>; break;
      case 2: kern = qk_norm_vec_kernel<E, 2>; break;
      case 4: kern = qk_norm_vec_kernel<E, 4>; break;
      case 8: kern = qk_norm_vec_kernel<E, 8>; break;
      default: kern = qk_norm_vec_kernel<E, 16>; break;
    }
  }
  return launch_dependent(kern, grid, block, 0, stream, p);
}

}  // namespace

int launch_qk_norm_rope_append(const b200_cache_desc* c, const b200_qk_norm_args* a,
                               const void* query, const void* key, const void* value,
                               const void* q_weight, const void* k_weight, const void* cos,
                               const void* sin, const void* slots, void* query_out,
                               uint32_t* error_word, cudaStream_t stream) {
  if (c == nullptr || a == nullptr) return set_error(B200_ERR_INVALID, "null descriptor");
  if (c->num_layers <= 0 || c->num_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 ||
      c->head_dim <= 0)
    return set_error(B200_ERR_INVALID, "cache dimensions must be positive");
  if (c->dtype != B200_F16 && c->dtype != B200_BF16)
    return set_error(B200_ERR_UNSUPPORTED, "cache dtype must be float16 or bfloat16");
  if (a->layer < 0 || a->layer >= c->num_layers)
    return set_error(B200_ERR_LAYER, "layer is out of range");
  if (a->num_q_heads <= 0 || a->num_q_heads % c->num_kv_heads != 0)
    return set_error(B200_ERR_INVALID, "num_heads must be divisible by num_kv_heads");
  if (a->rotary_dim <= 0 || a->rotary_dim > c->head_dim || a->rotary_dim % 2 != 0)
    return set_error(B200_ERR_INVALID, "rotary_dim must be even and at most head_dim");
  if (!(a->eps >= 0.f)) return set_error(B200_ERR_INVALID, "eps must be non-negative");
  if (a->num_tokens < 0) return set_error(B200_ERR_INVALID, "num_tokens must be non-negative");
  if (a->num_tokens == 0) return B200_OK;
  if (a->num_tokens > 0x7fffffffLL)
    return set_error(B200_ERR_UNSUPPORTED, "limited to 2^31 - 1 tokens");
  if (a->num_q_heads + 2LL * c->num_kv_heads > 0xffffff)
    return set_error(B200_ERR_UNSUPPORTED, "too many heads per token");
  if (!query || !key || !value || !q_weight || !k_weight || !cos || !sin || !slots ||
      !query_out || !c->k_cache || !c->v_cache)
    return set_error(B200_ERR_INVALID, "null tensor pointer");
  QkNormParams p;
  p.q = static_cast<const uint8_t*>(query);
  p.k = static_cast<const uint8_t*>(key);
  p.v = static_cast<const uint8_t*>(value);
  p.q_weight = static_cast<const uint8_t*>(q_weight);
  p.k_weight = static_cast<const uint8_t*>(k_weight);
  p.cos = static_cast<const uint8_t*>(cos);
  p.sin = static_cast<const uint8_t*>(sin);
  p.q_out = static_cast<uint8_t*>(query_out);
  p.k_cache = static_cast<uint8_t*>(c->k_cache);
  p.v_cache = static_cast<uint8_t*>(c->v_cache);
  p.slots = slots;
  p.err = error_word;
  p.q_st = a->q_stride_token;
  p.q_sh = a->q_stride_head;
  p.k_st = a->k_stride_token;
  p.k_sh = a->k_stride_head;
  p.v_st = a->v_stride_token;
  p.v_sh = a->v_stride_head;
  p.qo_st = a->q_out_stride_token;
  p.qo_sh = a->q_out_stride_head;
  p.cos_st = a->cos_stride_token;
  p.sin_st = a->sin_stride_token;
  p.num_slots = static_cast<long long>(c->num_blocks) * c->block_size;
  p.layer_slot_base = static_cast<long long>(a->layer) * p.num_slots;
  p.eps = a->eps;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = c->num_kv_heads;
  p.head_dim = c->head_dim;
  p.rotary_dim = a->rotary_dim;
  p.slots64 = a->slots_dtype == B200_I64;
  // 16-byte vectors: D / 16 lanes per row (a power of two up to 16), the pairs of
  // both regions in whole vectors, and every row start 16-byte aligned.
  const int d = c->head_dim;
  const bool vec = (d == 16 || d == 32 || d == 64 || d == 128 || d == 256) &&
                   a->rotary_dim % 16 == 0 && p.q_st % 8 == 0 && p.q_sh % 8 == 0 &&
                   p.k_st % 8 == 0 && p.k_sh % 8 == 0 && p.v_st % 8 == 0 && p.v_sh % 8 == 0 &&
                   p.qo_st % 8 == 0 && p.qo_sh % 8 == 0 && p.cos_st % 8 == 0 &&
                   p.sin_st % 8 == 0 && aligned16(query) && aligned16(key) && aligned16(value) &&
                   aligned16(q_weight) && aligned16(k_weight) && aligned16(cos) &&
                   aligned16(sin) && aligned16(query_out) && aligned16(c->k_cache) &&
                   aligned16(c->v_cache);
  return cuda_status(c->dtype == B200_BF16 ? launch<BF16>(p, a->num_tokens, vec, stream)
                                           : launch<Half>(p, a->num_tokens, vec, stream),
                     "qk_norm kernel launch");
}

}  // namespace b200
