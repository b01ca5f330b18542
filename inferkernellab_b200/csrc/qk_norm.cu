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
// shared memory.  Measured (32 / 8 heads of 128, bf16): 8191 tokens 39.6 us, 5.2 TB/s
// (0.79 of the measured copy rate); one token 2.1 us.
#include <algorithm>
#include <cstdint>

#include "../../include/b200_paged_attn.h"
#include "common.cuh"
#include "host_common.h"
#include "qk_norm.h"

namespace b200 {

namespace {

constexpr int kRowsAtOnce = 4;

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
  uint32_t w[4];
};

// The two values of a packed pair.
template <typename E>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<Half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<BF16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

template <typename E>
__device__ __forceinline__ void widen(const Vec8& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack2<E>(v.w[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}
template <typename E>
__device__ __forceinline__ Vec8 narrow(const float (&f)[8]) {
  Vec8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = pack2<E>(f[2 * i], f[2 * i + 1]);
  return v;
}

// Row `row` of token t: q heads, then k heads, then v heads.
template <typename T>
__device__ __forceinline__ const T* source_row(const QkNormParams& p, long long t, int row) {
  if (row < p.num_q_heads) return reinterpret_cast<const T*>(p.q) + t * p.q_st + row * p.q_sh;
  const int h = row - p.num_q_heads;
  if (h < p.num_kv_heads) return reinterpret_cast<const T*>(p.k) + t * p.k_st + h * p.k_sh;
  return reinterpret_cast<const T*>(p.v) + t * p.v_st + (h - p.num_kv_heads) * p.v_sh;
}
template <typename T>
__device__ __forceinline__ T* target_row(const QkNormParams& p, long long t, int row,
                                         long long slot) {
  if (row < p.num_q_heads) return reinterpret_cast<T*>(p.q_out) + t * p.qo_st + row * p.qo_sh;
  const int h = row - p.num_q_heads;
  const bool is_k = h < p.num_kv_heads;
  return reinterpret_cast<T*>(is_k ? p.k_cache : p.v_cache) +
         ((p.layer_slot_base + slot) * p.num_kv_heads + (is_k ? h : h - p.num_kv_heads)) *
             p.head_dim;
}

// What a lane multiplies its 8 pairs (a, b) with, apart from the row's 1 / rms:
//   lo = a * ac + b * bs,   hi = b * bc + a * as
// the weight times cos or sin (1 and 0 where nothing is rotated).
struct Factors {
  float ac[8], bs[8], bc[8], as[8];
};

template <typename E>
__device__ __forceinline__ Factors factors(const void* weight, int lo, int hi, bool rotated,
                                           const Vec8& c1, const Vec8& c2, const Vec8& s1,
                                           const Vec8& s2) {
  using T = typename E::T;
  Factors f;
  float w1[8], w2[8], c[8], s[8];
  widen<E>(*reinterpret_cast<const Vec8*>(reinterpret_cast<const T*>(weight) + lo), w1);
  widen<E>(*reinterpret_cast<const Vec8*>(reinterpret_cast<const T*>(weight) + hi), w2);
  widen<E>(c1, c);
  widen<E>(s1, s);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f.ac[j] = rotated ? w1[j] * c[j] : w1[j];
    f.bs[j] = rotated ? -w2[j] * s[j] : 0.f;
  }
  widen<E>(c2, c);
  widen<E>(s2, s);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f.bc[j] = rotated ? w2[j] * c[j] : w2[j];
    f.as[j] = rotated ? w1[j] * s[j] : 0.f;
  }
  return f;
}

// Normalises and turns one row, whose LANES lanes all call it.
template <typename E, int LANES>
__device__ __forceinline__ void norm_turn(Vec8& x1, Vec8& x2, const Factors& f, float inv_dim,
                                          float eps) {
  float a[8], b[8];
  widen<E>(x1, a);
  widen<E>(x2, b);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(a[j], a[j], fmaf(b[j], b[j], ss));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss * inv_dim + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = a[j] * inv, y = b[j] * inv;
    a[j] = fmaf(x, f.ac[j], y * f.bs[j]);
    b[j] = fmaf(y, f.bc[j], x * f.as[j]);
  }
  x1 = narrow<E>(a);
  x2 = narrow<E>(b);
}

// One CTA per token; LANES = D / 16 lanes per row, the rows of the CTA's groups of
// lanes G apart.  A lane's factors are the same for all heads of q (of k), so they
// are formed once for the ROWS q rows that it takes at a time (all of their loads
// in flight together) and once more for its k row, which it reads with the v row.
template <typename E, int LANES, int ROWS>
__global__ void __launch_bounds__(512) qk_norm_vec_kernel(const QkNormParams p) {
  using T = typename E::T;
  const long long t = blockIdx.x;
  const int part = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES, groups = blockDim.x / LANES;
  const int rot_half = p.rotary_dim / 2;
  // The 8 pairs of this lane: rotated ones first, then the dimensions past R
  // taken as pairs half of their count apart.
  const bool rotated = part * 8 < rot_half;
  const int past = part * 8 - rot_half;
  const int lo = rotated ? part * 8 : p.rotary_dim + past;
  const int hi = rotated ? lo + rot_half : lo + (p.head_dim - p.rotary_dim) / 2;
  const float inv_dim = 1.f / static_cast<float>(p.head_dim);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long slot = load_index(p.slots, t, p.slots64);
  Vec8 c1 = {}, c2 = {}, s1 = {}, s2 = {};
  if (rotated) {
    const T* c = reinterpret_cast<const T*>(p.cos) + t * p.cos_st;
    const T* s = reinterpret_cast<const T*>(p.sin) + t * p.sin_st;
    c1 = *reinterpret_cast<const Vec8*>(c + lo);
    c2 = *reinterpret_cast<const Vec8*>(c + hi);
    s1 = *reinterpret_cast<const Vec8*>(s + lo);
    s2 = *reinterpret_cast<const Vec8*>(s + hi);
  }
  // k and v rows start at the group after the last q row's, so that a CTA with a
  // group per row works on all of them at once.
  const int kv0 = (group + groups - p.num_q_heads % groups) % groups;
  Vec8 k1 = {}, k2 = {}, v1 = {}, v2 = {};
  if (kv0 < p.num_kv_heads) {
    const T* k = reinterpret_cast<const T*>(p.k) + t * p.k_st + kv0 * p.k_sh;
    const T* v = reinterpret_cast<const T*>(p.v) + t * p.v_st + kv0 * p.v_sh;
    k1 = *reinterpret_cast<const Vec8*>(k + lo);
    k2 = *reinterpret_cast<const Vec8*>(k + hi);
    v1 = *reinterpret_cast<const Vec8*>(v + lo);
    v2 = *reinterpret_cast<const Vec8*>(v + hi);
  }
  // Whole warps walk the rows together: the sums need every lane.
  const int warp_group = static_cast<int>(threadIdx.x & ~31) / LANES;
  if (warp_group < p.num_q_heads) {
    const T* q = reinterpret_cast<const T*>(p.q) + t * p.q_st;
    T* out = reinterpret_cast<T*>(p.q_out) + t * p.qo_st;
    for (int base = 0; base + warp_group < p.num_q_heads; base += groups * ROWS) {
      Vec8 x1[ROWS], x2[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int row = base + i * groups + group;
        x1[i] = x2[i] = Vec8{};
        if (row < p.num_q_heads) {
          x1[i] = *reinterpret_cast<const Vec8*>(q + row * p.q_sh + lo);
          x2[i] = *reinterpret_cast<const Vec8*>(q + row * p.q_sh + hi);
        }
      }
      const Factors f = factors<E>(p.q_weight, lo, hi, rotated, c1, c2, s1, s2);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int row = base + i * groups + group;
        norm_turn<E, LANES>(x1[i], x2[i], f, inv_dim, p.eps);
        if (row < p.num_q_heads) {
          *reinterpret_cast<Vec8*>(out + row * p.qo_sh + lo) = x1[i];
          *reinterpret_cast<Vec8*>(out + row * p.qo_sh + hi) = x2[i];
        }
      }
    }
  }
  if (slot < 0 || slot >= p.num_slots) {  // CTA-uniform: nothing to append
    if (slot >= p.num_slots && threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadSlot);
    return;
  }
  if (!__any_sync(0xffffffffu, kv0 < p.num_kv_heads)) return;
  const Factors f = factors<E>(p.k_weight, lo, hi, rotated, c1, c2, s1, s2);
  const long long at = (p.layer_slot_base + slot) * p.num_kv_heads;
  for (int h = kv0; __any_sync(0xffffffffu, h < p.num_kv_heads); h += groups) {
    const bool live = h < p.num_kv_heads;
    if (h != kv0 && live) {
      const T* k = reinterpret_cast<const T*>(p.k) + t * p.k_st + h * p.k_sh;
      const T* v = reinterpret_cast<const T*>(p.v) + t * p.v_st + h * p.v_sh;
      k1 = *reinterpret_cast<const Vec8*>(k + lo);
      k2 = *reinterpret_cast<const Vec8*>(k + hi);
      v1 = *reinterpret_cast<const Vec8*>(v + lo);
      v2 = *reinterpret_cast<const Vec8*>(v + hi);
    }
    norm_turn<E, LANES>(k1, k2, f, inv_dim, p.eps);
    if (live) {
      T* k = reinterpret_cast<T*>(p.k_cache) + (at + h) * p.head_dim;
      T* v = reinterpret_cast<T*>(p.v_cache) + (at + h) * p.head_dim;
      *reinterpret_cast<Vec8*>(k + lo) = k1;
      *reinterpret_cast<Vec8*>(k + hi) = k2;
      *reinterpret_cast<Vec8*>(v + lo) = v1;
      *reinterpret_cast<Vec8*>(v + hi) = v2;
    }
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
    const T* src = source_row<T>(p, t, row);
    T* dst = target_row<T>(p, t, row, slot);
    const int kind = row < p.num_q_heads ? 0 : row < p.num_q_heads + p.num_kv_heads ? 1 : 2;
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

// Whether tokens x heads rows of `dim` elements share memory, unless one stride's
// steps clear the extent of the other's.
bool rows_overlap(int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride,
                  int64_t dim) {
  if (tokens == 1) token_stride = INT64_MAX;
  if (heads == 1) head_stride = INT64_MAX;
  const bool heads_inside = head_stride <= token_stride;
  const int64_t inner = heads_inside ? head_stride : token_stride;
  const int64_t outer = heads_inside ? token_stride : head_stride;
  const int64_t count = heads_inside ? heads : tokens;
  return inner < dim || (outer != INT64_MAX && outer < inner * (count - 1) + dim);
}

template <typename E, int ROWS>
void (*vec_kernel(int lanes))(QkNormParams) {
  switch (lanes) {
    case 1: return qk_norm_vec_kernel<E, 1, ROWS>;
    case 2: return qk_norm_vec_kernel<E, 2, ROWS>;
    case 4: return qk_norm_vec_kernel<E, 4, ROWS>;
    case 8: return qk_norm_vec_kernel<E, 8, ROWS>;
    default: return qk_norm_vec_kernel<E, 16, ROWS>;
  }
}

template <typename E>
cudaError_t launch(const QkNormParams& p, long long tokens, bool vec, int sms,
                   cudaStream_t stream) {
  const int lanes = vec ? p.head_dim / 16 : 32;
  // More than a token per SM: ROWS q rows per thread, for the bytes in flight and
  // the factors formed once (4000 tokens: 21.6 us against 63; 160: 3.4 against 3.8).
  // Fewer: a group of lanes per row, for the shortest way through (148 tokens: 2.4 us
  // against 3.4; 8: 2.1 against 3.0).
  const bool many = vec && tokens > sms;
  const long long groups = many  ? ceil_div64(p.num_q_heads, kRowsAtOnce)
                           : vec ? p.num_q_heads + p.num_kv_heads
                                 : p.num_q_heads + 2LL * p.num_kv_heads;
  const dim3 block(static_cast<unsigned>(
      std::min<long long>(vec ? 512 : 1024, (groups * lanes + 31) / 32 * 32)));
  const dim3 grid(static_cast<unsigned>(tokens));
  void (*kern)(QkNormParams) = !vec ? qk_norm_any_kernel<E>
                               : many   ? vec_kernel<E, kRowsAtOnce>(lanes)
                                      : vec_kernel<E, 1>(lanes);
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
  if (rows_overlap(a->num_tokens, a->q_out_stride_token, a->num_q_heads, a->q_out_stride_head,
                   c->head_dim))
    return set_error(B200_ERR_INVALID, "rows of query_out must not overlap");
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
  DeviceInfo info;
  const int rc = current_device_info(&info);
  if (rc != B200_OK) return rc;
  return cuda_status(c->dtype == B200_BF16
                         ? launch<BF16>(p, a->num_tokens, vec, info.num_sms, stream)
                         : launch<Half>(p, a->num_tokens, vec, info.num_sms, stream),
                     "qk_norm kernel launch");
}

}  // namespace b200
