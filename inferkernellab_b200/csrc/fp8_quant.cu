// 16-bit values to 8-bit floating point (e4m3, largest value 448) with one
// 32-bit scale per block: a row and 128 columns (activations), or 128 x 128
// (weights).
//
//   peak  = max |x| over the block (0 if below 2^-100)
//   scale = peak / 448,   q = rn_e4m3(x * (448 * (1 / peak))),   x ~ q * scale
//
// every product and quotient rounded to 32 bits: the order of the 32-bit torch form,
// one rounding more than 448 / peak.  The peak lands within 2^-21 of 448 (up to a peak
// of 2^126 within 2^-22; above it 1 / peak is subnormal), far from the next step of
// e4m3, so nothing saturates.  A block whose
// peak is below 2^-100 is stored as zeros with scale 0: 1 / peak would leave the
// range of 32 bits.  A block with a NaN gets a NaN peak (the largest magnitude
// is taken on the bit patterns, where NaN sorts above infinity), and one with
// an infinity gets scale infinity; both come back as NaN, like the product of a
// 16-bit row that holds one.
//
// Bound: 2 bytes read and 1 written per value.  Eight lanes share a row's block
// (16 values, two 16-byte loads and one 16-byte store each), so the peak takes
// three shuffles and no shared memory.  Scales of activations are written
// block-major ([cols / 128][rows]): a CTA's 32 rows store 128 neighbouring
// bytes, and the product reads a tile's scales of one block in one run.  Measured
// (bf16): 8191 x 14336 in 57.4 us, 6.2 TB/s (0.95 of the measured copy rate); 64 x
// 4096 in 1.6 us.
#include "../../include/b200_paged_attn.h"
#include "common.cuh"
#include "fp8.cuh"
#include "fp8_quant.h"
#include "host_common.h"

namespace b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                       // lanes of a (row, block)
constexpr int kRowsPerCta = kThreads / kLanes;  // 32

struct QuantParams {
  const uint16_t* x;
  uint8_t* q;
  float* scales;
  long long rows, cols, x_stride, q_stride, s_row, s_block;
  int blocks;
};

// Largest of two packed pairs of magnitudes (sign bits cleared).
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

template <typename E>
__device__ __forceinline__ float f32_of_bits(uint32_t bits) {
  const uint16_t b = static_cast<uint16_t>(bits);
  typename E::T t;
  memcpy(&t, &b, 2);
  return to_float<E>(t);
}

// scale and 448 * (1 / peak) of a block from the bits of its largest magnitude.
template <typename E>
__device__ __forceinline__ void block_scale(uint32_t peak_bits, float* scale, float* inverse) {
  float peak = f32_of_bits<E>(peak_bits);
  if (peak < kFp8Flush) peak = 0.f;
  *scale = __fdiv_rn(peak, kFp8Max);
  *inverse = peak == 0.f ? 0.f : __fmul_rn(__frcp_rn(peak), kFp8Max);
}

// grid.x = row tile * blocks + block: neighbouring CTAs read neighbouring columns.
template <typename E>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantParams p) {
  const int lane8 = threadIdx.x % kLanes;
  const int block = blockIdx.x % p.blocks;
  const long long row =
      static_cast<long long>(blockIdx.x / p.blocks) * kRowsPerCta + threadIdx.x / kLanes;
  const long long col = block * 128LL + lane8 * 16;
  const bool live = row < p.rows && col < p.cols;  // cols % 16 == 0 here
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The product that follows may begin to load its weight: it waits for this grid
  // before it reads what this grid writes.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint4 a = {}, b = {};
  if (live) {
    const uint4* src = reinterpret_cast<const uint4*>(p.x + row * p.x_stride + col);
    a = src[0];
    b = src[1];
  }
  const uint32_t m = 0x7fff7fffu;
  uint32_t peak = max_u16x2(max_u16x2(max_u16x2(a.x & m, a.y & m), max_u16x2(a.z & m, a.w & m)),
                            max_u16x2(max_u16x2(b.x & m, b.y & m), max_u16x2(b.z & m, b.w & m)));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
    peak = max_u16x2(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  peak = max(peak & 0xffffu, peak >> 16);
  if (!live) return;
  float scale, inv;
  block_scale<E>(peak, &scale, &inv);
  const uint32_t in[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = pack_e4m3x4(f32_of_bits<E>(in[2 * i]) * inv, f32_of_bits<E>(in[2 * i] >> 16) * inv,
                         f32_of_bits<E>(in[2 * i + 1]) * inv,
                         f32_of_bits<E>(in[2 * i + 1] >> 16) * inv);
  *reinterpret_cast<uint4*>(p.q + row * p.q_stride + col) =
      make_uint4(out[0], out[1], out[2], out[3]);
  if (lane8 == 0) p.scales[row * p.s_row + block * p.s_block] = scale;
}

// Any width, stride and alignment: a warp per (row, block).
template <typename E>
__global__ void __launch_bounds__(kThreads) quantize_rows_any_kernel(const QuantParams p) {
  const int lane = threadIdx.x & 31;
  const int block = blockIdx.x % p.blocks;
  const long long row = static_cast<long long>(blockIdx.x / p.blocks) * (kThreads / 32) +
                        (threadIdx.x >> 5);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= p.rows) return;  // warp-uniform
  uint32_t bits[4], peak = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long col = block * 128LL + i * 32 + lane;
    bits[i] = col < p.cols ? p.x[row * p.x_stride + col] : 0u;
    peak = max(peak, bits[i] & 0x7fffu);
  }
  peak = __reduce_max_sync(0xffffffffu, peak);
  float scale, inv;
  block_scale<E>(peak, &scale, &inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long col = block * 128LL + i * 32 + lane;
    if (col < p.cols)
      p.q[row * p.q_stride + col] =
          static_cast<uint8_t>(pack_e4m3x4(f32_of_bits<E>(bits[i]) * inv, 0.f, 0.f, 0.f));
  }
  if (lane == 0) p.scales[row * p.s_row + block * p.s_block] = scale;
}

// One CTA per 128 x 128 block; used once per weight, when it is loaded.
template <typename E>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const QuantParams p) {
  __shared__ uint32_t red[kThreads / 32];
  const int block = blockIdx.x % p.blocks;
  const long long row0 = static_cast<long long>(blockIdx.x / p.blocks) * 128;
  const long long col = block * 128LL + threadIdx.x % 128;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t peak = 0;
  for (long long r = row0 + threadIdx.x / 128; r < min(row0 + 128, p.rows); r += kThreads / 128)
    if (col < p.cols) peak = max(peak, p.x[r * p.x_stride + col] & 0x7fffu);
  peak = __reduce_max_sync(0xffffffffu, peak);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) peak = max(peak, red[i]);
  float scale, inv;
  block_scale<E>(peak, &scale, &inv);
  for (long long r = row0 + threadIdx.x / 128; r < min(row0 + 128, p.rows); r += kThreads / 128)
    if (col < p.cols)
      p.q[r * p.q_stride + col] = static_cast<uint8_t>(
          pack_e4m3x4(f32_of_bits<E>(p.x[r * p.x_stride + col]) * inv, 0.f, 0.f, 0.f));
  if (threadIdx.x == 0) p.scales[(row0 / 128) * p.s_row + block * p.s_block] = scale;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int launch_quantize_fp8(const void* x, int64_t rows, int64_t cols, int64_t x_stride, int32_t dtype,
                        int32_t block_rows, void* q, int64_t q_stride, float* scales,
                        int64_t scale_stride_row, int64_t scale_stride_block,
                        cudaStream_t stream) {
  if (dtype != B200_F16 && dtype != B200_BF16)
    return set_error(B200_ERR_UNSUPPORTED, "dtype must be float16 or bfloat16");
  if (block_rows != 1 && block_rows != 128)
    return set_error(B200_ERR_INVALID, "a scale covers 1 row or 128 rows");
  if (rows < 0 || cols <= 0) return set_error(B200_ERR_INVALID, "rows/cols out of range");
  if (rows == 0) return B200_OK;
  if (!x || !q || !scales) return set_error(B200_ERR_INVALID, "null tensor pointer");
  QuantParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.q = static_cast<uint8_t*>(q);
  p.scales = scales;
  p.rows = rows;
  p.cols = cols;
  p.x_stride = x_stride;
  p.q_stride = q_stride;
  p.s_row = scale_stride_row;
  p.s_block = scale_stride_block;
  const long long blocks = ceil_div64(cols, 128);
  const bool vec = block_rows == 1 && cols % 16 == 0 && x_stride % 8 == 0 && q_stride % 16 == 0 &&
                   aligned16(x) && aligned16(q);
  const long long per_cta = block_rows == 128 ? 128 : (vec ? kRowsPerCta : kThreads / 32);
  const long long ctas = ceil_div64(rows, per_cta) * blocks;
  if (ctas > 0x7fffffffLL) return set_error(B200_ERR_UNSUPPORTED, "too many blocks");
  p.blocks = static_cast<int>(blocks);
  const bool bf16 = dtype == B200_BF16;
  void (*kern)(QuantParams);
  if (block_rows == 128)
    kern = bf16 ? quantize_blocks_kernel<BF16> : quantize_blocks_kernel<Half>;
  else if (vec)
    kern = bf16 ? quantize_rows_kernel<BF16> : quantize_rows_kernel<Half>;
  else
    kern = bf16 ? quantize_rows_any_kernel<BF16> : quantize_rows_any_kernel<Half>;
  return cuda_status(
      launch_dependent(kern, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, stream, p),
      "quantize_fp8 kernel launch");
}

}  // namespace b200
