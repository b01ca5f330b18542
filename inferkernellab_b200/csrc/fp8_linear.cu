// Product of 8-bit activations and an 8-bit weight with block scales on the
// 5th-generation tensor cores (tcgen05 + TMEM, TMA), sm_100a.
//
//   out[m, n] = rnd( sum_b sx[m, b] * sw[n / 128, b] * sum_{k in b} x[m, k] w[n, k] + bias[n] )
//
// b runs over blocks of 128 columns of K; x, w are e4m3, the scales and all sums
// 32-bit, with one rounding to the 16-bit output at the end.
//
// The scales differ per row and block, so a block's product cannot simply be
// accumulated by the tensor core: one block is one accumulator (4 MMAs of K = 32
// on a 128-byte swizzled row), which the epilogue warps read from TMEM, scale and
// add to sums in registers while the tensor core fills the next buffer.
//
// Orientation: the weight's rows are M of the MMA (128 per tile) and the tokens
// are N (kTokens per tile, 16 to 256), for a decode step's few tokens as for a
// prefill.  A thread then owns one weight row and adds, per token,
// product * (sx * sw); the scale products of a block sit in shared memory, where
// all 32 lanes read the same four at once.
//
//   warps 0..kEpi-1    epilogue: warp i reads lanes 32 (i % 4) .., the columns are
//                      split over kEpi / 4 groups
//   warp kEpi          TMA producer: weight and token tile of a block per stage
//   warp kEpi + 1      MMA issuer (one thread)
//   warp kEpi + 2      scale products of the blocks ahead
//
// Work: tiles of 128 weight rows x kTokens tokens, tokens innermost so that
// neighbouring CTAs share weight rows in L2.  CTAs are persistent.  Where tiles
// are fewer than SMs, a cluster of CTAs splits K and joins its sums through
// distributed shared memory in rank order (the result does not depend on timing).
//
// Every mbarrier wait is bounded (1 s); on a timeout the CTA raises its abort
// flag, records the error bit, waits (bounded) for its own copies and MMAs and
// frees its TMEM.
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/b200_paged_attn.h"
#include "attn_core.cuh"
#include "common.cuh"
#include "fp8_linear.h"
#include "host_common.h"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

typedef unsigned long long u64;

constexpr int kRows = 128;    // weight rows of a tile = MMA M
constexpr int kBlock = 128;   // K per scale block = bytes of a swizzled row
constexpr int kScaleRing = 8;
constexpr int kMaxSplits = 8;

template <int TOKENS>
struct Shape {
  static constexpr int kEpi = TOKENS > 128 ? 8 : 4;  // epilogue warps
  static constexpr int kThreads = (kEpi + 4) * 32;
  static constexpr int kCols = TOKENS / (kEpi / 4);  // token columns of an epilogue thread
  static constexpr int kStep = kCols < 32 ? kCols : 32;  // columns of one TMEM load
  // 256 tokens: 128 sums and 64 loaded values per epilogue thread are more than the
  // 168 registers of 384 threads, so that the other four warps give some of theirs.
  static constexpr bool kSplitRegisters = TOKENS > 128;
  static constexpr int kEpiRegisters = 224, kOtherRegisters = 56, kLaunchRegisters = 168;
  static_assert(kEpi * kEpiRegisters + 4 * kOtherRegisters <= (kEpi + 4) * kLaunchRegisters ||
                    !kSplitRegisters,
                "what the epilogue takes is what the other warps give");
  static constexpr int kStageBytes = kRows * kBlock + TOKENS * kBlock;
  // Up to 64 tokens a CTA takes under half an SM, so that two share it: the
  // product is then bound by the weight's bytes, and 296 CTAs spread them
  // better than 148.
  static constexpr int kCtasPerSm = TOKENS <= 64 ? 2 : 1;
  static constexpr int kStages = TOKENS <= 32 ? 5 : TOKENS <= 64 ? 4 : TOKENS <= 128 ? 6 : 4;
  static constexpr int kBuffers = TOKENS > 128 ? 2 : 4;  // accumulators
  static constexpr int kBufferCols = TOKENS < 32 ? 32 : TOKENS;
  static constexpr int kTmemCols = kBuffers * kBufferCols;
  static constexpr int kScaleBytes = kScaleRing * TOKENS * 4;
  static constexpr int kBars = 2 * kStages + 2 * kBuffers + 2 * kScaleRing + 1;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleBytes + kBars * 8 + 16;
  static_assert(kTmemCols <= 512 / kCtasPerSm, "TMEM columns");
  static_assert(kRows * TOKENS * 4 <= kStages * kStageBytes || TOKENS > 128,
                "the split sums reuse the stages");
  static_assert(kSmem <= 227 * 1024 / kCtasPerSm - 1024, "shared memory");
};

struct LinearParams {
  const float* x_scales;
  const float* w_scales;
  const void* bias;
  void* out;
  uint32_t* err;
  long long m, n;
  long long xs_row, xs_block, ws_row, ws_block, out_stride;
  int blocks;         // of K
  int token_tiles;
  long long tiles;
  int splits;
};

// d += a * b on two packed 32-bit values.
__device__ __forceinline__ void fma2(u64& d, u64 a, u64 b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ u64 pack_f32x2(uint32_t lo, uint32_t hi) {
  u64 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ float2 unpack_f32x2(u64 v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}

__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&v)[32]) {
  tc::ld32(taddr, v);
}
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&v)[16]) {
  tc::ld16(taddr, v);
}

template <typename E, int TOKENS>
__global__ void __launch_bounds__(Shape<TOKENS>::kThreads, Shape<TOKENS>::kCtasPerSm)
    fp8_linear_kernel(const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ CUtensorMap xmap, const LinearParams p) {
  using S = Shape<TOKENS>;
  using T = typename E::T;
  constexpr int kStages = S::kStages, kBuffers = S::kBuffers;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* stages = smem;
  float* scales = reinterpret_cast<float*>(smem + kStages * S::kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes + S::kScaleBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + kBuffers;
  uint64_t* sc_full = acc_empty + kBuffers;
  uint64_t* sc_empty = sc_full + kScaleRing;
  uint64_t* mma_idle = sc_empty + kScaleRing;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(mma_idle + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_idle + 1) + 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const long long tile0 = blockIdx.x / p.splits;
  const long long tile_step = gridDim.x / p.splits;
  const int kb0 = static_cast<int>(static_cast<long long>(p.blocks) * rank / p.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(p.blocks) * (rank + 1) / p.splits);

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], S::kEpi);
    }
    for (int i = 0; i < kScaleRing; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&sc_empty[i], S::kEpi);
    }
    mbar_init(mma_idle, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == S::kEpi + 1) {
    tc::tmem_alloc(tmem_slot, S::kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  bool ok = true;
  const int row = (warp & 3) * 32 + lane;  // of the tile; TMEM lane
  const int col0 = (warp >> 2) * S::kCols;
  if (warp >= S::kEpi) {
    if (S::kSplitRegisters)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegisters));
    if (warp == S::kEpi) {
      // ------------------------------ producer ------------------------------
      if (lane == 0) {
        tma_prefetch_desc(&wmap);
        tma_prefetch_desc(&xmap);
        int it = 0;
        for (long long tile = tile0; tile < p.tiles && ok; tile += tile_step) {
          const int n0 = static_cast<int>(tile / p.token_tiles) * kRows;
          const int m0 = static_cast<int>(tile % p.token_tiles) * TOKENS;
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % kStages;
            ok = mbar_wait_bounded(&empty[s], ((it / kStages) & 1) ^ 1, abort_flag, p.err,
                                   kErrWaitEmpty);
            if (!ok) break;
            uint8_t* dst = stages + s * S::kStageBytes;
            mbar_arrive_expect_tx(&full[s], S::kStageBytes);
            tma_load_2d(dst, &wmap, &full[s], kb * kBlock, n0);
            tma_load_2d(dst + kRows * kBlock, &xmap, &full[s], kb * kBlock, m0);
          }
        }
        drain_stages<kStages>(full, it, p.err);
      }
    } else if (warp == S::kEpi + 1) {
      // ------------------------------ MMA issuer ----------------------------
      if (lane == 0) {
        const uint32_t idesc = tc::idesc_e4m3(kRows, TOKENS);
        const uint32_t st0 = smem_u32(stages);
        int it = 0;
        for (long long tile = tile0; tile < p.tiles && ok; tile += tile_step) {
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % kStages, b = it % kBuffers;
            ok = mbar_wait_bounded(&acc_empty[b], ((it / kBuffers) & 1) ^ 1, abort_flag, p.err,
                                   kErrWaitEmpty) &&
                 mbar_wait_bounded(&full[s], (it / kStages) & 1, abort_flag, p.err, kErrWaitFull);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t w = st0 + s * S::kStageBytes;
            const uint32_t x = w + kRows * kBlock;
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
              tc::mma_e4m3(tmem + b * S::kBufferCols, tc::sdesc_sw128(w + k * 32, 16, 1024),
                           tc::sdesc_sw128(x + k * 32, 16, 1024), idesc, k > 0);
            tc::commit(&empty[s]);
            tc::commit(&acc_full[b]);
          }
        }
        // Every MMA this thread issued has finished before TMEM can be freed.
        tc::commit(mma_idle);
        mbar_wait_bounded(mma_idle, 0, abort_flag, p.err, kErrDrain);
      }
    } else if (warp == S::kEpi + 2) {
      // ---------------------------- scale products --------------------------
      // kAhead blocks at a time, so that their loads are in flight together.
      constexpr int kAhead = TOKENS > 128 ? 2 : 4;
      constexpr int kPer = (TOKENS + 31) / 32;
      int it = 0;
      for (long long tile = tile0; tile < p.tiles && ok; tile += tile_step) {
        const long long m0 = tile % p.token_tiles * TOKENS;
        const float* sw = p.w_scales + tile / p.token_tiles * p.ws_row;
        for (int kb = kb0; kb < kb1 && ok; kb += kAhead) {
          float v[kAhead][kPer];
#pragma unroll
          for (int a = 0; a < kAhead; ++a) {
            if (kb + a >= kb1) break;
            const float ws = sw[(kb + a) * p.ws_block];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              const long long m = m0 + i * 32 + lane;
              v[a][i] = m < p.m && i * 32 + lane < TOKENS
                            ? p.x_scales[m * p.xs_row + (kb + a) * p.xs_block] * ws
                            : 0.f;
            }
          }
#pragma unroll
          for (int a = 0; a < kAhead; ++a) {
            if (kb + a >= kb1) break;
            const int r = it % kScaleRing;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sc_empty[r], ((it / kScaleRing) & 1) ^ 1,
                                                           abort_flag, p.err, kErrWaitEmpty));
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
              if (i * 32 + lane < TOKENS) scales[r * TOKENS + i * 32 + lane] = v[a][i];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[r]);
            ++it;
          }
        }
      }
    }
  } else {
    // ------------------------------ epilogue ------------------------------
    if (S::kSplitRegisters)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kEpiRegisters));
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + col0;
    int it = 0;
    for (long long tile = tile0; tile < p.tiles && ok; tile += tile_step) {
      u64 acc[S::kCols / 2];
#pragma unroll
      for (int i = 0; i < S::kCols / 2; ++i) acc[i] = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int b = it % kBuffers, r = it % kScaleRing;
        ok = __all_sync(
            0xffffffffu,
            mbar_wait_bounded(&sc_full[r], (it / kScaleRing) & 1, abort_flag, p.err,
                              kErrWaitFull) &&
                mbar_wait_bounded(&acc_full[b], (it / kBuffers) & 1, abort_flag, p.err,
                                  kErrWaitFull));
        if (!ok) break;
        tc::fence_after_sync();
        const ulonglong2* sc =
            reinterpret_cast<const ulonglong2*>(scales + r * TOKENS + col0);
        // The next columns are on their way while these are added.
        constexpr int kStep = S::kStep, kSteps = S::kCols / kStep;
        uint32_t v[2][kStep];
        const uint32_t base = lane_base + b * S::kBufferCols;
        load_columns(base, v[0]);
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          tc::wait_ld(v[c & 1]);
          if (c + 1 < kSteps) {
            load_columns(base + (c + 1) * kStep, v[(c + 1) & 1]);
          } else {  // the buffer has been read
            tc::fence_before_sync();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
          }
#pragma unroll
          for (int i = 0; i < kStep / 4; ++i) {
            const ulonglong2 s2 = sc[c * (kStep / 4) + i];
            const int a = (c * kStep) / 2 + 2 * i;
            fma2(acc[a], pack_f32x2(v[c & 1][4 * i], v[c & 1][4 * i + 1]), s2.x);
            fma2(acc[a + 1], pack_f32x2(v[c & 1][4 * i + 2], v[c & 1][4 * i + 3]), s2.y);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_empty[r]);
      }
      if (!ok) break;
      const long long n = tile / p.token_tiles * kRows + row;
      const long long m0 = tile % p.token_tiles * TOKENS + col0;
      if (p.splits == 1) {
        if (n < p.n) {
          const float bias = p.bias ? to_float<E>(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
          T* out = reinterpret_cast<T*>(p.out) + m0 * p.out_stride + n;
#pragma unroll
          for (int i = 0; i < S::kCols / 2; ++i) {
            const float2 f = unpack_f32x2(acc[i]);
            if (m0 + 2 * i < p.m) out[2 * i * p.out_stride] = from_float<E>(f.x + bias);
            if (m0 + 2 * i + 1 < p.m) out[(2 * i + 1) * p.out_stride] = from_float<E>(f.y + bias);
          }
        }
      } else if (TOKENS <= 128) {
        // One tile per CTA: its stages are free, every copy and MMA has finished.
        float* part = reinterpret_cast<float*>(stages);
#pragma unroll
        for (int i = 0; i < S::kCols / 2; ++i) {
          const float2 f = unpack_f32x2(acc[i]);
          part[(col0 + 2 * i) * kRows + row] = f.x;
          part[(col0 + 2 * i + 1) * kRows + row] = f.y;
        }
      }
    }
  }
  __syncwarp();  // single-thread roles rejoin their warp
  if (p.splits > 1) {
    // Join: rank r adds the columns [TOKENS r / splits, ...) of all ranks, in rank order.
    cluster.sync();
    if (warp < S::kEpi && ok) {
      const long long n = tile0 / p.token_tiles * kRows + row;
      const long long m0 = tile0 % p.token_tiles * TOKENS;
      const int c1 = static_cast<int>(min(static_cast<long long>(TOKENS * (rank + 1) / p.splits),
                                          p.m - m0));
      float* part = reinterpret_cast<float*>(stages);
      if (n < p.n) {
        const float bias = p.bias ? to_float<E>(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
        for (int c = TOKENS * rank / p.splits; c < c1; ++c) {
          float sum = 0.f;
          for (int o = 0; o < p.splits; ++o)
            sum += *cluster.map_shared_rank(part + c * kRows + row, o);
          reinterpret_cast<T*>(p.out)[(m0 + c) * p.out_stride + n] = from_float<E>(sum + bias);
        }
      }
    }
    cluster.sync();  // no CTA leaves while another may still read its sums
  }
  // ---- teardown: every TMEM access is done, the MMA warp frees TMEM ----
  tc::fence_before_sync();
  __syncthreads();
  if (warp == S::kEpi + 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <typename E, int TOKENS>
int launch(const CUtensorMap& wmap, const CUtensorMap& xmap, const LinearParams& p, int ctas,
           cudaStream_t stream) {
  using S = Shape<TOKENS>;
  auto kern = fp8_linear_kernel<E, TOKENS>;
  const cudaError_t err =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (err != cudaSuccess) return cuda_status(err, "fp8_linear_kernel shared memory");
  if (S::kSplitRegisters) {
    // Taking registers that the launch did not reserve would wait for good.
    cudaFuncAttributes fa;
    const cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return cuda_status(e, "fp8_linear_kernel attributes");
    if (fa.numRegs != S::kLaunchRegisters)
      return set_error(B200_ERR_UNSUPPORTED, "fp8_linear_kernel was not built for 168 registers");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, wmap, xmap, p), "fp8_linear_kernel launch");
}

template <int TOKENS>
int launch_any(const b200_fp8_linear_args* a, const void* x, const void* w, LinearParams p,
               int sms, cudaStream_t stream) {
  const int slots = sms * Shape<TOKENS>::kCtasPerSm;
  p.token_tiles = static_cast<int>(ceil_div64(a->m, TOKENS));
  p.tiles = ceil_div64(a->n, kRows) * p.token_tiles;
  // Splits of K that still fit the CTAs at once, each with two blocks or more.
  p.splits = 1;
  if (TOKENS <= 128)
    p.splits = static_cast<int>(std::max<long long>(
        1, std::min<long long>({kMaxSplits, slots / p.tiles, p.blocks / 2})));
  const long long ctas = p.splits > 1 ? p.tiles * p.splits : std::min<long long>(p.tiles, slots);
  const uint64_t wdims[2] = {static_cast<uint64_t>(a->k), static_cast<uint64_t>(a->n)};
  const uint64_t xdims[2] = {static_cast<uint64_t>(a->k), static_cast<uint64_t>(a->m)};
  const uint64_t wstride[1] = {static_cast<uint64_t>(a->w_stride)};
  const uint64_t xstride[1] = {static_cast<uint64_t>(a->x_stride)};
  const uint32_t wbox[2] = {kBlock, kRows};
  const uint32_t xbox[2] = {kBlock, TOKENS};
  CUtensorMap wmap, xmap;
  int rc = encode_tensor_map_8b(w, 2, wdims, wstride, wbox, &wmap);
  if (rc == B200_OK) rc = encode_tensor_map_8b(x, 2, xdims, xstride, xbox, &xmap);
  if (rc != B200_OK) return rc;
  return a->dtype == B200_BF16
             ? launch<BF16, TOKENS>(wmap, xmap, p, static_cast<int>(ctas), stream)
             : launch<Half, TOKENS>(wmap, xmap, p, static_cast<int>(ctas), stream);
}

}  // namespace

int launch_fp8_linear(const b200_fp8_linear_args* a, const void* x, const float* x_scales,
                      const void* w, const float* w_scales, const void* bias, void* out,
                      uint32_t* error_word, cudaStream_t stream) {
  if (a == nullptr) return set_error(B200_ERR_INVALID, "null descriptor");
  if (a->dtype != B200_F16 && a->dtype != B200_BF16)
    return set_error(B200_ERR_UNSUPPORTED, "the output must be float16 or bfloat16");
  if (a->m < 0 || a->n <= 0 || a->k <= 0)
    return set_error(B200_ERR_INVALID, "rows/outputs/columns out of range");
  if (a->m > 0x7fffff00LL || a->n > 0x7fffff00LL || a->k > 0x7fffff00LL)
    return set_error(B200_ERR_UNSUPPORTED, "sizes are limited to 2^31 - 256");
  if (a->x_stride % 16 != 0 || a->w_stride % 16 != 0)
    return set_error(B200_ERR_INVALID, "rows of x and weight must start on 16-byte boundaries");
  if (a->m == 0) return B200_OK;
  if (!x || !x_scales || !w || !w_scales || !out)
    return set_error(B200_ERR_INVALID, "null tensor pointer");
  DeviceInfo info;
  const int rc = current_device_info(&info);
  if (rc != B200_OK) return rc;
  LinearParams p;
  p.x_scales = x_scales;
  p.w_scales = w_scales;
  p.bias = bias;
  p.out = out;
  p.err = error_word;
  p.m = a->m;
  p.n = a->n;
  p.xs_row = a->x_scale_stride_row;
  p.xs_block = a->x_scale_stride_block;
  p.ws_row = a->w_scale_stride_row;
  p.ws_block = a->w_scale_stride_block;
  p.out_stride = a->out_stride;
  p.blocks = static_cast<int>(ceil_div64(a->k, kBlock));
  if (a->m <= 16) return launch_any<16>(a, x, w, p, info.num_sms, stream);
  if (a->m <= 32) return launch_any<32>(a, x, w, p, info.num_sms, stream);
  if (a->m <= 64) return launch_any<64>(a, x, w, p, info.num_sms, stream);
  if (a->m <= 128) return launch_any<128>(a, x, w, p, info.num_sms, stream);
  return launch_any<256>(a, x, w, p, info.num_sms, stream);
}

}  // namespace b200
