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
// Orientation.  An epilogue thread owns one row of the accumulator (a TMEM lane).
//   Many tokens: tokens are the rows and 128 or 256 outputs the columns, so that a
//   thread has one scale product per block and 128 outputs, and writes neighbouring
//   outputs of its token.  (With the outputs as rows the scales differ per column;
//   reading 256 of them from shared memory took twice the MMAs' time, since a load
//   returns 128 bytes a clock even where all lanes read the same.)
//   Few tokens (up to 128): outputs are the rows and the tokens the columns, 16 to
//   128 of them, so that the weight, which is all that counts, fills the MMA's M.
//
//   warps 0..kEpi-1    epilogue: warp i reads lanes 32 (i % 4) .., the columns are
//                      split over kEpi / 4 groups
//   warp kEpi          TMA producer: both tiles of a block per stage
//   warp kEpi + 1      MMA issuer (one thread)
//   warp kEpi + 2      scales of the blocks ahead, by asynchronous copies
//
// Pairs.  With 256 columns, two CTAs share a tile of 256 x 256 (cta_group::2): each
// loads its 128 rows and half of the columns, 32 KB a block instead of 48.  Alone, a
// CTA's tile of 128 x 256 asks 96 KB a block of shared memory (48 written, 48 read by
// the MMAs), which at 128 bytes a clock is 1.5 times the MMAs' 512 clocks.
//
// Work: tiles of 128 rows x COLS columns, tokens innermost so that neighbouring
// CTAs share weight rows in L2.  CTAs are persistent.  Where tiles are fewer than
// SMs, a cluster of CTAs splits K and joins its sums through distributed shared
// memory in rank order (the result does not depend on timing).
//
// Measured on a B200, quantiser included: 4099 tokens x 4096 x 28672 in 484 us in a
// burst (graph replay), 1990 TFLOP/s, 0.60 of twice the measured bf16 burst rate; back
// to back 554 to 566 us, 1740 to 1700 TFLOP/s, 0.61 to 0.62 of twice the sustained rate
// (power-capped).  Tensor pipe active 53 % of the time.
// What bounds it is the way of a block through its two accumulators: 512 clocks of
// MMAs, the signal to the epilogue, the reads, the signal back, and at each block's
// start the TMEM latency with nothing of the block before left to add.  64 tokens x 4096
// x 28672 in 28.6 us, 4.3 TB/s of weight: 224 tiles on 296 places for CTAs, so that 76
// SMs work on two tiles and 72 on one.  One token x 4096 x 6144 in 13.4 to 14.9 us, of
// which the weight's bytes would take 3.9: the quantiser's launch, the pipeline's fill
// and the join of 6 splits.
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
#include "fp8_quant.h"
#include "host_common.h"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

typedef unsigned long long u64;

constexpr int kRows = 128;   // rows of a tile = MMA M
constexpr int kBlock = 128;  // K per scale block = bytes of a swizzled row
constexpr int kScaleRing = 8;
constexpr int kMaxSplits = 8;
constexpr int kManyBlocks = 64;  // of K, from which tokens as rows are worth a join
constexpr int kPartPitch = kRows + 1;  // of the sums that a cluster joins: both ways conflict-free

// TOKEN_ROWS: tokens are the tile's rows and outputs its columns; else the reverse.
template <int COLS, bool TOKEN_ROWS>
struct Shape {
  static constexpr int kGroups = COLS > 128 ? 2 : 1;  // of epilogue warps, by columns
  static constexpr int kEpi = 4 * kGroups;
  static constexpr int kThreads = (kEpi + 4) * 32;
  static constexpr int kCols = COLS / kGroups;         // columns of an epilogue thread
  // Columns of the TMEM loads, in turn.  128 columns: 32, 16, 32, 16, 32 -- twice 32
  // do not fit the registers, twice 16 leave more of a load's latency uncovered.
  static constexpr int kStepA = kCols >= 128 ? 32 : 16, kStepB = 16;
  static_assert(kCols % (kStepA + kStepB) == 0 || kCols % (kStepA + kStepB) == kStepA,
                "the loads end with the columns");
  // 256 columns: 128 sums and 48 loaded values per epilogue thread are more than the
  // 168 registers of 384 threads, so that the other four warps give some of theirs.
  static constexpr bool kSplitRegisters = COLS > 128;
  static constexpr int kEpiRegisters = 224, kOtherRegisters = 56, kLaunchRegisters = 168;
  static_assert(kEpi * kEpiRegisters + 4 * kOtherRegisters <= (kEpi + 4) * kLaunchRegisters ||
                    !kSplitRegisters,
                "what the epilogue takes is what the other warps give");
  static constexpr bool kPair = COLS > 128;
  static constexpr int kLoadCols = kPair ? COLS / 2 : COLS;  // columns that a CTA loads
  static constexpr int kStageBytes = (kRows + kLoadCols) * kBlock;
  // Up to 64 columns a CTA takes under half an SM, so that two share it: the
  // product is then bound by the weight's bytes, which more CTAs spread better (one
  // token, 4096 x 28672: 24.4 us, and 31.3 with one CTA of 8 stages per SM).
  static constexpr int kCtasPerSm = COLS <= 64 ? 2 : 1;
  static constexpr int kStages = COLS <= 32 ? 5 : COLS <= 64 ? 4 : 6;
  static constexpr int kBuffers = COLS > 128 ? 2 : 4;  // accumulators
  static constexpr int kBufferCols = COLS < 32 ? 32 : COLS;
  static constexpr int kTmemCols = kBuffers * kBufferCols;
  // Scales of a block: one per token of the tile, then one per 128 outputs.
  static constexpr int kTokens = TOKEN_ROWS ? kRows : COLS;
  static constexpr int kScales = (kTokens + 4 + 3) / 4 * 4;
  static constexpr int kScaleBytes = kScaleRing * kScales * 4;
  static constexpr int kBars = 2 * kStages + 2 * kBuffers + 2 * kScaleRing + 1;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleBytes + kBars * 8 + 16;
  static_assert(kTmemCols <= 512 / kCtasPerSm, "TMEM columns");
  static_assert(kPartPitch * COLS * 4 <= kStages * kStageBytes || kPair,
                "the split sums reuse the stages");
  static_assert(kSmem <= 227 * 1024 / kCtasPerSm - 1024, "shared memory");
  // Two pairs (of launches on two streams) that each held one SM's TMEM and waited for
  // the other's would wait for good: a pair's CTA leaves no room for another on its SM.
  static_assert(!kPair || 2 * kSmem > 227 * 1024, "one CTA of a pair per SM");
};

struct LinearParams {
  const float* x_scales;
  const float* w_scales;
  const void* bias;
  void* out;
  uint32_t* err;
  int m, n;
  long long xs_row, xs_block, ws_row, ws_block, out_stride;
  int blocks;  // of K
  int token_tiles;
  int tiles, splits;
  int wide_stores;   // 32-byte stores of a token's outputs
  int weight_first;  // the weight may be read ahead of griddepcontrol.wait
};

// d += a * b on two packed 32-bit values.
__device__ __forceinline__ void fma2(u64& d, u64 a, u64 b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 4 bytes global -> shared, asynchronous.
__device__ __forceinline__ void copy_async_4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
// Arrive on `bar` when this thread's asynchronous copies so far have landed.
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void store_32b(void* dst, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
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

// A bounded wait whose outcome every lane of the warp shares; out of line where it
// has to wait.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          uint32_t* err) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, err, kErrWaitFull));
}

// Adds the sums of a tile's `p.splits` <= RANKS CTAs and stores this rank's share of
// its tokens.  Remote loads of RANKS x TOKENS values are in flight at once: a loop
// over them pays their latency each time (8 splits, one token: 10 us).
template <typename E, typename S, bool TOKEN_ROWS, int RANKS, int TOKENS>
__device__ __forceinline__ void join(cg::cluster_group& cluster, const LinearParams& p,
                                     const float* part, int rank, int m0, int n0) {
  using T = typename E::T;
  constexpr int kTileOuts = TOKEN_ROWS ? S::kCols * S::kGroups : kRows;
  constexpr int kSlices = S::kThreads / kTileOuts;
  const int o = threadIdx.x % kTileOuts, n = n0 + o;
  const int t1 = min(S::kTokens * (rank + 1) / p.splits, p.m - m0);
  if (n >= p.n) return;
  const float bias = p.bias ? to_float<E>(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
  for (int t0 = S::kTokens * rank / p.splits + threadIdx.x / kTileOuts; t0 < t1;
       t0 += kSlices * TOKENS) {
    float from[RANKS][TOKENS];
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      const float* there = cluster.map_shared_rank(part, min(r, p.splits - 1));
#pragma unroll
      for (int i = 0; i < TOKENS; ++i) {
        const int t = t0 + i * kSlices;
        from[r][i] = 0.f;
        if (r < p.splits && t < t1)
          from[r][i] = there[TOKEN_ROWS ? o * kPartPitch + t : t * kPartPitch + o];
      }
    }
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
      const int t = t0 + i * kSlices;
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < RANKS; ++r) sum += from[r][i];
      if (t < t1)
        reinterpret_cast<T*>(p.out)[static_cast<long long>(m0 + t) * p.out_stride + n] =
            from_float<E>(sum + bias);
    }
  }
}

template <typename E, int COLS, bool TOKEN_ROWS>
__global__ void __launch_bounds__(Shape<COLS, TOKEN_ROWS>::kThreads,
                                  Shape<COLS, TOKEN_ROWS>::kCtasPerSm)
    fp8_linear_kernel(const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ CUtensorMap xmap, const LinearParams p) {
  using S = Shape<COLS, TOKEN_ROWS>;
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
  constexpr bool kPair = S::kPair;
  const int per_tile = kPair ? 2 : p.splits;  // CTAs of a tile
  const int tile0 = blockIdx.x / per_tile, tile_step = gridDim.x / per_tile;
  const int part = kPair ? 0 : rank;  // of K
  const int kb0 = static_cast<int>(static_cast<long long>(p.blocks) * part / p.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(p.blocks) * (part + 1) / p.splits);

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kPair ? 2 * S::kEpi : S::kEpi);  // of a pair: rank 0's is used
    }
    for (int i = 0; i < kScaleRing; ++i) {
      mbar_init(&sc_full[i], 32);  // every lane's copies
      mbar_init(&sc_empty[i], S::kEpi);
    }
    mbar_init(mma_idle, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == S::kEpi + 1) {
    if (kPair) {
      tc::tmem_alloc_pair(tmem_slot, S::kTmemCols);
      tc::tmem_relinquish_pair();
    } else {
      tc::tmem_alloc(tmem_slot, S::kTmemCols);
      tc::tmem_relinquish();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (kPair) cluster.sync();  // the other CTA's barriers are in place, too
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // Launched with programmatic stream serialization: nothing of the previous kernel
  // may be read, and nothing that it reads be written, ahead of this wait.  Only the
  // producer has something to do before it.
  if (warp != S::kEpi) asm volatile("griddepcontrol.wait;" ::: "memory");

  bool ok = true;
  const int row = (warp & 3) * 32 + lane;  // of the tile; TMEM lane
  const int group = warp >> 2, col0 = group * S::kCols;
  constexpr int kTileOuts = TOKEN_ROWS ? COLS : kRows;
  constexpr int per_pair = kPair ? 2 : 1;  // token tiles of a CTA pair
  const int pair_rank = kPair ? rank : 0;
  if (warp >= S::kEpi) {
    if (S::kSplitRegisters)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegisters));
    if (warp == S::kEpi) {
      // ------------------------------ producer ------------------------------
      if (lane == 0) {
        tma_prefetch_desc(&wmap);
        tma_prefetch_desc(&xmap);
        auto load_w = [&](int s, int kb, int n0) {
          uint8_t* dst = stages + s * S::kStageBytes + (TOKEN_ROWS ? kRows * kBlock : 0);
          if (kPair)
            tma_load_2d_pair(dst, &wmap, cluster_address(&full[s], 0), kb * kBlock, n0);
          else
            tma_load_2d(dst, &wmap, &full[s], kb * kBlock, n0);
        };
        auto expect = [&](int s) {  // of a pair: both CTAs' bytes, on rank 0's barrier
          if (!kPair)
            mbar_arrive_expect_tx(&full[s], S::kStageBytes);
          else if (rank == 0)
            mbar_arrive_expect_tx(&full[s], 2 * S::kStageBytes);
        };
        // The weight does not come from the previous kernel where that is this call's
        // quantiser, which has itself waited for everything before it: the first
        // stages' weight tiles are loaded while it runs.
        int early = 0;
        if (p.weight_first && tile0 < p.tiles) {
          const int n0 = tile0 / p.token_tiles * kTileOuts + (kPair ? rank * S::kLoadCols : 0);
          for (; early < kStages && kb0 + early < kb1; ++early) {
            expect(early);
            load_w(early, kb0 + early, n0);
          }
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int it = 0;
        for (int tile = tile0; tile < p.tiles && ok; tile += tile_step) {
          const int n0 = tile / p.token_tiles * kTileOuts + (kPair ? rank * S::kLoadCols : 0);
          const int m0 = (tile % p.token_tiles * per_pair + pair_rank) * S::kTokens;
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % kStages;
            if (it >= early) {
              ok = mbar_wait_bounded(&empty[s], ((it / kStages) & 1) ^ 1, abort_flag, p.err,
                                     kErrWaitEmpty);
              if (!ok) break;
              expect(s);
              load_w(s, kb, n0);
            }
            uint8_t* dst = stages + s * S::kStageBytes + (TOKEN_ROWS ? 0 : kRows * kBlock);
            if (kPair)
              tma_load_2d_pair(dst, &xmap, cluster_address(&full[s], 0), kb * kBlock, m0);
            else
              tma_load_2d(dst, &xmap, &full[s], kb * kBlock, m0);
          }
        }
        // Rank 0's commits arrive on both CTAs' barriers.  Rank 1 sees the last of them,
        // the stages' releases and then mma_idle, before its shared memory is given up.
        if (kPair && rank == 1) {
          for (int i = it; ok && i < it + kStages; ++i)
            ok = mbar_wait_bounded(&empty[i % kStages], ((i / kStages) & 1) ^ 1, abort_flag,
                                   p.err, kErrWaitEmpty);
          mbar_drain(mma_idle, 0, p.err);
        } else {
          drain_stages<kStages>(full, it, p.err);
        }
        // After an abort, rank 1's copies have no barrier of its own to wait for: far
        // longer than any copy takes.
        if (kPair && !ok)
          for (const unsigned long long t0 = global_timer_ns();
               global_timer_ns() - t0 < 2000000ull;) {
          }
      }
    } else if (warp == S::kEpi + 1) {
      // ------------------------------ MMA issuer ----------------------------
      if (lane == 0 && (!kPair || rank == 0)) {
        // The issue of a block has to fit into the MMAs of the one before: descriptors
        // of stage 0 to which a stage's and a K step's 16-byte units are added (the
        // address field does not overflow), and counters instead of divisions.
        const uint32_t idesc = tc::idesc_e4m3(kPair ? 2 * kRows : kRows, COLS);
        const uint64_t rows0 = tc::sdesc_sw128(smem_u32(stages), 16, 1024);
        const uint64_t cols0 = tc::sdesc_sw128(smem_u32(stages) + kRows * kBlock, 16, 1024);
        int s = 0, b = 0;
        uint32_t stage_phase = 0, buffer_phase = 1;
        for (int tile = tile0; tile < p.tiles && ok; tile += tile_step) {
          for (int kb = kb0; kb < kb1; ++kb) {
            ok = mbar_wait_bounded(&full[s], stage_phase, abort_flag, p.err, kErrWaitFull) &&
                 mbar_wait_bounded(&acc_empty[b], buffer_phase, abort_flag, p.err,
                                   kErrWaitEmpty);
            if (!ok) break;
            tc::fence_after_sync();
            const uint64_t da = rows0 + static_cast<uint32_t>(s) * (S::kStageBytes / 16);
            const uint64_t db = cols0 + static_cast<uint32_t>(s) * (S::kStageBytes / 16);
            const uint32_t d = tmem + b * S::kBufferCols;
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k) {
              if (kPair)
                tc::mma_e4m3_pair(d, da + 2 * k, db + 2 * k, idesc, k > 0);
              else
                tc::mma_e4m3(d, da + 2 * k, db + 2 * k, idesc, k > 0);
            }
            if (kPair) {
              tc::commit_pair(&acc_full[b]);
              tc::commit_pair(&empty[s]);
            } else {
              tc::commit(&acc_full[b]);
              tc::commit(&empty[s]);
            }
            if (++s == kStages) {
              s = 0;
              stage_phase ^= 1;
            }
            if (++b == kBuffers) {
              b = 0;
              buffer_phase ^= 1;
            }
          }
        }
        // Every MMA this thread issued has finished before TMEM can be freed.
        if (kPair)
          tc::commit_pair(mma_idle);
        else
          tc::commit(mma_idle);
        mbar_drain(mma_idle, 0, p.err);
      }
    } else if (warp == S::kEpi + 2) {
      // -------------------------------- scales ------------------------------
      int it = 0;
      for (int tile = tile0; tile < p.tiles && ok; tile += tile_step) {
        const int m0 = (tile % p.token_tiles * per_pair + pair_rank) * S::kTokens;
        const int n0 = tile / p.token_tiles * kTileOuts;
        const float* sx = p.x_scales + (m0 + lane) * p.xs_row;
        const float* sw = p.w_scales + (n0 / 128 + lane) * p.ws_row;
        const bool has_w = lane < S::kGroups && n0 + lane * 128 < p.n;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int r = it % kScaleRing;
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sc_empty[r], ((it / kScaleRing) & 1) ^ 1,
                                                         abort_flag, p.err, kErrWaitEmpty));
          if (!ok) break;
          float* dst = scales + r * S::kScales;
#pragma unroll
          for (int i = 0; i < (S::kTokens + 31) / 32; ++i) {
            const int c = i * 32 + lane;
            if (c < S::kTokens && m0 + c < p.m)
              copy_async_4(dst + c, sx + i * 32 * p.xs_row + kb * p.xs_block);
          }
          if (has_w) copy_async_4(dst + S::kTokens + lane, sw + kb * p.ws_block);
          copy_async_arrive(&sc_full[r]);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    // ------------------------------ epilogue ------------------------------
    if (S::kSplitRegisters)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kEpiRegisters));
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + col0;
    auto release = [&](uint64_t* bar) {  // the accumulator has been read
      tc::fence_before_sync();
      if (lane == 0) {
        if (kPair)
          mbar_arrive_remote(cluster_address(bar, 0));
        else
          mbar_arrive(bar);
      }
    };
    int it = 0;
    for (int tile = tile0; tile < p.tiles && ok; tile += tile_step) {
      u64 acc[S::kCols / 2];
#pragma unroll
      for (int i = 0; i < S::kCols / 2; ++i) acc[i] = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int b = it % kBuffers, r = it % kScaleRing;
        ok = warp_wait(&acc_full[b], (it / kBuffers) & 1, abort_flag, p.err);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t base = lane_base + b * S::kBufferCols;
        uint32_t va[S::kStepA], vb[S::kStepB];
        load_columns(base, va);
        // Meanwhile the scales: with tokens as rows, this row's.
        ok = warp_wait(&sc_full[r], (it / kScaleRing) & 1, abort_flag, p.err);
        if (!ok) {
          tc::wait_ld(va);
          break;
        }
        const float* sc = scales + r * S::kScales;
        const float sw = sc[S::kTokens + group];
        const float s1 = TOKEN_ROWS ? sc[row] * sw : sw;
        const u64 s2 = pack_f32x2(__float_as_uint(s1), __float_as_uint(s1));
        const ulonglong2* sx = reinterpret_cast<const ulonglong2*>(sc);
        if (TOKEN_ROWS) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[r]);
        }
        auto add = [&](auto& v, int c0) {  // columns c0 .. to the sums
          constexpr int kN = sizeof(v) / 4;
#pragma unroll
          for (int i = 0; i < kN / 4; ++i) {
            ulonglong2 f = make_ulonglong2(s2, s2);
            if (!TOKEN_ROWS) {
              f = sx[c0 / 4 + i];
              f.x = mul2(f.x, s2);
              f.y = mul2(f.y, s2);
            }
            const int a = c0 / 2 + 2 * i;
            fma2(acc[a], pack_f32x2(v[4 * i], v[4 * i + 1]), f.x);
            fma2(acc[a + 1], pack_f32x2(v[4 * i + 2], v[4 * i + 3]), f.y);
          }
        };
        // The next columns are on their way while these are added.
        constexpr int kA = S::kStepA, kB = S::kStepB, kAB = kA + kB;
#pragma unroll
        for (int c = 0; c < S::kCols; c += kAB) {
          tc::wait_ld(va);
          if (c + kA < S::kCols)
            load_columns(base + c + kA, vb);
          else
            release(acc_empty + b);
          add(va, c);
          if (c + kA < S::kCols) {
            tc::wait_ld(vb);
            if (c + kAB < S::kCols)
              load_columns(base + c + kAB, va);
            else
              release(acc_empty + b);
            add(vb, c + kA);
          }
        }
        if (!TOKEN_ROWS) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[r]);
        }
      }
      if (!ok) break;
      if (!kPair && p.splits > 1) {
        // One tile per CTA: its stages are free, every copy and MMA has finished.
        float* part = reinterpret_cast<float*>(stages) + col0 * kPartPitch + row;
#pragma unroll
        for (int i = 0; i < S::kCols / 2; ++i) {
          const float2 f = unpack_f32x2(acc[i]);
          part[2 * i * kPartPitch] = f.x;
          part[(2 * i + 1) * kPartPitch] = f.y;
        }
      } else if (TOKEN_ROWS) {
        const int m = (tile % p.token_tiles * per_pair + pair_rank) * kRows + row;
        const int n0 = tile / p.token_tiles * COLS + col0;
        if (m < p.m && n0 < p.n) {
          T* out = reinterpret_cast<T*>(p.out) + static_cast<long long>(m) * p.out_stride + n0;
          const T* bias = reinterpret_cast<const T*>(p.bias);
#pragma unroll
          for (int i = 0; i < S::kCols / 16; ++i) {
            float f[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 pair = unpack_f32x2(acc[8 * i + j]);
              f[2 * j] = pair.x;
              f[2 * j + 1] = pair.y;
            }
            if (bias) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (n0 + 16 * i + j < p.n) f[j] += to_float<E>(bias[n0 + 16 * i + j]);
            }
            if (p.wide_stores && n0 + 16 * i + 16 <= p.n) {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j] = pack2<E>(f[2 * j], f[2 * j + 1]);
              store_32b(out + 16 * i, w);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (n0 + 16 * i + j < p.n) out[16 * i + j] = from_float<E>(f[j]);
            }
          }
        }
      } else {
        const int n = tile / p.token_tiles * kRows + row;
        const int m0 = tile % p.token_tiles * COLS + col0;
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
      }
    }
  }
  __syncwarp();  // single-thread roles rejoin their warp
  if (!kPair && p.splits > 1) {
    // Join: rank r adds the tokens [kTokens r / splits, ...) of all ranks, in rank
    // order; neighbouring threads take neighbouring outputs.
    cluster.sync();
    if (*abort_flag == 0) {
      const int m0 = tile0 % p.token_tiles * S::kTokens;
      const int n0 = tile0 / p.token_tiles * kTileOuts;
      const float* part = reinterpret_cast<const float*>(stages);
      if (p.splits <= 2)
        join<E, S, TOKEN_ROWS, 2, 8>(cluster, p, part, rank, m0, n0);
      else if (p.splits <= 4)
        join<E, S, TOKEN_ROWS, 4, 4>(cluster, p, part, rank, m0, n0);
      else
        join<E, S, TOKEN_ROWS, 8, 2>(cluster, p, part, rank, m0, n0);
    }
    cluster.sync();  // no CTA leaves while another may still read its sums
  }
  // ---- teardown: every TMEM access is done, the MMA warp frees TMEM ----
  tc::fence_before_sync();
  __syncthreads();
  if (kPair) cluster.sync();  // rank 0's MMAs read and write both CTAs' memory
  if (warp == S::kEpi + 1) {
    tc::fence_after_sync();
    if (kPair)
      tc::tmem_dealloc_pair(tmem, S::kTmemCols);
    else
      tc::tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <typename E, int COLS, bool TOKEN_ROWS>
int launch(const CUtensorMap& wmap, const CUtensorMap& xmap, const LinearParams& p, int ctas,
           cudaStream_t stream) {
  using S = Shape<COLS, TOKEN_ROWS>;
  auto kern = fp8_linear_kernel<E, COLS, TOKEN_ROWS>;
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
  attr[0].val.clusterDim.x = static_cast<unsigned>(S::kPair ? 2 : p.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, wmap, xmap, p), "fp8_linear_kernel launch");
}

template <int COLS, bool TOKEN_ROWS>
int launch_any(const b200_fp8_linear_args* a, const void* x, const void* w, LinearParams p,
               int sms, cudaStream_t stream) {
  using S = Shape<COLS, TOKEN_ROWS>;
  const int slots = sms * S::kCtasPerSm;
  const int tile_outs = TOKEN_ROWS ? COLS : kRows;
  const int per_tile = S::kPair ? 2 : 1;
  p.token_tiles = static_cast<int>(ceil_div64(a->m, S::kTokens * per_tile));
  const long long tiles = ceil_div64(a->n, tile_outs) * p.token_tiles;
  if (tiles > 0x7fffffffLL / kMaxSplits)
    return set_error(B200_ERR_UNSUPPORTED, "too many output tiles");
  p.tiles = static_cast<int>(tiles);
  // Splits of K that still fit the CTAs at once, each with two blocks or more.  With
  // tokens as rows a join moves 64 KB a CTA and costs about 25 blocks' time (256
  // tokens, 4096 outputs: 29.5 us split and 19.7 whole at 32 blocks, 47 and 54 us at
  // 112), so that K is split from 64 blocks on.
  p.splits = S::kPair || (TOKEN_ROWS && p.blocks < kManyBlocks)
                 ? 1
                 : static_cast<int>(std::max<long long>(
                       1, std::min<long long>({kMaxSplits, slots / tiles, p.blocks / 2})));
  const long long ctas = p.splits > 1 ? tiles * p.splits
                                      : std::min<long long>(tiles, slots / per_tile) * per_tile;
  const uint64_t wdims[2] = {static_cast<uint64_t>(a->k), static_cast<uint64_t>(a->n)};
  const uint64_t xdims[2] = {static_cast<uint64_t>(a->k), static_cast<uint64_t>(a->m)};
  // A single row has no stride of its own; a map's must hold the row.
  const int64_t pitch = ceil_div64(a->k, 16) * 16;
  const uint64_t wstride[1] = {static_cast<uint64_t>(std::max<int64_t>(a->w_stride, pitch))};
  const uint64_t xstride[1] = {static_cast<uint64_t>(std::max<int64_t>(a->x_stride, pitch))};
  const uint32_t wbox[2] = {kBlock, static_cast<uint32_t>(S::kPair ? S::kLoadCols : tile_outs)};
  const uint32_t xbox[2] = {kBlock, static_cast<uint32_t>(S::kTokens)};
  CUtensorMap wmap, xmap;
  int rc = encode_tensor_map_8b(w, 2, wdims, wstride, wbox, &wmap);
  if (rc == B200_OK) rc = encode_tensor_map_8b(x, 2, xdims, xstride, xbox, &xmap);
  if (rc != B200_OK) return rc;
  return a->dtype == B200_BF16
             ? launch<BF16, COLS, TOKEN_ROWS>(wmap, xmap, p, static_cast<int>(ctas), stream)
             : launch<Half, COLS, TOKEN_ROWS>(wmap, xmap, p, static_cast<int>(ctas), stream);
}

}  // namespace

int launch_fp8_linear(const b200_fp8_linear_args* args, const void* x, const float* x_scales,
                      const void* w, const float* w_scales, const void* bias, void* out,
                      void* workspace, size_t workspace_bytes, uint32_t* error_word,
                      cudaStream_t stream) {
  if (args == nullptr) return set_error(B200_ERR_INVALID, "null descriptor");
  b200_fp8_linear_args quantized = *args;
  b200_fp8_linear_args* a = &quantized;
  if (a->dtype != B200_F16 && a->dtype != B200_BF16)
    return set_error(B200_ERR_UNSUPPORTED, "the output must be float16 or bfloat16");
  if (a->x_dtype != B200_E4M3 && a->x_dtype != a->dtype)
    return set_error(B200_ERR_INVALID, "x must be e4m3 or have the output's type");
  if (a->m < 0 || a->n <= 0 || a->k <= 0)
    return set_error(B200_ERR_INVALID, "rows/outputs/columns out of range");
  if (a->m > 0x7fffff00LL || a->n > 0x7fffff00LL || a->k > 0x7fffff00LL)
    return set_error(B200_ERR_UNSUPPORTED, "sizes are limited to 2^31 - 256");
  if (a->w_stride % 16 != 0 || (a->x_dtype == B200_E4M3 && a->x_stride % 16 != 0))
    return set_error(B200_ERR_INVALID, "rows of x and weight must start on 16-byte boundaries");
  if ((a->n > 1 && a->w_stride < a->k) ||
      (a->x_dtype == B200_E4M3 && a->m > 1 && a->x_stride < a->k))
    return set_error(B200_ERR_INVALID, "rows of x and weight must not overlap");
  if (a->m > 1 && a->out_stride < a->n)
    return set_error(B200_ERR_INVALID, "rows of out must not overlap");
  if (a->m == 0) return B200_OK;
  if (!x || !w || !w_scales || !out || (a->x_dtype == B200_E4M3 && !x_scales))
    return set_error(B200_ERR_INVALID, "null tensor pointer");
  DeviceInfo info;
  int rc = current_device_info(&info);
  if (rc != B200_OK) return rc;
  if (a->x_dtype != B200_E4M3) {
    const int64_t pitch = ceil_div64(a->k, 16) * 16, blocks = ceil_div64(a->k, kBlock);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
        workspace_bytes < static_cast<size_t>(a->m) * (pitch + 4 * blocks))
      return set_error(B200_ERR_WORKSPACE, "fp8_linear workspace missing, unaligned or too small");
    float* scales = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + a->m * pitch);
    rc = launch_quantize_fp8(x, a->m, a->k, a->x_stride, a->x_dtype, 1, workspace, pitch, scales, 1,
                             a->m, stream);
    if (rc != B200_OK) return rc;
    x = workspace;
    x_scales = scales;
    a->x_stride = pitch;
    a->x_scale_stride_row = 1;
    a->x_scale_stride_block = a->m;
  }
  LinearParams p;
  p.x_scales = x_scales;
  p.w_scales = w_scales;
  p.bias = bias;
  p.weight_first = args->x_dtype != B200_E4M3;  // the previous kernel is the quantiser above
  p.out = out;
  p.err = error_word;
  p.m = static_cast<int>(a->m);
  p.n = static_cast<int>(a->n);
  p.xs_row = a->x_scale_stride_row;
  p.xs_block = a->x_scale_stride_block;
  p.ws_row = a->w_scale_stride_row;
  p.ws_block = a->w_scale_stride_block;
  p.out_stride = a->out_stride;
  p.blocks = static_cast<int>(ceil_div64(a->k, kBlock));
  p.wide_stores = a->out_stride % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  const int sms = info.num_sms;
  if (a->m <= 16) return launch_any<16, false>(a, x, w, p, sms, stream);
  if (a->m <= 32) return launch_any<32, false>(a, x, w, p, sms, stream);
  if (a->m <= 64) return launch_any<64, false>(a, x, w, p, sms, stream);
  // Up to 128 tokens the weight's rows as MMA rows still pay where a long K has to be
  // split over few tiles (128 tokens, 4096 outputs, 112 blocks: 31 us against 44);
  // else tokens as rows, whose scales cost nothing per column (28672 outputs, 32
  // blocks: 41 us against 55; 6144 outputs: 20 against 35).
  if (a->m <= 128 && p.blocks >= kManyBlocks && ceil_div64(a->n, kRows) * 2 <= sms)
    return launch_any<128, false>(a, x, w, p, sms, stream);
  // Single CTAs of 128 x 128 while one wave holds them, else pairs (512 tokens x 4096 x
  // 4096, 128 tiles: 20 us against 23; 512 x 4096 x 6144, 192 tiles: 34 against 24).
  if (ceil_div64(a->m, kRows) * ceil_div64(a->n, 128) > sms)
    return launch_any<256, true>(a, x, w, p, sms, stream);
  return launch_any<128, true>(a, x, w, p, sms, stream);
}

}  // namespace b200
