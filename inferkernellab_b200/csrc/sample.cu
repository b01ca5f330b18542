// Next tokens of a batch from its logits, one launch: temperature, min-p, top-k
// and top-p, and a draw from one given uniform number per row.
//
//   l   = logits in 32 bits, NaN taken as -inf;  m = max l
//   w_i = exp((l_i - m) / T)                 (m = +inf: 1 where l_i = m, else 0)
//   tokens in order of w, equal ones by index; kept is the longest prefix with
//     w_i >= min_p,   rank < top_k,   mass before i < top_p * (mass of the first two)
//   token = the first index, in order of index, where the running mass of the
//           kept tokens passes floor(u * their mass)
//   logprob = log w - log sum w,   sampling logprob = log w - log (sum of kept w)
// T <= 0 takes the first largest logit (its logprobs are those of T = 1).
//
// Masses are whole numbers: q_i = rint(w_i * 2^31), summed in 64 bits.  Whole
// sums do not depend on the order of the additions, so the cut and the token are
// the same for every split of the row and every run; a weight below 2^-32 of the
// largest is never drawn.  The two log-probabilities use 32-bit weights, summed
// per thread and joined in 64 bits.
//
// Layout.  A cluster of 1..8 CTAs owns a row and reads it from memory once: each
// CTA keeps its slice in shared memory, first the logits, then the weights, and
// everything that follows runs from there, with what the CTAs have to tell each
// other read through distributed shared memory.  Warps own runs of neighbouring
// tokens, so a prefix over warps is a prefix over indices.
//
// Search.  Nothing is sorted.  The bits of w (w >= 0) are an order-preserving
// key.  A histogram of counts and masses over 249 bins of an eighth of an
// octave each finds the bin where the cut falls.  If at most kList tokens lie in
// it (the usual case) they are gathered and the cut is resolved by counting, for
// each of them, what precedes it.  Otherwise the bin is split into 1024 bins, as
// often as it takes (equal weights at the end: the cut is then between indices).
// The masses of a bin are kept as two 32-bit sums (low and high 16 bits; a CTA
// holds at most 2^16 tokens), since 64-bit shared-memory atomics are loops.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "../../include/b200_paged_attn.h"
#include "common.cuh"
#include "host_common.h"
#include "sample.h"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 1024;
constexpr int kFirstShift = 20;                         // bits below an eighth of an octave
constexpr uint32_t kFirstBase = (127u - 31u) << 3;      // key >> 20 of w = 2^-31
constexpr int kFirstBins = (127 << 3) - kFirstBase + 1;  // 249: the last one holds w = 1
constexpr int kList = 512;                              // tokens that are resolved by counting
constexpr int kMaxSlice = 46 * 1024;                    // tokens of a CTA (184 KB of weights)
constexpr float kLargest = 3.402823466e38f, kSmallest = 1.175494351e-38f;
static_assert(kMaxSlice <= (1 << 16), "the 32-bit mass sums hold 2^16 tokens");
static_assert(kList <= kThreads, "one thread per gathered token");

struct SampleParams {
  const void* logits;
  const float* uniforms;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long* tokens;
  float* logprobs;
  float* sampling_logprobs;
  long long stride;
  int vocab, slice;
};

struct Cut {       // kept: key > cut.key, or key == cut.key and index <= cut.index
  uint32_t key;
  int index;
};

struct Shared {
  uint32_t count[2][kBins], low[2][kBins], high[2][kBins];  // the first histogram, the finer ones
  uint2 list[2][kList];                                     // key, index (rank 0's is used)
  int listed[2];
  // What the other CTAs read, one slot per step.
  float pub_max;
  double pub_sum;
  u64 pub_mass;
  int pub_first, pub_pass;
  u64 pub_warp_mass[kWarps];
  float pub_warp_sum[kWarps];
  int pub_warp_ties[kWarps];
  int pub_tie_index;
  // Of this CTA alone.
  uint2 local_list[kList];
  u64 scan_mass[kWarps + 1];
  uint32_t scan_count[kWarps + 1];
  float red_f[kWarps];
  double red_d[kWarps];
  u64 red_u[kWarps];
  int red_i[kWarps], red_p[kWarps];
  int found_bin;
  uint32_t found_count, before_count;
  u64 before_mass, found_mass;
  Cut cut;
  u64 cut_mass;
};

static_assert(sizeof(Shared) + 16 + (kMaxSlice + 8) * 4 <= 227 * 1024, "shared memory of a CTA");

template <typename L>
__device__ __forceinline__ float logit_f32(L x);
template <>
__device__ __forceinline__ float logit_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float logit_f32<__half>(__half x) {
  return __half2float(x);
}
template <>
__device__ __forceinline__ float logit_f32<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

__device__ __forceinline__ float no_nan(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ uint32_t mass_of(float w) {
  return __float2uint_rn(__fmul_rn(w, 2147483648.0f));
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Which measure a cut is made on.
enum Measure { kCount, kMass };

template <typename L>
class Row {
 public:
  __device__ Row(const SampleParams& p, Shared& s, float* w, cg::cluster_group cluster)
      : p(p), s(s), w(w), cluster(cluster), ranks(cluster.num_blocks()),
        rank(cluster.block_rank()), tid(threadIdx.x), warp(threadIdx.x >> 5),
        lane(threadIdx.x & 31) {
    first = rank * p.slice;
    n = max(0, min(p.slice, p.vocab - first));
    const int run = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
    run0 = min(n, warp * run);
    run1 = min(n, run0 + run);
  }

  const SampleParams& p;
  Shared& s;
  float* w;  // the slice: logits, then weights
  cg::cluster_group cluster;
  const unsigned ranks, rank;
  const int tid, warp, lane;
  int first, n;    // the slice's first token and its length
  int run0, run1;  // this warp's part of the slice
  int level = 0;   // 0: the first histogram, 1: a finer one
  int lists = 0;   // lists gathered so far (at most one per search)

  __device__ Shared* at(unsigned r) { return cluster.map_shared_rank(&s, r); }

  // Reads the slice; returns the largest logit of the row (every thread).
  __device__ float load(const L* row) {
    constexpr int kVec = 16 / sizeof(L);
    const L* src = row + first;
    // 16-byte vectors from the first aligned element; w is shifted so that
    // those elements are aligned in shared memory, too.
    const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(src) / sizeof(L)) % kVec);
    const int head = min(n, skip ? kVec - skip : 0);
    w += skip;
    const int vecs = (n - head) / kVec;
    const int tail = head + vecs * kVec;
    float m = -INFINITY;
    if (tid < head) {
      const float x = no_nan(logit_f32<L>(src[tid]));
      w[tid] = x;
      m = x;
    }
    if (tid < n - tail) {
      const float x = no_nan(logit_f32<L>(src[tail + tid]));
      w[tail + tid] = x;
      m = fmaxf(m, x);
    }
    const uint4* vsrc = reinterpret_cast<const uint4*>(src + head);
    float4* vdst = reinterpret_cast<float4*>(w + head);
#pragma unroll 4
    for (int i = tid; i < vecs; i += kThreads) {
      const uint4 raw = vsrc[i];
      L x[kVec];
      memcpy(x, &raw, 16);
      float f[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        f[j] = no_nan(logit_f32<L>(x[j]));
        m = fmaxf(m, f[j]);
      }
#pragma unroll
      for (int j = 0; j < kVec / 4; ++j)
        vdst[i * (kVec / 4) + j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s.red_f[warp] = m;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kWarps; ++i) m = fmaxf(m, s.red_f[i]);
      s.pub_max = m;
    }
    cluster.sync();
    m = -INFINITY;
    for (unsigned r = 0; r < ranks; ++r) m = fmaxf(m, at(r)->pub_max);
    return m;
  }

  __device__ void clear_histogram(int bins) {
    for (int i = tid; i < bins; i += kThreads)
      s.count[level][i] = s.low[level][i] = s.high[level][i] = 0;
  }

  __device__ void add_to_bin(int bin, uint32_t q, bool with_mass) {
    atomicAdd(&s.count[level][bin], 1u);
    if (with_mass) {
      atomicAdd(&s.low[level][bin], q & 0xffffu);
      atomicAdd(&s.high[level][bin], q >> 16);
    }
  }

  // The bin of the row's histogram in which `target` is reached, counted from the
  // last bin down, on top of `count0` / `mass0` above the whole histogram; bin 0
  // of the first histogram is given by what the row's totals leave.  Sets
  // s.found_bin (-1: the row has less than target), found_count / found_mass (of
  // the bin) and before_count / before_mass (above it).
  __device__ void find_bin(int bins, Measure measure, u64 target, uint32_t count0, u64 mass0,
                           bool first_level, uint32_t row_count, u64 row_mass) {
    if (tid == 0) s.found_bin = -1;
    __syncthreads();
    uint32_t run_count = count0;
    u64 run_mass = mass0;
    for (int base = 0; base < bins; base += kThreads) {
      const int bin = bins - 1 - (base + tid);
      uint32_t c = 0;
      u64 q = 0;
      if (bin >= (first_level ? 1 : 0)) {
        u64 lo = 0, hi = 0;
        for (unsigned r = 0; r < ranks; ++r) {
          const Shared* o = at(r);
          c += o->count[level][bin];
          lo += o->low[level][bin];
          hi += o->high[level][bin];
        }
        q = lo + (hi << 16);
      }
      // Inclusive prefix over the block.
      uint32_t ci = c;
      u64 qi = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o);
        const u64 qu = __shfl_up_sync(0xffffffffu, qi, o);
        if (lane >= o) {
          ci += cu;
          qi += qu;
        }
      }
      if (lane == 31) {
        s.scan_count[warp] = ci;
        s.scan_mass[warp] = qi;
      }
      __syncthreads();
      uint32_t total_c = 0;
      u64 total_q = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i == warp) {
          ci += total_c;
          qi += total_q;
        }
        total_c += s.scan_count[i];
        total_q += s.scan_mass[i];
      }
      uint32_t before_c = run_count + ci - c;
      u64 before_q = run_mass + qi - q;
      if (first_level && bin == 0) {  // what the bins above leave of the row
        c = row_count - before_c;
        q = row_mass - before_q;
      }
      if (bin >= 0) {
        const u64 before = measure == kCount ? before_c : before_q;
        const u64 with = before + (measure == kCount ? static_cast<u64>(c) : q);
        if (before < target && target <= with) {
          s.found_bin = bin;
          s.found_count = c;
          s.found_mass = q;
          s.before_count = before_c;
          s.before_mass = before_q;
        }
      }
      run_count += total_c;
      run_mass += total_q;
      __syncthreads();
      if (s.found_bin >= 0) break;  // block-uniform
    }
  }

  // The cut of the prefix that reaches `target` (>= 1): tokens up to and with the
  // one whose inclusive measure reaches it.  Returns false if all tokens with
  // w >= floor_w together have less; else sets s.cut and s.cut_mass (mass kept,
  // meaningful if the histograms carry masses).  The first histogram is in place
  // (buffer 0) and visible to the cluster.
  __device__ bool cut_at(Measure measure, u64 target, bool with_mass, float floor_w,
                         uint32_t row_count, u64 row_mass) {
    level = 0;
    find_bin(kFirstBins, measure, target, 0, 0, true, row_count, row_mass);
    if (s.found_bin < 0) return false;
    uint32_t lo = s.found_bin == 0 ? 0u : (kFirstBase + s.found_bin) << kFirstShift;
    uint32_t size = s.found_bin == 0 ? (kFirstBase + 1) << kFirstShift : 1u << kFirstShift;
    const uint32_t floor_key = __float_as_uint(floor_w);
    while (s.found_count > kList && size > 1) {
      const int shift = size > (1u << kFirstShift) ? kFirstShift : (size > 1024u ? 10 : 0);
      const int bins = static_cast<int>((size + (1u << shift) - 1) >> shift);
      const uint32_t before_count = s.before_count;
      const u64 before_mass = s.before_mass;
      level = 1;  // its last readers have passed the cluster barrier at the end of this loop
      clear_histogram(kBins);
      __syncthreads();
      for (int i = run0 + lane; i < run1; i += 32) {
        const float x = w[i];
        const uint32_t key = __float_as_uint(x);
        if (key - lo < size && key >= floor_key) add_to_bin((key - lo) >> shift, mass_of(x), true);
      }
      cluster.sync();
      find_bin(bins, measure, target, before_count, before_mass, false, 0, 0);
      // Totals of the bin above are exact, so one of its bins holds the target.
      if (s.found_bin < 0) return false;
      lo += static_cast<uint32_t>(s.found_bin) << shift;
      size = 1u << shift;
      cluster.sync();
    }
    if (s.found_count <= kList) {
      resolve_listed(measure, target, lo, size, floor_key);
    } else {
      resolve_ties(measure, target, lo);
    }
    return true;
  }

  // At most kList tokens with keys in [lo, lo + size): all of them to every CTA,
  // one thread each, and the one that reaches the target is the cut.
  __device__ void resolve_listed(Measure measure, u64 target, uint32_t lo, uint32_t size,
                                 uint32_t floor_key) {
    const int slot = lists++;
    Shared* home = at(0);
    for (int i = run0 + lane; i < run1; i += 32) {
      const uint32_t key = __float_as_uint(w[i]);
      if (key - lo < size && key >= floor_key) {
        const int to = atomicAdd(&home->listed[slot], 1);
        if (to < kList) home->list[slot][to] = make_uint2(key, static_cast<uint32_t>(first + i));
      }
    }
    cluster.sync();
    const int m = min(home->listed[slot], kList);
    if (tid < m) s.local_list[tid] = home->list[slot][tid];
    __syncthreads();
    if (tid < m) {
      const uint2 me = s.local_list[tid];
      const uint32_t mine = mass_of(__uint_as_float(me.x));
      u64 c = s.before_count, q = s.before_mass;
      for (int j = 0; j < m; ++j) {
        const uint2 o = s.local_list[j];
        if (o.x > me.x || (o.x == me.x && o.y < me.y)) {
          ++c;
          q += mass_of(__uint_as_float(o.x));
        }
      }
      const u64 before = measure == kCount ? c : q;
      const u64 with = before + (measure == kCount ? 1u : mine);
      if (before < target && target <= with) {
        s.cut.key = me.x;
        s.cut.index = static_cast<int>(me.y);
        s.cut_mass = q + mine;
      }
    }
    __syncthreads();
  }

  // More than kList tokens of one and the same weight: the cut is the r-th of them
  // in order of index.
  __device__ void resolve_ties(Measure measure, u64 target, uint32_t key) {
    const uint32_t q = mass_of(__uint_as_float(key));
    const u64 r = measure == kCount ? target - s.before_count
                                    : (target - s.before_mass + q - 1) / max(q, 1u);
    int ties = 0;
    for (int i = run0 + lane; i < run1; i += 32) ties += __float_as_uint(w[i]) == key;
    ties = warp_sum(ties);
    if (lane == 0) s.pub_warp_ties[warp] = ties;
    if (tid == 0) s.pub_tie_index = -1;
    cluster.sync();
    u64 before = 0;
    for (unsigned o = 0; o < rank; ++o)
      for (int i = 0; i < kWarps; ++i) before += at(o)->pub_warp_ties[i];
    for (int i = 0; i < warp; ++i) before += s.pub_warp_ties[i];
    if (before < r && r <= before + ties) {  // warp-uniform: the r-th is in this run
      for (int base = run0; base < run1; base += 32) {
        const int i = base + lane;
        const bool tie = i < run1 && __float_as_uint(w[i]) == key;
        const unsigned vote = __ballot_sync(0xffffffffu, tie);
        const u64 here = before + __popc(vote & ((2u << lane) - 1u));
        if (tie && here == r) s.pub_tie_index = first + i;
        before += __popc(vote);
      }
    }
    cluster.sync();
    int index = -1;
    for (unsigned o = 0; o < ranks; ++o) index = max(index, at(o)->pub_tie_index);
    if (tid == 0) {
      s.cut.key = key;
      s.cut.index = index;
      s.cut_mass = s.before_mass + r * q;
    }
    __syncthreads();
  }

};

template <typename L>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  float* w_base = reinterpret_cast<float*>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  Row<L> row(p, s, w_base, cluster);
  const int tid = row.tid, warp = row.warp, lane = row.lane;
  const long long b = blockIdx.x / row.ranks;
  row.clear_histogram(kFirstBins);
  if (tid == 0) {
    s.listed[0] = s.listed[1] = 0;
    s.pub_first = p.vocab;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const L* logits = reinterpret_cast<const L*>(p.logits) + b * p.stride;
  const float temperature = p.temperature ? p.temperature[b] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  float min_p = p.min_p ? p.min_p[b] : p.min_p_all;
  int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float u = p.uniforms[b];
  const bool greedy = !(temperature > 0.f);
  const bool cut_k = top_k > 0 && top_k < p.vocab;
  const bool cut_p = top_p < 1.f;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  // Finite and not zero, so that 0 and -inf keep their meaning when multiplied.
  const float inv = greedy ? 1.f : fmaxf(fminf(__fdiv_rn(1.f, temperature), kLargest), kSmallest);

  const float m = row.load(logits);
  if (m == -INFINITY) {  // cluster-uniform: nothing in this row can be drawn
    if (row.rank == 0 && tid == 0) {
      p.tokens[b] = -1;
      p.logprobs[b] = -INFINITY;
      p.sampling_logprobs[b] = -INFINITY;
    }
    cluster.sync();  // no CTA leaves while another may still read its pub_max
    return;
  }

  // Weights, their sums and the first histogram.
  float* w = row.w;
  float sum = 0.f;
  u64 mass = 0;
  int pass = 0;
  for (int i = row.run0 + lane; i < row.run1; i += 32) {
    const float l = w[i];
    const float x = m == INFINITY ? (l == m ? 0.f : -INFINITY) : __fmul_rn(__fsub_rn(l, m), inv);
    const float e = expf(x);
    w[i] = e;
    sum += e;
    if (l == m) atomicMin(&s.pub_first, row.first + i);
    if (e >= min_p) {
      const uint32_t q = mass_of(e);
      mass += q;
      ++pass;
      if (cut_k || cut_p) {
        const uint32_t hi = __float_as_uint(e) >> kFirstShift;
        if (hi > kFirstBase) row.add_to_bin(hi - kFirstBase, q, cut_p);
      }
    }
  }
  double dsum = warp_sum(static_cast<double>(sum));
  mass = warp_sum(mass);
  pass = warp_sum(pass);
  if (lane == 0) {
    s.red_d[warp] = dsum;
    s.red_u[warp] = mass;
    s.red_p[warp] = pass;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kWarps; ++i) {
      dsum += s.red_d[i];
      mass += s.red_u[i];
      pass += s.red_p[i];
    }
    s.pub_sum = dsum;
    s.pub_mass = mass;
    s.pub_pass = pass;
  }
  cluster.sync();
  double row_sum = 0;
  u64 row_mass = 0;
  uint32_t row_pass = 0;
  int row_first = p.vocab;
  for (unsigned r = 0; r < row.ranks; ++r) {
    const Shared* o = row.at(r);
    row_sum += o->pub_sum;
    row_mass += o->pub_mass;
    row_pass += o->pub_pass;
    row_first = min(row_first, o->pub_first);
  }

  // The cut: top_k first, then top_p of the mass that is left.
  Cut cut = {__float_as_uint(min_p), 0x7fffffff};
  u64 left = row_mass;
  if (cut_k && row.cut_at(kCount, static_cast<u64>(top_k), cut_p, min_p, row_pass, row_mass)) {
    cut = s.cut;
    left = s.cut_mass;
  }
  if (cut_p) {
    const double t = ceil(static_cast<double>(top_p) * static_cast<double>(left));
    const u64 target = t >= 1.0 ? static_cast<u64>(t) : 1ull;
    __syncthreads();  // s.cut and s.found_* of the first search have been read
    if (row.cut_at(kMass, target, true, min_p, row_pass, row_mass)) cut = s.cut;
  }

  // Kept mass and sum of every warp's run.
  u64 kept_mass = 0;
  float kept_sum = 0.f;
  for (int i = row.run0 + lane; i < row.run1; i += 32) {
    const float e = w[i];
    const uint32_t key = __float_as_uint(e);
    if (key > cut.key || (key == cut.key && row.first + i <= cut.index)) {
      kept_mass += mass_of(e);
      kept_sum += e;
    }
  }
  kept_mass = warp_sum(kept_mass);
  kept_sum = warp_sum(kept_sum);
  if (lane == 0) {
    s.pub_warp_mass[warp] = kept_mass;
    s.pub_warp_sum[warp] = kept_sum;
  }
  cluster.sync();
  u64 total = 0, before = 0;
  double sampling_sum = 0;
  for (unsigned r = 0; r < row.ranks; ++r) {
    const Shared* o = row.at(r);
    for (int i = 0; i < kWarps; ++i) {
      if (r == row.rank && i == warp) before = total;
      total += o->pub_warp_mass[i];
      sampling_sum += o->pub_warp_sum[i];
    }
  }
  const double at = floor(static_cast<double>(u > 0.f ? u : 0.f) * static_cast<double>(total));
  u64 t = static_cast<u64>(at);
  if (t >= total) t = total - 1;
  int token = -1;
  if (greedy) {
    if (row.rank == 0 && warp == 0) token = row_first;
  } else if (before <= t && t < before + kept_mass) {  // warp-uniform
    for (int base = row.run0; base < row.run1 && token < 0; base += 32) {
      const int i = base + lane;
      uint32_t q = 0;
      if (i < row.run1) {
        const float e = w[i];
        const uint32_t key = __float_as_uint(e);
        if (key > cut.key || (key == cut.key && row.first + i <= cut.index)) q = mass_of(e);
      }
      u64 sums = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += up;
      }
      const unsigned vote = __ballot_sync(0xffffffffu, before + sums > t);
      if (vote) token = row.first + base + __ffs(vote) - 1;
      before += __shfl_sync(0xffffffffu, sums, 31);
    }
  }
  if (token >= 0 && lane == 0) {
    const float l = no_nan(logit_f32<L>(logits[token]));
    const double x = m == INFINITY ? 0.0 : static_cast<double>(__fmul_rn(__fsub_rn(l, m), inv));
    p.tokens[b] = token;
    p.logprobs[b] = static_cast<float>(x - log(row_sum));
    p.sampling_logprobs[b] = static_cast<float>(x - log(sampling_sum));
  }
  cluster.sync();  // no CTA leaves while another may still read its shared memory
}

template <typename L>
int launch(const SampleParams& p, long long rows, int ranks, cudaStream_t stream) {
  // Head elements ahead of the first aligned one shift the slice by up to a vector.
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (static_cast<size_t>(p.slice) + 8) * 4;
  const cudaError_t err = cudaFuncSetAttribute(
      sample_kernel<L>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (err != cudaSuccess) return cuda_status(err, "sample_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, sample_kernel<L>, p), "sample_kernel launch");
}

}  // namespace

int launch_sample_tokens(const b200_sample_args* a, const void* logits, const float* uniforms,
                         const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, int64_t* tokens, float* logprobs,
                         float* sampling_logprobs, cudaStream_t stream) {
  if (a == nullptr) return set_error(B200_ERR_INVALID, "null descriptor");
  if (a->dtype != B200_F16 && a->dtype != B200_BF16 && a->dtype != B200_F32)
    return set_error(B200_ERR_UNSUPPORTED, "logits must be float16, bfloat16 or float32");
  if (a->rows < 0 || a->vocab <= 0) return set_error(B200_ERR_INVALID, "rows/vocab out of range");
  if (a->vocab > kMaxCluster * kMaxSlice)
    return set_error(B200_ERR_UNSUPPORTED, "vocabularies are limited to 376832 tokens");
  if (a->rows == 0) return B200_OK;
  if (a->rows > 0x7fffffffLL / kMaxCluster) return set_error(B200_ERR_UNSUPPORTED, "too many rows");
  if (!logits || !uniforms || !tokens || !logprobs || !sampling_logprobs)
    return set_error(B200_ERR_INVALID, "null tensor pointer");
  SampleParams p;
  p.logits = logits;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = a->temperature;
  p.top_k_all = a->top_k;
  p.top_p_all = a->top_p;
  p.min_p_all = a->min_p;
  p.tokens = reinterpret_cast<long long*>(tokens);
  p.logprobs = logprobs;
  p.sampling_logprobs = sampling_logprobs;
  p.stride = a->row_stride;
  p.vocab = a->vocab;
  int ranks = 1;
  while (ranks < kMaxCluster && ranks * 4096 < a->vocab) ranks *= 2;
  p.slice = static_cast<int>(ceil_div64(ceil_div64(a->vocab, ranks), 32) * 32);
  if (a->dtype == B200_F32) return launch<float>(p, a->rows, ranks, stream);
  if (a->dtype == B200_BF16) return launch<__nv_bfloat16>(p, a->rows, ranks, stream);
  return launch<__half>(p, a->rows, ranks, stream);
}

}  // namespace b200
