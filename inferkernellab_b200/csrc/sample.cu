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
// Layout.  A cluster of 1..8 CTAs owns a row and reads it from memory once; each
// CTA keeps its slice in shared memory as it came.  What the CTAs have to tell
// each other is stored into the others' shared memory before a cluster barrier
// and read locally after it.  Warps own runs of neighbouring tokens, so a prefix
// over warps is a prefix over indices.
//
// Nothing that is as long as the vocabulary is sorted.  Without filters the masses
// of the warps' runs name the run that holds the draw.  With filters few tokens
// matter, and the threads' own largest tokens (known from the search for m) say
// which: k of them above a bound prove that the first k tokens are above it, and
// a mass of top_p among them proves the same of the top_p prefix.  The tokens
// above that bound are gathered (kList at most) in one CTA, cut, and
// drawn from (few of them by counting what precedes each, more by sorting).  Where the
// bound leaves too many (a flat row, equal logits, a large
// top_k), the cut is found by histograms of counts and masses over the bits of w
// (w >= 0: they order like w), 1024 bins a level, until the bin's tokens fit the
// list or are all equal, and the draw takes another pass over the slice.
//
// Bound: latency.  A row goes through three cluster barriers (m; sums and bounds; the
// list), each 0.5 to 1 us, and the passes between them; a fourth, that every CTA of the
// cluster runs, ends while the first pass loads.  Measured (graph replay): one
// row of 128256 bf16 logits with top_p 11.6 us, 64 rows with mixed settings 53 us (a
// flat row that needs the exact search takes 37 us of it, any other 11 to 17), 256
// rows of 128257 32-bit logits with top_k 105 us, 1.25 TB/s: two slices of 64 KB share
// an SM, so that 37 rows are in flight.
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
constexpr int kList = 1024;      // tokens that are sorted
// List entries up to which counting beats sorting (16 rows: 18.9 us against 20.0 at
// 120 entries, 24.6 against 21.6 at 200).
constexpr int kCounted = 160;
// top_k up to which the threads' largest tokens bound the list (16 rows, top_k 300:
// 25.2 us against 33.8 by the exact search).
constexpr int kFewTokens = 512;
// Bins of the threads' largest tokens: 11 per unit of (m - l) / T, so that 255 of
// them span the weights above 2^-32; the last one holds everything below.
constexpr int kCoarse = 256;
constexpr float kCoarsePerUnit = 11.f;
// Bins of the exact search.
constexpr int kBins = 1024;
constexpr int kFirstShift = 18;                          // bits below 1/32 octave
constexpr uint32_t kFirstBase = (127u - 31u) << 5;       // key >> 18 of w = 2^-31
constexpr int kFirstBins = (127 << 5) - kFirstBase + 1;  // 993: the last one holds w = 1
constexpr int kMaxSlice = 46 * 1024;                     // tokens of a CTA
constexpr int kSharedSlice = 80 * 1024;                  // bytes of a slice of which two share an SM
constexpr float kLargest = 3.402823466e38f, kSmallest = 1.175494351e-38f;
constexpr float kLog2e = 1.4426950408889634f;
static_assert(kMaxSlice <= (1 << 16), "the 32-bit mass sums hold 2^16 tokens");
static_assert(kList <= 2 * kThreads, "two list entries per thread");
static_assert(kCoarse <= kThreads, "a thread per coarse bin");

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

struct Cut {  // kept: key > cut.key, or key == cut.key and index <= cut.index
  uint32_t key;
  int index;
  u64 mass;  // of the kept tokens
};

struct Shared {
  // Rank 0: gathered tokens, key << 32 | ~index, and their logits.  A CTA of the
  // cluster has kList / ranks places of its own.
  u64 list[kList];
  float list_logit[kList];
  // The exact search: a bin's mass is two 32-bit sums (low and high 16 bits; a CTA
  // holds at most 2^16 tokens), since 64-bit shared-memory atomics are loops.
  uint32_t count[kBins], low[kBins], high[kBins];
  // The threads' largest tokens: count, and mass in units of 2^-22.
  uint32_t coarse_count[kCoarse], coarse_mass[kCoarse];
  // Written by every CTA of the cluster, read here after the next cluster barrier.
  float max_of[kMaxCluster];
  double sum_of[kMaxCluster];
  int first_of[kMaxCluster], pass_of[kMaxCluster], listed_of[kMaxCluster];
  u64 warp_mass[kMaxCluster * kWarps];
  float warp_sum[kMaxCluster * kWarps];
  int warp_ties[kMaxCluster * kWarps];
  int listed[2];  // rank 0: list entries taken, by search
  Cut cut;
  // Of this CTA alone.
  int local_first, local_listed;
  float red_f[kWarps];
  double red_d[kWarps];
  int red_i[kWarps];
  u64 scan_mass[kWarps];
  uint32_t scan_count[kWarps];
  int found_bin;
  uint32_t found_count, before_count;
  u64 before_mass;
  int found;
};

constexpr int kSharedBytes = (static_cast<int>(sizeof(Shared)) + 15) / 16 * 16;
static_assert(kSharedBytes + kMaxSlice * 4 <= 227 * 1024, "shared memory of a CTA");

// 16 bytes of logits.
template <typename L>
struct Vec;

template <>
struct Vec<float> {
  static constexpr int kN = 4;
  float4 v;
  __device__ float get(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
  // NaN to -inf (the maximum of the two is the one that is a number); returns the largest.
  __device__ float clean() {
    v.x = fmaxf(v.x, -INFINITY);
    v.y = fmaxf(v.y, -INFINITY);
    v.z = fmaxf(v.z, -INFINITY);
    v.w = fmaxf(v.w, -INFINITY);
    return largest();
  }
  __device__ float largest() const { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
};

template <typename L, typename L2>
struct Vec16 {
  static constexpr int kN = 8;
  L2 v[4];
  __device__ float get(int i) const {
    return static_cast<float>(i % 2 ? v[i / 2].y : v[i / 2].x);
  }
  __device__ float clean() {
    L2 low;
    low.x = low.y = L(-INFINITY);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmax2(v[i], low);
    return largest();
  }
  __device__ float largest() const {
    const L2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(static_cast<float>(m.x), static_cast<float>(m.y));
  }
};

template <>
struct alignas(16) Vec<__half> : Vec16<__half, __half2> {};
template <>
struct alignas(16) Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {};

__device__ __forceinline__ uint32_t mass_of(float w) {
  return __float2uint_rn(__fmul_rn(w, 2147483648.0f));
}
__device__ __forceinline__ uint32_t mass_of_key(uint32_t key) {
  return mass_of(__uint_as_float(key));
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Inclusive prefix over the lanes of a warp.
template <typename V>
__device__ __forceinline__ V warp_prefix(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

enum Measure { kCount, kMass };  // what a cut is made on

template <typename L>
class Row {
 public:
  using V = Vec<L>;
  static constexpr int kN = V::kN;

  __device__ Row(const SampleParams& p, Shared& s, V* raw, cg::cluster_group cluster)
      : p(p), s(s), raw(raw), cluster(cluster), ranks(static_cast<int>(cluster.num_blocks())),
        rank(static_cast<int>(cluster.block_rank())), tid(threadIdx.x), warp(threadIdx.x >> 5),
        lane(threadIdx.x & 31) {}

  const SampleParams& p;
  Shared& s;
  V* raw;  // the slice, -inf past its end
  cg::cluster_group cluster;
  const int ranks, rank, tid, warp, lane;
  int origin;            // token of raw's first element
  int run0, run1;        // this warp's vectors
  float thread_max;      // largest logit of this thread's vectors
  float m, inv, min_p;   // largest logit of the row, 1 / T
  int searches = 0;

  __device__ Shared* at(int r) { return cluster.map_shared_rank(&s, r); }

  // ---------------------------------------------------------------- pass 1
  // The vector that starts `skip` elements into `a` and ends in `b`.
  __device__ static V shifted(const V& a, const V& b, int skip) {
    uint32_t w[8], out[4];
    memcpy(w, &a, 16);
    memcpy(w + 4, &b, 16);
    const int words = skip * static_cast<int>(sizeof(L)) / 4;
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = words & 1 ? w[i + 1] : w[i];
    const int bits = sizeof(L) == 2 ? (skip & 1) * 16 : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __funnelshift_r(w[i], w[i + 1], bits);
    V x;
    memcpy(&x, out, 16);
    return x;
  }

  // Reads the slice into shared memory; sets m.
  __device__ void load(const L* row) {
    const int first = min(rank * p.slice, p.vocab);
    const int n = min(p.slice, p.vocab - first);
    const L* src = row + first;
    const int vecs = (n + kN - 1) / kN;
    origin = first;
    const int run = ((vecs + kWarps - 1) / kWarps + 31) / 32 * 32;
    run0 = min(vecs, warp * run);
    run1 = min(vecs, run0 + run);
    // A row off the 16-byte grid is read as two neighbouring vectors and shifted,
    // so that a thread's tokens (and the rounding of its sum) do not depend on the
    // address; vectors that reach past the slice on either side by element.
    const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(src) / sizeof(L)) % kN);
    const V* vsrc = reinterpret_cast<const V*>(src - skip);
    const int whole0 = skip ? 1 : 0;
    const int whole1 = skip ? (n + skip) / kN - 1 : n / kN;
    thread_max = -INFINITY;
    constexpr int kBatch = 4;  // loads in flight of a thread
    for (int base = run0 + lane; base < run1; base += 32 * kBatch) {
      V x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int v = base + 32 * j;
        if (v >= whole0 && v < min(whole1, run1)) x[j] = vsrc[v];
      }
      if (skip) {
        V next[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int v = base + 32 * j;
          if (v >= whole0 && v < min(whole1, run1)) next[j] = vsrc[v + 1];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) x[j] = shifted(x[j], next[j], skip);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int v = base + 32 * j;
        if (v >= run1) break;
        if (v < whole0 || v >= whole1) {
          L e[kN];
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const int at = v * kN + i;
            e[i] = at < n ? src[at] : static_cast<L>(-INFINITY);
          }
          memcpy(&x[j], e, 16);
        }
        thread_max = fmaxf(thread_max, x[j].clean());
        raw[v] = x[j];
      }
    }
    m = thread_max;
    m = warp_max(m);
    if (lane == 0) s.red_f[warp] = m;
    __syncthreads();
    cluster_wait();  // of the arrival at entry: every CTA runs, its shared memory may be written
    if (warp == 0) {
      m = warp_max(s.red_f[lane % kWarps]);
      if (lane < ranks) at(lane)->max_of[rank] = m;
    }
    cluster.sync();
    m = warp_max(s.max_of[min(lane, ranks - 1)]);
  }

  __device__ float argument(float l) const {  // of the exponential
    return m == INFINITY ? (l == m ? 0.f : -INFINITY) : __fmul_rn(__fsub_rn(l, m), inv);
  }
  __device__ float weight(float l) const { return expf(argument(l)); }

  __device__ static int coarse_bin(float x) {
    return static_cast<int>(fminf(__fmul_rn(-x, kCoarsePerUnit), kCoarse - 1));
  }

  // f(token, logit) for this warp's tokens in the slice's vectors.
  template <typename F>
  __device__ void each(F&& f) {
#pragma unroll 2
    for (int v = run0 + lane; v < run1; v += 32) {
      const V x = raw[v];
#pragma unroll
      for (int i = 0; i < kN; ++i) f(origin + v * kN + i, x.get(i));
    }
  }

  // ---------------------------------------------------------------- pass 2
  __device__ void push_sum(float sum) {
    const double d = warp_sum(static_cast<double>(sum));
    if (lane == 0) s.red_d[warp] = d;
  }
  __device__ void push_block_sums(bool exact, bool first) {
    __syncthreads();
    if (tid < ranks) {
      double d = 0;
      for (int i = 0; i < kWarps; ++i) d += s.red_d[i];
      Shared* o = at(tid);
      o->sum_of[rank] = d;
      if (first) o->first_of[rank] = s.local_first;
      if (exact) {
        int pass = 0;
        for (int i = 0; i < kWarps; ++i) pass += s.red_i[i];
        // With min_p = 0 all tokens pass, and the padding after the slice would, too.
        o->pass_of[rank] = min_p > 0.f ? pass : max(0, min(p.slice, p.vocab - rank * p.slice));
      }
    }
  }
  // The sum of w alone.  The 2-ulp exponential is enough for a logarithm's sake.
  __device__ void sum_weights() {
    const float c = fminf(inv * kLog2e, kLargest);
    float sum = 0.f;
    each([&](int, float l) { sum += fast_exp2((l - m) * c); });
    push_sum(sum);
  }
  // The sum of w, and mass and number of the tokens that pass min_p, by warp.
  __device__ void sum_masses() {
    float sum = 0.f;
    u64 mass = 0;
    int pass = 0;
    if (m != INFINITY && min_p == 0.f) {  // the usual case, without the tests
      each([&](int, float l) {
        const float w = expf(__fmul_rn(__fsub_rn(l, m), inv));
        sum += w;
        mass += mass_of(w);
      });
    } else {
      each([&](int, float l) {
        const float w = weight(l);
        sum += w;
        if (w >= min_p) {
          mass += mass_of(w);
          ++pass;
        }
      });
    }
    push_sum(sum);
    mass = warp_sum(mass);
    pass = warp_sum(pass);
    if (lane == 0) s.red_i[warp] = pass;
    if (lane < ranks) at(lane)->warp_mass[rank * kWarps + warp] = mass;
  }
  __device__ void find_first_largest() {
    if (thread_max == m)
      each([&](int token, float l) {
        if (l == m) atomicMin(&s.local_first, token);
      });
  }

  // Mass of the first `warps` warps of the row (whole warps call it).
  __device__ u64 mass_before(int warps) const {
    u64 q = 0;
    for (int i = lane; i < warps; i += 32) q += s.warp_mass[i];
    return warp_sum(q);
  }
  __device__ u64 row_mass() const { return mass_before(ranks * kWarps); }
  __device__ double row_sum() const {
    double d = 0;
    for (int r = 0; r < ranks; ++r) d += s.sum_of[r];
    return d;
  }

  __device__ void add_coarse() {
    if (thread_max == -INFINITY) return;
    const float x = argument(thread_max);
    const float w = expf(x);
    if (!(w >= min_p)) return;
    const int bin = coarse_bin(x);
    atomicAdd(&s.coarse_count[bin], 1u);
    atomicAdd(&s.coarse_mass[bin], mass_of(w) >> 9);
  }

  // The first coarse bin at which the threads' largest tokens of the row reach
  // `target`, or -1.
  __device__ int coarse_bound(Measure measure, u64 target) {
    u64 c = 0;  // 8 CTAs x 512 threads x 2^22: 35 bits
    if (tid < kCoarse) {
      uint32_t part[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {  // every remote load in flight at once
        const Shared* o = at(min(r, ranks - 1));
        part[r] = measure == kCount ? o->coarse_count[tid] : o->coarse_mass[tid];
      }
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) c += r < ranks ? part[r] : 0;
    }
    u64 sum = warp_prefix(c, lane);
    if (lane == 31) s.scan_mass[warp] = sum;
    if (tid == 0) s.found = -1;
    __syncthreads();
    for (int i = 0; i < warp; ++i) sum += s.scan_mass[i];
    const u64 scale = measure == kCount ? 1 : 512;
    if (tid < kCoarse && sum * scale >= target && (sum - c) * scale < target) s.found = tid;
    __syncthreads();
    return s.found;
  }

  // Every token above coarse bin `bound` that passes min_p to rank 0's list; true
  // if they fit.  Has a cluster barrier.
  __device__ bool gather(int bound) {
    // A bound on l below the bin's edge by more than its rounding.
    const float edge = (bound + 1) / kCoarsePerUnit / inv;
    const float limit =
        bound >= kCoarse - 1 ? -kLargest : m - edge * 1.0001f - (fabsf(m) + 1e-30f) * 1e-6f;
    const int places = kList / ranks;
    if (thread_max >= limit) {
      Shared* home = at(0);
      for (int v = run0 + lane; v < run1; v += 32) {
        const V x = raw[v];
        if (x.largest() < limit) continue;
#pragma unroll 1
        for (int i = 0; i < kN; ++i) {
          const float l = reinterpret_cast<const L*>(raw + v)[i];
          if (l < limit) continue;
          const float w = weight(l);
          if (w < min_p || w == 0.f) continue;
          const int to = atomicAdd(&s.local_listed, 1);
          if (to < places) {
            home->list[rank * places + to] = entry(w, origin + v * kN + i);
            home->list_logit[rank * places + to] = l;
          }
        }
      }
    }
    __syncthreads();
    if (tid < ranks) at(tid)->listed_of[rank] = s.local_listed;
    cluster.sync();
    return warp_max(static_cast<float>(s.listed_of[min(lane, ranks - 1)])) <= places;
  }

  // Closes the gaps between the CTAs' parts of the list (rank 0); returns its length.
  __device__ int close_list() {
    const int places = kList / ranks;
    u64 e[2];
    float l[2];
    int to[2], n = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = tid + i * kThreads;
      n = 0;
      to[i] = -1;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < ranks) {
          const int at = from - r * places, of = s.listed_of[r];
          if (at >= 0 && at < of) to[i] = n + at;  // of <= places
          n += of;
        }
      if (to[i] >= 0) {
        e[i] = s.list[from];
        l[i] = s.list_logit[from];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (to[i] >= 0) {
        s.list[to[i]] = e[i];
        s.list_logit[to[i]] = l[i];
      }
    __syncthreads();
    return n;
  }

  __device__ static u64 entry(float w, int token) {
    return static_cast<u64>(__float_as_uint(w)) << 32 | static_cast<uint32_t>(~token);
  }

  // ------------------------------------------------------------- the list
  // One bitonic step of a lane's entry `x` of index `e` with the one j lanes away.
  __device__ static u64 exchanged(u64 x, int e, int k, int j) {
    const u64 y = __shfl_xor_sync(0xffffffffu, x, j);
    const bool take_larger = ((e & k) == 0) == ((e & j) == 0);
    return (y > x) == take_larger ? y : x;
  }

  // Sorts the first n list entries, largest first (rank 0; the rest up to the next
  // power of two is cleared).  Bitonic: a warp holds 64 neighbouring entries in
  // registers, so that only the steps over 64 and more go through shared memory.
  __device__ void sort_list(int n) {
    int size = 64;
    while (size < n) size *= 2;
    const bool mine = warp * 64 < size;
    const int ea = warp * 64 + lane, eb = ea + 32;
    u64 a = mine && ea < n ? s.list[ea] : 0, b = mine && eb < n ? s.list[eb] : 0;
    for (int k = 2; k <= size; k *= 2) {
      if (k > 64) {
        __syncthreads();
        if (mine) {
          s.list[ea] = a;
          s.list[eb] = b;
        }
        for (int j = k / 2; j >= 64; j /= 2) {
          __syncthreads();
          if (tid < size / 2) {
            const int p0 = 2 * tid - (tid & (j - 1)), p1 = p0 + j;
            const u64 x = s.list[p0], y = s.list[p1];
            if ((x < y) == ((p0 & k) == 0)) {
              s.list[p0] = y;
              s.list[p1] = x;
            }
          }
        }
        __syncthreads();
        if (mine) {
          a = s.list[ea];
          b = s.list[eb];
        }
      }
      if (!mine) continue;
      if (k >= 64 && (a < b) == ((ea & k) == 0)) {  // 32 apart: both in this lane
        const u64 x = a;
        a = b;
        b = x;
      }
      for (int j = min(k, 32) / 2; j > 0; j /= 2) {
        a = exchanged(a, ea, k, j);
        b = exchanged(b, eb, k, j);
      }
    }
    __syncthreads();
    if (mine) {
      s.list[ea] = a;
      s.list[eb] = b;
    }
    __syncthreads();
  }

  // The position among the first n list entries at which the running measure,
  // on top of `before`, reaches target (n: it does not); *sum gets the mass of
  // the entries up to and with it.  key_shift: where an entry holds its key.
  __device__ int list_position(int n, int key_shift, Measure measure, u64 before, u64 target,
                               u64 before_mass, u64* sum) {
    u64 q[2], c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * tid + i;
      q[i] = at < n ? mass_of_key(static_cast<uint32_t>(s.list[at] >> key_shift)) : 0;
      c[i] = measure == kMass ? q[i] : (at < n ? 1 : 0);
    }
    u64 mass = warp_prefix(q[0] + q[1], lane);
    if (lane == 31) s.scan_mass[warp] = mass;
    if (tid == 0) s.found = n;
    __syncthreads();
    for (int i = 0; i < warp; ++i) mass += s.scan_mass[i];
    mass -= q[0] + q[1];  // before this thread
    u64 run = before + (measure == kMass ? mass : static_cast<u64>(min(n, 2 * tid)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mass += q[i];
      if (run < target && run + c[i] >= target) {
        s.found = 2 * tid + i;
        s.before_mass = before_mass + mass;
      }
      run += c[i];
    }
    __syncthreads();
    const int found = s.found;
    if (sum && found < n) *sum = s.before_mass;
    __syncthreads();
    return found;
  }

  __device__ u64 list_mass(int n) {
    u64 q = 0;
    for (int i = tid; i < n; i += kThreads) q += mass_of_key(static_cast<uint32_t>(s.list[i] >> 32));
    q = warp_sum(q);
    if (lane == 0) s.scan_mass[warp] = q;
    __syncthreads();
    q = 0;
    for (int i = 0; i < kWarps; ++i) q += s.scan_mass[i];
    __syncthreads();
    return q;
  }

  // Barrier of the first `warps` warps, and a sum over their threads.
  __device__ void sync_warps(int warps) {
    if (warps == 1)
      __syncwarp();
    else
      named_bar_sync(1, warps * 32);
  }
  template <typename T>
  __device__ T sum_over(int warps, T v, T* red) {
    v = warp_sum(v);
    if (warps == 1) return v;
    if (lane == 0) red[warp] = v;
    sync_warps(warps);
    v = warp_sum(lane < warps ? red[lane] : T(0));
    sync_warps(warps);
    return v;
  }

  // The cut and the draw among the first n list entries (rank 0), by counting for
  // each entry what precedes it; only the warps that hold entries take part.
  template <typename F>
  __device__ void finish(int n, int top_k, bool cut_p, bool of_list, F&& top_p_target, u64 mass,
                         bool greedy, float u, long long b, double sum) {
    const int warps = (n + 31) / 32;
    if (warp >= warps) return;
    const u64 mine = tid < n ? s.list[tid] : 0;
    const uint32_t key = static_cast<uint32_t>(mine >> 32);
    const uint32_t q = mass_of_key(key);
    int rank_of = 0;
    u64 before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 o = s.list[j];
      const uint32_t oq = mass_of_key(static_cast<uint32_t>(o >> 32));
      rank_of += o > mine;
      before += o > mine ? oq : 0;
    }
    bool kept = tid < n && rank_of < top_k;
    if (cut_p) {
      if (of_list) mass = sum_over(warps, static_cast<u64>(kept ? q : 0), s.scan_mass);
      kept = kept && before < top_p_target(mass);
    }
    const double kept_sum =
        sum_over(warps, static_cast<double>(kept ? __uint_as_float(key) : 0.f), s.red_d);
    if (greedy) {  // the first largest logit, which is always kept
      if (tid == 0) write(b, first_largest(), m, sum, kept_sum);
      return;
    }
    const u64 t = draw_target(u, sum_over(warps, static_cast<u64>(kept ? q : 0), s.scan_mass));
    // Kept entries alone, then what precedes mine in order of index (~index falls).
    sync_warps(warps);
    if (tid < n && !kept) s.list[tid] = 0;
    sync_warps(warps);
    before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 o = s.list[j];
      const uint32_t oq = mass_of_key(static_cast<uint32_t>(o >> 32));
      before += static_cast<uint32_t>(o) > static_cast<uint32_t>(mine) ? oq : 0;
    }
    if (kept && before <= t && t < before + q)
      write(b, static_cast<int>(~static_cast<uint32_t>(mine)), s.list_logit[tid], sum, kept_sum);
  }

  // The same by sorting, where counting would take longer.
  template <typename F>
  __device__ void finish_sorted(int n, int top_k, bool cut_p, bool of_list, F&& top_p_target,
                                u64 mass, bool greedy, float u, long long b, const L* logits,
                                double sum) {
    sort_list(n);
    int kept = min(n, top_k);
    if (cut_p) {
      if (of_list) mass = list_mass(kept);
      const int pos = list_position(kept, 32, kMass, 0, top_p_target(mass), 0, nullptr);
      kept = min(kept, pos + 1);
    }
    double kept_sum = 0;
    u64 e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = tid + i * kThreads;
      e[i] = at < kept ? s.list[at] : 0;
      kept_sum += __uint_as_float(static_cast<uint32_t>(e[i] >> 32));
    }
    kept_sum = sum_over(kWarps, kept_sum, s.red_d);
    if (greedy) {
      if (tid == 0) write(b, first_largest(), m, sum, kept_sum);
      return;
    }
    const u64 total = list_mass(kept);
    // The kept tokens by index: ~index above the key.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = tid + i * kThreads;
      if (at < kept) s.list[at] = e[i] << 32 | e[i] >> 32;
    }
    __syncthreads();
    sort_list(kept);
    const int pos = list_position(kept, 0, kMass, 0, draw_target(u, total) + 1, 0, nullptr);
    if (tid == 0) {
      const int token = static_cast<int>(~static_cast<uint32_t>(s.list[pos] >> 32));
      write(b, token, fmaxf(static_cast<float>(logits[token]), -INFINITY), sum, kept_sum);
    }
  }

  __device__ int first_largest() const {
    int first = p.vocab;
    for (int r = 0; r < ranks; ++r) first = min(first, s.first_of[r]);
    return first;
  }

  // --------------------------------------------------------- exact search
  __device__ void clear_histogram() {
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0;
    __syncthreads();
  }
  __device__ void add_to_bin(int bin, uint32_t q) {
    atomicAdd(&s.count[bin], 1u);
    atomicAdd(&s.low[bin], q & 0xffffu);
    if (q >> 16) atomicAdd(&s.high[bin], q >> 16);
  }

  // The bin of the row's histogram in which `target` is reached, counted from the
  // last bin down, on top of `count0` / `mass0` above the whole histogram; bin 0
  // of the first level is what the row's totals leave.  Sets s.found_bin (-1: the
  // row has less than target), found_count (of the bin) and before_count /
  // before_mass (above it).
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
        uint32_t part[3][kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {  // every remote load in flight at once
          const Shared* o = at(min(r, ranks - 1));
          part[0][r] = o->count[bin];
          part[1][r] = o->low[bin];
          part[2][r] = o->high[bin];
        }
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < ranks) {
            c += part[0][r];
            q += part[1][r] + (static_cast<u64>(part[2][r]) << 16);
          }
      }
      uint32_t ci = warp_prefix(c, lane);
      u64 qi = warp_prefix(q, lane);
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
      const uint32_t before_c = run_count + ci - c;
      const u64 before_q = run_mass + qi - q;
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
  // one whose inclusive measure reaches it, into s.cut.  False if all tokens that
  // pass min_p together have less.
  __device__ bool cut_at(Measure measure, u64 target, uint32_t row_count, u64 row_mass) {
    clear_histogram();
    each([&](int, float l) {
      const float w = weight(l);
      const uint32_t hi = __float_as_uint(w) >> kFirstShift;
      if (hi > kFirstBase && w >= min_p) add_to_bin(hi - kFirstBase, mass_of(w));
    });
    cluster.sync();
    find_bin(kFirstBins, measure, target, 0, 0, true, row_count, row_mass);
    cluster.sync();  // the histograms may be cleared again
    if (s.found_bin < 0) return false;
    uint32_t lo = s.found_bin == 0 ? 0u : (kFirstBase + s.found_bin) << kFirstShift;
    uint32_t size = s.found_bin == 0 ? (kFirstBase + 1) << kFirstShift : 1u << kFirstShift;
    while (s.found_count > kList && size > 1) {
      int shift = 0;  // 1024 bins or fewer over [lo, lo + size)
      while (((size - 1) >> shift) >= kBins) ++shift;
      const int bins = static_cast<int>((size - 1) >> shift) + 1;
      const uint32_t before_count = s.before_count;
      const u64 before_mass = s.before_mass;
      clear_histogram();
      each_in(lo, size, [&](int, uint32_t key) {
        add_to_bin(static_cast<int>((key - lo) >> shift), mass_of_key(key));
      });
      cluster.sync();
      // The totals above are exact, so one of these bins holds the target.
      find_bin(bins, measure, target, before_count, before_mass, false, 0, 0);
      cluster.sync();
      lo += static_cast<uint32_t>(s.found_bin) << shift;
      size = 1u << shift;
    }
    if (s.found_count <= kList)
      resolve_listed(measure, target, lo, size);
    else
      resolve_ties(measure, target, lo);
    return true;
  }

  // A logit that is surely below (side -1) or above (1) those of weight `key`: past
  // it by more than the rounding of exp and of its argument.
  __device__ float logit_near(uint32_t key, float side) const {
    const float w = __uint_as_float(key);
    if (m == INFINITY || w < 1e-37f) return side < 0.f ? -INFINITY : INFINITY;
    const float x = logf(w) / inv;
    return m + x + side * (1e-4f * fabsf(x) + 1e-4f / inv + 1e-6f * fabsf(m));
  }

  // f(token, key) for the tokens that pass min_p with keys in [lo, lo + size).
  template <typename F>
  __device__ void each_in(uint32_t lo, uint32_t size, F&& f) {
    const float low = logit_near(lo, -1.f), high = logit_near(lo + size, 1.f);
    each([&](int token, float l) {
      if (l < low || l > high) return;
      const float w = weight(l);
      const uint32_t key = __float_as_uint(w);
      if (key - lo < size && w >= min_p && in_slice(token)) f(token, key);
    });
  }
  __device__ bool in_slice(int token) const {  // false for the padding after it
    return token < min(p.vocab, (rank + 1) * p.slice);
  }

  // At most kList tokens with keys in [lo, lo + size): sorted by rank 0.
  __device__ void resolve_listed(Measure measure, u64 target, uint32_t lo, uint32_t size) {
    const int slot = searches;
    const u64 before_mass = s.before_mass;
    const u64 before = measure == kCount ? s.before_count : before_mass;
    Shared* home = at(0);
    each_in(lo, size, [&](int token, uint32_t key) {
      const int to = atomicAdd(&home->listed[slot], 1);
      if (to < kList) home->list[to] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~token);
    });
    cluster.sync();
    if (rank == 0) {
      const int n = min(s.listed[slot], kList);
      sort_list(n);
      Cut cut = {0, 0x7fffffff, 0};
      const int pos = list_position(n, 32, measure, before, target, before_mass, &cut.mass);
      if (pos < n) {
        cut.key = static_cast<uint32_t>(s.list[pos] >> 32);
        cut.index = static_cast<int>(~static_cast<uint32_t>(s.list[pos]));
      }
      if (tid < ranks) at(tid)->cut = cut;
    }
    cluster.sync();
  }

  // More than kList tokens of one and the same weight: the cut is the r-th of them
  // in order of index.
  __device__ void resolve_ties(Measure measure, u64 target, uint32_t key) {
    const uint32_t q = mass_of_key(key);
    const u64 r = measure == kCount ? target - s.before_count
                                    : (target - s.before_mass + q - 1) / max(q, 1u);
    const Cut found = {key, 0, s.before_mass + r * q};
    int ties = 0;
    each_in(key, 1, [&](int, uint32_t) { ++ties; });
    ties = warp_sum(ties);
    if (lane < ranks) at(lane)->warp_ties[rank * kWarps + warp] = ties;
    cluster.sync();
    u64 before = 0;
    for (int i = 0; i < rank * kWarps + warp; ++i) before += s.warp_ties[i];
    if (before < r && r <= before + ties) {  // warp-uniform: the r-th is in this run
      walk(before, [&](int token, float l) {
        const float w = weight(l);
        return static_cast<u64>(__float_as_uint(w) == key && w >= min_p && in_slice(token));
      }, r - 1, [&](int token, float) {
        Cut cut = found;
        cut.index = token;
        for (int o = 0; o < ranks; ++o) at(o)->cut = cut;
      });
    }
    cluster.sync();
  }

  // Walks this warp's run in order of index, adding value(token, logit) to
  // `running`; done(token, logit) is called by one lane for the first token that takes it
  // past t.
  template <typename F, typename G>
  __device__ void walk(u64 running, F&& value, u64 t, G&& done) {
    for (int v = run0; v < run1; v += 32) {
      const bool live = v + lane < run1;
      u64 q[kN], sum = 0;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        q[i] = live ? value(origin + (v + lane) * kN + i, raw[v + lane].get(i)) : 0;
        sum += q[i];
      }
      const u64 with = running + warp_prefix(sum, lane);
      const unsigned vote = __ballot_sync(0xffffffffu, with > t);
      if (vote) {
        if (lane == __ffs(vote) - 1) {
          u64 before = with - sum;
          int token = 0;
          float l = 0.f;
          bool open = true;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            before += q[i];
            if (open && before > t) {
              token = origin + (v + lane) * kN + i;
              l = raw[v + lane].get(i);
              open = false;
            }
          }
          done(token, l);
        }
        return;
      }
      running = __shfl_sync(0xffffffffu, with, 31);
    }
  }

  // ------------------------------------------------------------- the draw
  __device__ static u64 draw_target(float u, u64 total) {
    // u outside [0, 1) is taken as the nearest end
    const double at = floor(static_cast<double>(u > 0.f ? u : 0.f) * static_cast<double>(total));
    const u64 t = static_cast<u64>(at);
    return t < total ? t : total - 1;
  }

  // One thread of the cluster writes the row's results; sums are at least 1 (w of
  // the largest), and what they are above it keeps its digits.
  __device__ void write(long long b, int token, float l, double sum, double kept) {
    const float x = argument(l);
    p.tokens[b] = token;
    p.logprobs[b] = x - log1pf(static_cast<float>(sum - 1.0));
    p.sampling_logprobs[b] = x - log1pf(static_cast<float>(kept - 1.0));
  }

  // The token at mass t of the row, whose warps' masses are in place.
  template <typename F>
  __device__ void draw(float u, F&& value, long long b, double sum, double kept) {
    const u64 t = draw_target(u, row_mass());
    const int me = rank * kWarps + warp;
    const u64 before = mass_before(me);
    if (before <= t && t < before + s.warp_mass[me])  // warp-uniform
      walk(before, value, t, [&](int token, float l) { write(b, token, l, sum, kept); });
  }
};

template <typename L>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  Row<L> row(p, s, reinterpret_cast<Vec<L>*>(smem + kSharedBytes), cluster);
  const int tid = row.tid, warp = row.warp, lane = row.lane, rank = row.rank;
  const long long b = blockIdx.x / row.ranks;
  cluster_arrive_relaxed();  // Row::load waits for it
  if (tid < kCoarse) s.coarse_count[tid] = s.coarse_mass[tid] = 0;
  if (tid == 0) {
    s.listed[0] = s.listed[1] = s.local_listed = 0;
    s.local_first = p.vocab;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const L* logits = reinterpret_cast<const L*>(p.logits) + b * p.stride;
  const float temperature = p.temperature ? p.temperature[b] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float u = p.uniforms[b];
  const bool greedy = !(temperature > 0.f);
  const bool cut_k = top_k > 0 && top_k < p.vocab;
  const bool cut_p = top_p < 1.f;
  row.min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  // Finite and not zero, so that 0 and -inf keep their meaning when multiplied.
  row.inv = greedy ? 1.f : fmaxf(fminf(__fdiv_rn(1.f, temperature), kLargest), kSmallest);
  const bool filtered = cut_k || cut_p || row.min_p > 0.f;

  row.load(logits);
  if (row.m == -INFINITY) {  // cluster-uniform: nothing in this row can be drawn
    if (rank == 0 && tid == 0) {
      p.tokens[b] = -1;
      p.logprobs[b] = -INFINITY;
      p.sampling_logprobs[b] = -INFINITY;
    }
    return;
  }
  // Whether the threads' largest tokens can bound what has to be gathered.
  const bool few = cut_k && top_k <= kFewTokens;
  const bool listing = filtered && row.m != INFINITY && (few || !cut_k);
  // The masses of all tokens: to draw from, or for top_p of them.
  bool exact = filtered ? !listing || (cut_p && !few) : !greedy || row.m == INFINITY;
  if (listing && (few || cut_p)) row.add_coarse();
  if (exact)
    row.sum_masses();
  else
    row.sum_weights();
  if (greedy) row.find_first_largest();
  row.push_block_sums(exact, greedy);
  cluster.sync();
  const double sum = row.row_sum();
  if (!filtered) {
    if (!greedy)
      row.draw(u, [&](int, float l) { return static_cast<u64>(mass_of(row.weight(l))); }, b, sum,
               sum);
    else if (rank == 0 && tid == 0)
      row.write(b, row.first_largest(), row.m, sum, sum);
    return;
  }

  auto top_p_target = [&](u64 mass) {
    const double t = ceil(static_cast<double>(top_p) * static_cast<double>(mass));
    return t >= 1.0 ? static_cast<u64>(t) : 1ull;
  };
  if (listing) {
    int bound = kCoarse - 1;  // every token
    if (p.vocab > kList) {
      if (few) {
        bound = row.coarse_bound(kCount, static_cast<u64>(top_k));
        if (bound < 0) bound = kCoarse - 1;
      } else if (cut_p) {
        bound = row.coarse_bound(kMass, top_p_target(row.row_mass()));
      } else {
        bound = min(kCoarse - 1, Row<L>::coarse_bin(logf(row.min_p)) + 1);
      }
    }
    if (bound >= 0 && row.gather(bound)) {  // cluster-uniform
      if (rank != 0) return;
      const int n = row.close_list();
      const u64 mass = few || !cut_p ? 0 : row.row_mass();
      if (n <= kCounted) {
        row.finish(n, cut_k ? top_k : n, cut_p, few, top_p_target, mass, greedy, u, b, sum);
      } else {
        row.finish_sorted(n, cut_k ? top_k : n, cut_p, few, top_p_target, mass, greedy, u, b,
                          logits, sum);
      }
      return;
    }
  }

  // Too many tokens for the list: exact cuts, then a draw over the slices.
  if (!exact) {
    __syncthreads();
    row.sum_masses();
    row.push_block_sums(true, false);
    cluster.sync();
  }
  uint32_t pass = 0;
  for (int r = 0; r < row.ranks; ++r) pass += s.pass_of[r];
  const u64 mass = row.row_mass();
  Cut cut = {__float_as_uint(row.min_p), 0x7fffffff, mass};
  if (cut_k && row.cut_at(kCount, static_cast<u64>(top_k), pass, mass)) cut = s.cut;
  if (cut_p) {
    ++row.searches;
    __syncthreads();  // s.cut has been read
    if (row.cut_at(kMass, top_p_target(cut.mass), pass, mass)) cut = s.cut;
  }
  const float low = row.logit_near(cut.key, -1.f);
  auto kept_weight = [&](int token, float l) {
    if (l < low) return 0.f;
    const float w = row.weight(l);
    const uint32_t key = __float_as_uint(w);
    return key > cut.key || (key == cut.key && token <= cut.index) ? w : 0.f;
  };
  u64 kept_mass = 0;
  float kept_part = 0.f;
  row.each([&](int token, float l) {
    const float w = kept_weight(token, l);
    kept_mass += mass_of(w);
    kept_part += w;
  });
  kept_mass = warp_sum(kept_mass);
  kept_part = warp_sum(kept_part);
  cluster.sync();  // every warp_mass has been read
  if (lane < row.ranks) {
    Shared* o = row.at(lane);
    o->warp_mass[rank * kWarps + warp] = kept_mass;
    o->warp_sum[rank * kWarps + warp] = kept_part;
  }
  cluster.sync();
  double kept = 0;
  for (int i = lane; i < row.ranks * kWarps; i += 32) kept += s.warp_sum[i];
  kept = warp_sum(kept);
  if (greedy) {
    if (rank == 0 && tid == 0) row.write(b, row.first_largest(), row.m, sum, kept);
    return;
  }
  row.draw(u, [&](int token, float l) { return static_cast<u64>(mass_of(kept_weight(token, l))); },
           b, sum, kept);
}

template <typename L>
int launch(const SampleParams& p, long long rows, int ranks, cudaStream_t stream) {
  const size_t smem = kSharedBytes + static_cast<size_t>(p.slice) * sizeof(L);  // slice: whole vectors
  // The limit belongs to the function, not to the call: always the largest, so that
  // calls of other host threads never lower it ahead of this launch.
  const cudaError_t err =
      cudaFuncSetAttribute(sample_kernel<L>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           kSharedBytes + kMaxSlice * static_cast<int>(sizeof(L)));
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
  // CTAs per row: enough that two slices share an SM, then as many as 4096 tokens
  // each and the SMs' two CTAs allow.  256 rows of 32000: 30.7 us with 2, 70.4 with 8;
  // one row of 32000: 13.4 with 2, 10.1 with 8.
  DeviceInfo info;
  const int rc = current_device_info(&info);
  if (rc != B200_OK) return rc;
  const int64_t bytes = a->dtype == B200_F32 ? 4 : 2;
  int ranks = 1;
  while (ranks < kMaxCluster && ceil_div64(a->vocab, ranks) * bytes > kSharedSlice) ranks *= 2;
  while (ranks < kMaxCluster && ranks * 4096 < a->vocab && a->rows * ranks <= info.num_sms)
    ranks *= 2;
  p.slice = static_cast<int>(ceil_div64(ceil_div64(a->vocab, ranks), 32) * 32);
  if (a->dtype == B200_F32) return launch<float>(p, a->rows, ranks, stream);
  if (a->dtype == B200_BF16) return launch<__nv_bfloat16>(p, a->rows, ranks, stream);
  return launch<__half>(p, a->rows, ranks, stream);
}

}  // namespace b200
