// Drawing tokens from logits with temperature, top-k, top-p and min-p.
//
// Mathematics. Tokens are ordered by logit, larger first, equal ones by index.
// With M the row's largest logit and T its temperature, w_i = exp((x_i - M) / T).
// Kept are the first tokens of the order: at most top_k of them, those with
// w >= min_p, and of these the ones with less than top_p of their mass before
// them. The token for a given u is the first index whose kept mass so far is
// above u times all kept mass.
//
// Whether a token is kept, and which one u falls on, are decisions next to a
// border: with 2^17 tokens fp32 sums would miss one in about a hundred. So a
// weight is a 64-bit integer, 2^-t (to 2^-30 of itself, see Weigh) times 2^S with S
// as large as the sum over the vocabulary allows (45 bits for 2^17 tokens): errors
// of single tokens' weights next to a border matter, not those of the sum, whose
// parts' errors average out. Sums of integers do not depend on their order, so
// neither does a result.
//
// A row is worked on by a cluster of CTAs, each with a run of the vocabulary (kept
// in shared memory) and in it a run for each warp.
// - top_k up to kMostListed: the k-th largest of the threads' own maxima bounds
//   the k-th logit from below. What is at or above it, little more than k tokens,
//   is gathered in one CTA, sorted, and cut and drawn from there.
// - otherwise the border token of a cut is found in a histogram of 2048 bins of
//   log2 w (counts for top-k, masses for top-p), then among the tokens of one
//   bin: by rank if they are few, by histograms of their order's key (logit and
//   index, 64 bits) until they are.
#include <cooperative_groups.h>
#include <float.h>
#include <limits.h>

#include <type_traits>

#include "cache8.cuh"

using cxs_host::set_error;

namespace {

using cxs::cache8::to_float;
namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr float kCountBins = 32;     // bins of counts for an octave of the weight
constexpr int kPowers = 512;         // of two, in a table
constexpr int kFew = 512;            // tokens whose ranks are counted one by one
constexpr int kList = kThreads;      // tokens that are gathered for a small top_k
constexpr int kMostListed = 384;     // largest such top_k
constexpr int kMostCtas = 16;        // of a cluster
constexpr int kBlocks = 128;         // parts of a warp's run whose kept mass is kept
constexpr int kSliceBytes = 72 << 10;  // of a CTA's run in shared memory: two CTAs fit an SM
constexpr float kInf = INFINITY;
constexpr double kLog2e = 1.4426950408889634;

// Order's key: larger comes first.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 as 0)
  const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)k << 32 | (0xffffffffu - (uint32_t)index);
}
// Its logit and index.
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

// 2^(32 - i / kPowers), rounded (below 2^32 for i = 0), by Taylor's polynomial: the
// exponent is at most ln 2, the next term below 2^-48.
__device__ __forceinline__ uint32_t power_of(int i) {
  const double g = i * (-0.6931471805599453 / kPowers);
  double p = 1.0;
#pragma unroll
  for (int k = 13; k > 0; --k) p = fma(p, g * (1.0 / k), 1.0);
  return (uint32_t)fmin(p * 4294967296.0 + 0.5, 4294967295.0);
}

struct Settings {  // of a row
  float temperature, top_p, min_p;
  int top_k;
};

// A sum of 64 bits in two words of shared memory (an atomic addition of 64 bits
// there is a loop).
struct Wide {
  uint32_t* low;
  uint32_t* high;
  __device__ __forceinline__ void add(int i, unsigned long long v) const {
    const uint32_t lo = (uint32_t)v, old = atomicAdd(low + i, lo);
    const uint32_t hi = (uint32_t)(v >> 32) + (old + lo < lo);
    if (hi) atomicAdd(high + i, hi);
  }
  __device__ __forceinline__ unsigned long long get(int i) const {
    return (unsigned long long)high[i] << 32 | low[i];
  }
};

struct Found {  // a bin: its count, what is before it, the sum of all bins
  int bin, count;
  unsigned long long before, all;
};

struct Shared {
  union {
    struct {
      uint32_t counts[kBins];
      union {
        uint32_t masses[2][kBins];             // low and high words
        uint64_t gathered[kList];
      };
    };
    unsigned long long blocks[kWarps][kBlocks];  // kept mass of parts of a warp's run
  };
  union {
    struct {
      uint64_t list[kFew];                     // this CTA's few
      uint64_t all[kFew];                      // the cluster's
      unsigned long long weights[kFew];
    };
    struct {                                   // (of several CTAs) the cluster's bins,
      uint32_t part_masses[2][kBins / 2];      // this CTA's part of them
      uint32_t part_counts[kBins / 2];
    };
  };
  unsigned long long sums[kWarps];             // of a scan
  unsigned long long spans[kWarps];            // kept mass before each warp's tokens
  float top, bound;                            // read by the cluster: largest logit, a bound
                                               // below which the CTA has no first top_k,
  uint64_t bounds[2];                          // keys of a bin,
  unsigned long long mass;                     // kept mass of this CTA,
  float2 odds;                                 // its Odds,
  int listed;                                  // and what it has listed;
  int wanted;                                  // (first CTA's) how many it was sent
  unsigned long long part;                     // sum of this CTA's part of the bins
  Found found;
  uint64_t cut;
  float warp_totals[kWarps];
  float2 warp_odds[kWarps];
  uint32_t powers[kPowers];                    // 2^(32 - i / kPowers)
};

// Sum of v over the threads before this one; *total: over all.
__device__ __forceinline__ unsigned long long block_scan(Shared& s, unsigned long long v,
                                                         unsigned long long* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  unsigned long long sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();
  if (lane == 31) s.sums[warp] = sum;
  __syncthreads();
  unsigned long long all = lane < kWarps ? s.sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, kWarps - 1);
  const unsigned long long before = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);
  return sum - v + (warp > 0 ? before : 0);
}

// The sum of exp(x - M): x how many tokens have M, y of the others. (Apart, so
// that the log-probability of a token that takes nearly all of it keeps its bits.)
using Odds = float2;
__device__ __forceinline__ Odds block_sum(Shared& s, Odds v) {
  for (int o = 16; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.warp_odds[threadIdx.x / 32] = v;
  __syncthreads();
  v = make_float2(0.f, 0.f);
  for (int w = 0; w < kWarps; ++w) v.x += s.warp_odds[w].x, v.y += s.warp_odds[w].y;
  return v;
}
__device__ __forceinline__ float log_of(Odds v) {
  return v.x == 1.f ? log1pf(v.y) : logf(v.x + v.y);
}

// This CTA's part of a row, in 16-byte vectors (those of the row's memory: a row
// may begin inside one).
template <typename T>
struct Row {
  static constexpr int kVector = 16 / sizeof(T);
  const T* base;       // vector 0, or (kept) where vector `first` is in shared memory
  bool kept;
  int skip;            // values of vector 0 before the row
  int vocab;
  int first, count;    // the CTA's vectors
  int each;            // of them, a warp's

  __device__ __forceinline__ Row(const T* values, int vocab_, int rank, int ctas) {
    vocab = vocab_;
    kept = false;
    skip = (int)((uintptr_t)values % 16 / sizeof(T));
    base = values - skip;
    const int vectors = (int)(((long long)vocab + skip + kVector - 1) / kVector);
    const int part = (vectors + ctas - 1) / ctas;
    first = min(part * rank, vectors);
    count = min(part, vectors - first);
    each = (count + kWarps - 1) / kWarps;
  }
  __device__ __forceinline__ int begin(int warp) const { return min(each * warp, count); }
  __device__ __forceinline__ int index(int v, int e) const { return (first + v) * kVector + e - skip; }
  // Vector v of the CTA's; values that are not the row's: -infinity.
  __device__ __forceinline__ uint4 load(int v) const {
    if (kept) return *reinterpret_cast<const uint4*>(base + v * kVector);
    const int i = index(v, 0);
    const T* const from = base + (long long)(first + v) * kVector;
    if (i >= 0 && i + kVector <= vocab) return *reinterpret_cast<const uint4*>(from);
    alignas(16) T x[kVector];
#pragma unroll
    for (int e = 0; e < kVector; ++e)
      x[e] = i + e >= 0 && i + e < vocab ? from[e] : cxs::cache8::from_float<T>(-kInf);
    return *reinterpret_cast<const uint4*>(x);
  }
  // NaN as -infinity, in all values of a vector.
  static __device__ __forceinline__ uint4 without_nan(uint4 w) {
    auto two = [](uint32_t x) {
      if constexpr (sizeof(T) == 4) return __float_as_uint(fmaxf(__uint_as_float(x), -kInf));
      else return bits_of(larger(pair_of(x), pair_of(lowest())));
    };
    return make_uint4(two(w.x), two(w.y), two(w.z), two(w.w));
  }
  // The larger ones of two vectors' values, NaN counting as nothing.
  static __device__ __forceinline__ uint4 larger_of(uint4 a, uint4 b) {
    auto two = [](uint32_t x, uint32_t y) {
      if constexpr (sizeof(T) == 4)
        return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
      else return bits_of(larger(pair_of(x), pair_of(y)));
    };
    return make_uint4(two(a.x, b.x), two(a.y, b.y), two(a.z, b.z), two(a.w, b.w));
  }
  static __device__ __forceinline__ uint32_t lowest() {  // -infinity, one or two
    return sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  }
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  static __device__ __forceinline__ Pair pair_of(uint32_t x) { return *reinterpret_cast<Pair*>(&x); }
  static __device__ __forceinline__ uint32_t bits_of(Pair x) { return *reinterpret_cast<uint32_t*>(&x); }
  static __device__ __forceinline__ Pair larger(Pair a, Pair b) { return __hmax2(a, b); }
  static __device__ __forceinline__ void unpack(uint4 w, float (&x)[kVector]) {
    alignas(16) T y[kVector];
    *reinterpret_cast<uint4*>(y) = w;
#pragma unroll
    for (int e = 0; e < kVector; ++e) x[e] = to_float(y[e]);
  }
  // f(logit, index) for this warp's tokens; the next vector is on its way meanwhile.
  // Only four bytes' copies of f: what runs once in a launch runs from a cold
  // instruction cache, where its length counts.
  template <typename F>
  __device__ __forceinline__ void each_value(F f) const {
    constexpr int kPair = 4 / sizeof(T);
    const int warp = threadIdx.x / 32, stop = begin(warp + 1);
    int v = begin(warp) + threadIdx.x % 32;
    uint4 next = make_uint4(0, 0, 0, 0);
    if (v < stop) next = load(v);
#pragma unroll 1
    for (; v < stop; v += 32) {
      uint4 w = without_nan(next);
      if (v + 32 < stop) next = load(v + 32);
      int i = index(v, 0);
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        alignas(4) T y[kPair];
        *reinterpret_cast<uint32_t*>(y) = w.x;
        w.x = w.y, w.y = w.z, w.z = w.w;
#pragma unroll
        for (int e = 0; e < kPair; ++e, ++i) f(to_float(y[e]), i);
      }
    }
  }
};

// Kept tokens: those up to this one in the order.
struct Cut {
  float x;
  int index;
  // (A key without an index: all tokens of its logit. Key 0: every token.)
  __device__ __forceinline__ Cut(uint64_t key)
      : x(key ? logit_of(key) : -kInf), index((uint32_t)key ? index_of(key) : INT_MAX) {}
  __device__ __forceinline__ bool keeps(float y, int i) const {
    return y > -kInf && (y > x || (y == x && i <= index));
  }
};

// What a row's tokens are weighed by. 2^-t with t = n + i / 512 + r, r < 2^-9:
// t comes from fp64 as a fixed-point number (exact to 2^-33), 2^-(i / 512) from a
// table of 32 bits, and 1 - 2^-r, at most 2^-9.5, from its Taylor polynomial in
// fp32, whose rounding errors are then 2^-33 of the weight. Instructions bound the
// pass over all tokens: 97 a token with a polynomial in fp64, 44 now (256 rows of
// 128000 tokens 218 -> 74 us).
struct Weigh {
  float top;       // largest logit
  float least;     // below it a weight is nothing
  float rate32;    // log2(e) / T, and in fp64
  double rate;
  int bits;
  const uint32_t* powers;
  __device__ __forceinline__ Weigh(const uint32_t* powers_, float top_, double rate_, int vocab)
      : top(top_), rate(rate_), powers(powers_) {
    rate32 = fminf((float)rate, 1e30f);
    bits = min(51, 62 - (32 - __clz(vocab)));
    const float to = __double2float_rd((double)top - (bits + 2) / rate);
    least = to > -FLT_MAX ? to : -FLT_MAX;  // (never -infinity)
  }
  __device__ __forceinline__ float octaves(float x) const {
    return x == top ? 0.f : (top - x) * rate32;
  }
  __device__ __forceinline__ int bin(float x, float per_octave) const {
    const float t = octaves(x) * per_octave;
    return t < kBins - 1 ? (int)t : kBins - 1;  // (what is not a number, too)
  }
  // The weight added to `sum`, top being finite: what is far below it, -infinity
  // and NaN come out with so large an n that nothing is left.
  __device__ __forceinline__ unsigned long long add(unsigned long long sum, float x) const {
    // 1.5 * 2^20 + t: the low word is t's fraction in 2^-32.
    const double t = fma((double)top - (double)x, rate, 1572864.0);
    const uint32_t fraction = (uint32_t)__double2loint(t);
    const int n = __double2hiint(t) - 0x41380000;
    // r and 1 - 2^-r in units of 2^-32, in the low 23 bits of floats from 2^23 on.
    const float r = __uint_as_float(0x4b000000u | (fraction & 0x7fffffu)) - 8388608.f;
    const float kLn2 = 0.693147181f, kUnit = 2.32830644e-10f;  // 2^-32
    float less = fmaf(r, kLn2 * kLn2 * kLn2 / 6 * kUnit * kUnit, -kLn2 * kLn2 / 2 * kUnit);
    less = fmaf(r, less, kLn2);
    less = fmaf(r, less, 8388608.f);
    const uint32_t power = powers[fraction >> 23];
    const uint32_t w = power - __umulhi(power, __float_as_uint(less) - 0x4b000000u);
    // w 2^(bits - 32 - n): up by a product or down by a shift. (Shifts by more than
    // 31, or fewer than none, leave nothing: one of the two is 0.)
    uint32_t up, down;
    asm("shl.b32 %0, 2, %1;" : "=r"(up) : "r"(bits - 33 - n));
    asm("shr.u32 %0, %1, %2;" : "=r"(down) : "r"(w), "r"(n + 32 - bits));
    asm("mad.wide.u32 %0, %1, %2, %0;" : "+l"(sum) : "r"(w), "r"(up));
    asm("mad.wide.u32 %0, %1, 1, %0;" : "+l"(sum) : "r"(down));
    return sum;
  }
  __device__ __forceinline__ unsigned long long weight(float x) const {
    if (top == kInf) return x == top ? 1ull << bits : 0;
    return x >= least ? add(0, x) : 0;
  }
  __device__ __forceinline__ void add_odds(float x, Odds& sum) const {
    if (x == top) sum.x += 1.f; else sum.y += odds(x);
  }
  __device__ __forceinline__ float odds(float x) const {  // exp(x - M) for a finite M
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x - top) * (float)kLog2e));
    return y;
  }
};

// What lane c of a warp's first `ctas` lanes reads from CTA c (others: 0), summed
// over the lanes before, and over all.
template <typename V>
__device__ __forceinline__ V lanes_before(V v, V* all) {
  const int lane = threadIdx.x % 32;
  V sum = v;
#pragma unroll
  for (int o = 1; o < kMostCtas; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  *all = __shfl_sync(0xffffffffu, sum, kMostCtas - 1);
  return sum - v;
}

__device__ __forceinline__ Odds cluster_odds(cg::cluster_group& cluster, Shared& s) {
  const int lane = threadIdx.x % 32, ctas = cluster.num_blocks();
  const Odds its = lane < ctas ? cluster.map_shared_rank(&s, lane)->odds : make_float2(0.f, 0.f);
  Odds all;
  lanes_before(its.x, &all.x);
  lanes_before(its.y, &all.y);
  return all;
}

// The first bin at which the cluster's counts (MASS: masses), with `before`,
// reach the target: into s.found of every CTA, with what is before it, its count and the
// sum of all; bin -1 where they do not. Each CTA adds up its part of the bins, a
// thread four of them from one CTA: were every CTA to read all of them, 16 CTAs'
// reads of 24 KB each from 16 others took 50 us. With share >= 0 the target is
// that part of the sum, at least 1.
template <bool MASS>
__device__ void find_bin(cg::cluster_group& cluster, Shared& s, unsigned long long before,
                         unsigned long long target, float share) {
  static_assert(kBins == 4 * kThreads, "four bins of one CTA a thread");
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x % 32;
  const int bins = kBins / ctas, quads = bins / 4;  // of this CTA
  uint32_t* const counts = ctas > 1 ? s.part_counts : s.counts;
  const Wide masses = ctas > 1 ? Wide{s.part_masses[0], s.part_masses[1]}
                               : Wide{s.masses[0], s.masses[1]};
  if (ctas > 1) {
    for (int i = threadIdx.x; i < bins; i += kThreads)
      counts[i] = masses.low[i] = masses.high[i] = 0;
    __syncthreads();
    // (The CTAs begin with different ones.)
    const int c = (threadIdx.x / quads + rank) % ctas, q = threadIdx.x % quads;
    const Shared* from = cluster.map_shared_rank(&s, c);
    const uint4 n = *reinterpret_cast<const uint4*>(&from->counts[rank * bins + 4 * q]);
    const uint32_t count[4] = {n.x, n.y, n.z, n.w};
    if (MASS) {
      const uint4 lo = *reinterpret_cast<const uint4*>(&from->masses[0][rank * bins + 4 * q]);
      const uint4 hi = *reinterpret_cast<const uint4*>(&from->masses[1][rank * bins + 4 * q]);
      const unsigned long long mass[4] = {
          (unsigned long long)hi.x << 32 | lo.x, (unsigned long long)hi.y << 32 | lo.y,
          (unsigned long long)hi.z << 32 | lo.z, (unsigned long long)hi.w << 32 | lo.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (mass[e]) masses.add(4 * q + e, mass[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (count[e]) atomicAdd(&counts[4 * q + e], count[e]);
    __syncthreads();
  }
  const int each = (bins + kThreads - 1) / kThreads;  // 1 to 4
  unsigned long long amount[4], sum = 0, mine;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = threadIdx.x * each + e;
    amount[e] = e < each && i < bins ? MASS ? masses.get(i) : counts[i] : 0;
    sum += amount[e];
  }
  unsigned long long at = block_scan(s, sum, &mine), all;
  if (threadIdx.x == 0) s.part = mine;
  cluster.sync();
  const unsigned long long other =
      lane < ctas ? cluster.map_shared_rank(&s, lane)->part : 0;
  const unsigned long long ahead = lanes_before(other, &all);
  at += before + __shfl_sync(0xffffffffu, ahead, rank);
  if (MASS && share >= 0.f) {
    const double part = ceil((double)share * (double)all);
    target = part < 1.0 ? 1 : (unsigned long long)part;
    if (target > all) target = all;
  }
  if (before + all < target) {  // the same everywhere
    if (threadIdx.x == 0) s.found = Found{-1, 0, 0, all};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = threadIdx.x * each + e;
      if (at < target && at + amount[e] >= target) {
        const Found found{rank * bins + i, (int)counts[i], at, all};
        for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&s, c)->found = found;
      }
      at += amount[e];
    }
  }
  cluster.sync();
}

// The key of the first token (in the order) at which what is counted, 1 or the
// weight of every token that `cut` keeps, reaches `target` (at least 1); 0 where
// all of it does not. MASS: target is the part `share` of the mass.
template <bool MASS, typename T>
__device__ uint64_t border(cg::cluster_group& cluster, Shared& s, const Row<T>& row,
                           const Weigh& weigh, uint64_t cut_key, unsigned long long target,
                           float share) {
  const int lane = threadIdx.x % 32, ctas = cluster.num_blocks();
  const Cut cut(cut_key);
  // All tokens of t octaves below M have less than vocab 2^-t of the mass: its border
  // lies above, and bins may be the narrower (131072 tokens: 80 an octave, so that
  // those of one are few enough in the first round: 8 rows of 131071 57 -> 38 us). Counts'
  // borders may lie anywhere. The last bin has what is below.
  const float per_octave = MASS ? kBins / (40.f - __clz(row.vocab)) : kCountBins;
  uint64_t low = 0, high = ~0ull;      // keys still looked at, from the second round on
  int shift = 0, coarse_bin = -1;
  unsigned long long before = 0;       // of the tokens ahead of them
  for (int round = 0;; ++round) {
    const Wide masses{s.masses[0], s.masses[1]};
    for (int i = threadIdx.x; i < kBins; i += kThreads)
      s.counts[i] = masses.low[i] = masses.high[i] = 0;
    if (threadIdx.x == 0) s.listed = 0, s.bounds[0] = ~0ull, s.bounds[1] = 0;
    __syncthreads();
    row.each_value([&](float x, int i) {
      if (!cut.keeps(x, i)) return;
      int bin = weigh.bin(x, per_octave);
      if (round > 0) {
        const uint64_t key = key_of(x, i);
        if (bin != coarse_bin || key < low || key > high) return;
        bin = (int)((high - key) >> shift);
      }
      atomicAdd(&s.counts[bin], 1u);
      if (MASS) masses.add(bin, weigh.weight(x));
    });
    cluster.sync();
    find_bin<MASS>(cluster, s, before, target, round == 0 ? share : -1.f);
    const Found its = s.found;
    if (its.bin < 0) return 0;
    if (MASS && round == 0) {
      const double part = ceil((double)share * (double)its.all);
      target = part < 1.0 ? 1 : (unsigned long long)part;
      if (target > its.all) target = its.all;
    }
    const int bin = its.bin, found = its.count;
    before = its.before;
    if (round == 0) {
      coarse_bin = bin;
    } else {
      high -= (uint64_t)bin << shift;
      const uint64_t width = (1ull << shift) - 1;
      if (high - low > width) low = high - width;
    }
    if (found <= kFew) break;
    if (round == 0) {
      // Keys of the bin: the bounds of what is there.
      uint64_t least = ~0ull, most = 0;
      row.each_value([&](float x, int i) {
        if (!cut.keeps(x, i) || weigh.bin(x, per_octave) != coarse_bin) return;
        const uint64_t key = key_of(x, i);
        least = key < least ? key : least;
        most = key > most ? key : most;
      });
      __syncwarp();
      for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(0xffffffffu, least, o);
        const uint64_t b = __shfl_xor_sync(0xffffffffu, most, o);
        least = a < least ? a : least;
        most = b > most ? b : most;
      }
      if (lane == 0) {
        atomicMin((unsigned long long*)&s.bounds[0], (unsigned long long)least);
        atomicMax((unsigned long long*)&s.bounds[1], (unsigned long long)most);
      }
      cluster.sync();
      low = ~0ull, high = 0;
      if (lane < ctas) {
        const Shared* from = cluster.map_shared_rank(&s, lane);
        low = from->bounds[0];
        high = from->bounds[1];
      }
      for (int o = kMostCtas / 2; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(0xffffffffu, low, o);
        const uint64_t b = __shfl_xor_sync(0xffffffffu, high, o);
        low = a < low ? a : low;
        high = b > high ? b : high;
      }
      low = __shfl_sync(0xffffffffu, low, 0);
      high = __shfl_sync(0xffffffffu, high, 0);
    }
    shift = 0;
    while ((high - low) >> shift >= kBins) ++shift;
    cluster.sync();  // (the bins and bounds have been read)
  }
  // Few enough: a list of them all, the rank of each.
  row.each_value([&](float x, int i) {
    if (!cut.keeps(x, i) || weigh.bin(x, per_octave) != coarse_bin) return;
    const uint64_t key = key_of(x, i);
    if (key >= low && key <= high) s.list[atomicAdd(&s.listed, 1)] = key;
  });
  cluster.sync();
  // (A warp for each CTA's list.)
  static_assert(kWarps >= kMostCtas, "warps for lists");
  int n;
  {
    const int listed = lane < ctas ? cluster.map_shared_rank(&s, lane)->listed : 0;
    const int ahead = lanes_before(listed, &n), warp = threadIdx.x / 32;
    const int from0 = __shfl_sync(0xffffffffu, ahead, warp), some = __shfl_sync(0xffffffffu, listed, warp);
    if (warp < ctas) {
      const Shared* from = cluster.map_shared_rank(&s, warp);
      for (int i = lane; i < some; i += 32) {
        const uint64_t key = from->list[i];
        s.all[from0 + i] = key;
        s.weights[from0 + i] = MASS ? weigh.weight(logit_of(key)) : 1;
      }
    }
  }
  __syncthreads();
  // (Each CTA's share of them, as many lanes a token as there are.)
  const int rank = cluster.block_rank(), share_of = (n + ctas - 1) / ctas;
  const int stop = min(n, share_of * (rank + 1));
  int lanes = 1;
  while (lanes < 32 && 2 * lanes * share_of <= kThreads) lanes *= 2;
  for (int i0 = share_of * rank; i0 < stop; i0 += kThreads / lanes) {
    const int i = i0 + threadIdx.x / lanes;
    const uint64_t key = i < stop ? s.all[i] : ~0ull;
    unsigned long long ahead = 0;
    for (int j = threadIdx.x % lanes; j < n; j += lanes) ahead += s.all[j] > key ? s.weights[j] : 0;
    for (int o = lanes / 2; o; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    ahead += before;
    if (i < stop && threadIdx.x % lanes == 0 && ahead < target && ahead + s.weights[i] >= target)
      for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&s, c)->cut = key;
  }
  cluster.sync();  // (the lists have been read, the border is there)
  return s.cut;
}

// Where u falls in `mass`.
__device__ __forceinline__ unsigned long long place_of(const cxs_sample_call& a, long long draw,
                                                       unsigned long long mass) {
  double u = a.wide_uniforms ? ((const double*)a.uniforms)[draw]
                             : (double)((const float*)a.uniforms)[draw];
  u = u > 0.0 ? u : 0.0;  // (NaN, too)
  const double part = u * (double)mass;
  const unsigned long long at = part < (double)mass ? (unsigned long long)part : mass - 1;
  return at < mass ? at : mass - 1;
}

// Draws from the `n` gathered tokens (all that may be kept, and perhaps some
// more): one CTA. Their places in the order and by index are counted, each
// token's by as many lanes of a warp as there are for it: two bitonic sorts took
// 4 us each for 200 tokens. log_total: of the sum of exp(x - M).
__device__ __forceinline__ void draw_listed(const cxs_sample_call& a, Shared& s, const Weigh& weigh,
                                            const Settings& set, int n, long long draws,
                                            float log_total) {
  int lanes = 1;
  while (lanes < 32 && 2 * lanes * n <= kThreads) lanes *= 2;
  const int mine = threadIdx.x / lanes, from = threadIdx.x % lanes;
  uint64_t key = mine < n ? s.gathered[mine] : 0;
  int place = 0;
  for (int j = from; j < n; j += lanes) place += s.gathered[j] > key;
  for (int o = lanes / 2; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
  if (from == 0 && mine < n) s.all[place] = key;
  __syncthreads();
  // The kept ones are the first: at most top_k, with w >= min_p, and then top_p.
  key = threadIdx.x < n ? s.all[threadIdx.x] : 0;
  float x = key ? logit_of(key) : -kInf;
  const bool kept = threadIdx.x < min(n, set.top_k) && (set.min_p == 0.f || x == weigh.top ||
      (double)x >= (double)weigh.top + (double)set.temperature * log((double)set.min_p));
  unsigned long long w = kept ? weigh.weight(x) : 0, mass;
  unsigned long long before = block_scan(s, w, &mass);
  if (threadIdx.x > 0 && set.top_p < 1.f && !((double)before < (double)set.top_p * (double)mass))
    w = 0;
  s.weights[threadIdx.x] = w;
  const int count = __syncthreads_count(w > 0);
  // (Tokens without weight lie behind those that have some.)
  block_scan(s, w, &mass);
  key = mine < count ? s.all[mine] : 0;
  w = mine < count ? s.weights[mine] : 0;
  before = 0;
  for (int j = from; j < count; j += lanes)
    before += (uint32_t)s.all[j] > (uint32_t)key ? s.weights[j] : 0;
  for (int o = lanes / 2; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  x = logit_of(key);
  for (int d = from; d < a.draws; d += lanes) {
    const unsigned long long at = place_of(a, draws + d, mass);
    if (at < before || at >= before + w) continue;
    a.tokens[draws + d] = index_of(key);
    if (a.logprobs) a.logprobs[draws + d] = (x == weigh.top ? 0.f : x - weigh.top) - log_total;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const cxs_sample_call a, int slice) {
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint8_t slice_memory[];
  __shared__ __align__(16) Shared s;
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int r = blockIdx.x / ctas, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Row<T> row((const T*)a.logits + r * a.row_stride, a.vocab, rank, ctas);
  constexpr int kVector = Row<T>::kVector;
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.counts[i] = 0;
  static_assert(kPowers == kThreads, "a power a thread");
  s.powers[threadIdx.x] = power_of(threadIdx.x);
  if (threadIdx.x == 0) s.wanted = 0;
  // (The next call's CTAs come when these have ended, not before: beside them they
  // would sit two to an SM, 64 rows of 32000 in 21.5 us against 17.)
  cxs::after_earlier();
  Settings set{a.temperature ? a.temperature[r] : a.temperature_all,
               a.top_p ? a.top_p[r] : a.top_p_all, a.min_p ? a.min_p[r] : a.min_p_all,
               a.top_k ? a.top_k[r] : a.top_k_all};
  const bool wrong = !(set.temperature >= 0.f && set.temperature < kInf) || !(set.top_p >= 0.f) ||
                     !(set.min_p >= 0.f && set.min_p <= 1.f) || set.top_k < 0;
  const bool greedy = set.temperature == 0.f || set.top_k == 1;
  const bool listed = greedy || (set.top_k > 0 && set.top_k <= kMostListed &&
                                 set.top_k <= ctas * kThreads / 2);

  // The largest logit, of the thread and of the row; the run into shared memory.
  float mine = -kInf;
  {
    uint4 largest = make_uint4(Row<T>::lowest(), Row<T>::lowest(), Row<T>::lowest(), Row<T>::lowest());
    T* const keep = slice ? reinterpret_cast<T*>(slice_memory) : nullptr;
    constexpr int kAtOnce = 8;
    const int stop = row.begin(warp + 1);
    for (int v0 = row.begin(warp) + lane; v0 < stop; v0 += 32 * kAtOnce) {
      uint4 w[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (v0 + 32 * j < stop) w[j] = row.load(v0 + 32 * j);
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (v0 + 32 * j >= stop) break;
        if (keep) *reinterpret_cast<uint4*>(keep + (v0 + 32 * j) * kVector) = w[j];
        largest = Row<T>::larger_of(largest, w[j]);
      }
    }
    float x[kVector];
    Row<T>::unpack(largest, x);
#pragma unroll
    for (int e = 0; e < kVector; ++e) mine = fmaxf(mine, x[e]);
    if (keep) row.base = keep, row.kept = true;
  }
  {
    float top = mine;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s.warp_totals[warp] = top;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s.warp_totals[w]);
    if (threadIdx.x == 0) s.top = top, s.bound = -kInf;
    if (listed && !greedy && top > -kInf && !wrong) {
      // At least 1 / ctas of top_k tokens of this CTA lie in the bins that as many
      // of its threads' maxima reach; the least of these maxima bounds them.
      const Weigh local(s.powers, top, kLog2e / set.temperature, a.vocab);
      const int bin = mine > -kInf ? local.bin(mine, kCountBins) : kBins;
      if (bin < kBins) atomicAdd(&s.counts[bin], 1u);
      __syncthreads();
      const uint4 n = *reinterpret_cast<const uint4*>(&s.counts[4 * threadIdx.x]);
      const unsigned wanted = (set.top_k + ctas - 1) / ctas;
      unsigned long long all;
      const unsigned sum = n.x + n.y + n.z + n.w, at = (unsigned)block_scan(s, sum, &all);
      if (at < wanted && at + sum >= wanted)
        s.found.bin = 4 * threadIdx.x + (at + n.x < wanted) + (at + n.x + n.y < wanted) +
                      (at + n.x + n.y + n.z < wanted);
      __syncthreads();
      float least = all >= wanted && bin <= s.found.bin ? mine : kInf;
      for (int o = 16; o; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
      if (lane == 0) s.warp_totals[warp] = least;
      __syncthreads();
      if (threadIdx.x == 0 && all >= wanted) {
        for (int w = 0; w < kWarps; ++w) least = fminf(least, s.warp_totals[w]);
        s.bound = least;
      }
    }
  }
  cluster.sync();
  float top = lane < ctas ? cluster.map_shared_rank(&s, lane)->top : -kInf;
  float bound = lane < ctas ? cluster.map_shared_rank(&s, lane)->bound : kInf;
  for (int o = kMostCtas / 2; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bound = fminf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
  }
  top = __shfl_sync(0xffffffffu, top, 0);
  bound = __shfl_sync(0xffffffffu, bound, 0);
  const long long draws = (long long)r * a.draws;
  if (wrong || top == -kInf) {  // no answer
    if (rank == 0)
      for (int d = threadIdx.x; d < a.draws; d += kThreads) {
        a.tokens[draws + d] = -1;
        if (a.logprobs) a.logprobs[draws + d] = -kInf;
      }
    cluster.sync();
    return;
  }
  const Weigh weigh(s.powers, top, greedy ? 0.0 : kLog2e / set.temperature, a.vocab);
  const bool want = a.logprobs != nullptr;

  if (listed) {
    if (greedy) set.top_k = 1, bound = top;
    Shared* const first = cluster.map_shared_rank(&s, 0);
    Odds total = make_float2(0.f, 0.f);
    row.each_value([&](float x, int i) {
      if (x >= bound && x > -kInf) {
        const int at = atomicAdd(&first->wanted, 1);
        if (at < kList) first->gathered[at] = key_of(x, i);
      }
      if (want) weigh.add_odds(x, total);
    });
    if (want) {
      total = block_sum(s, total);
      if (threadIdx.x == 0) s.odds = total;
    }
    cluster.sync();
    const int n = first->wanted;
    if (n <= kList) {
      if (rank == 0 && want) total = cluster_odds(cluster, s);
      cluster.sync();  // (what is read of other CTAs has been)
      if (rank == 0) draw_listed(a, s, weigh, set, n, draws, log_of(total));
      return;
    }
    cluster.sync();  // (`wanted` and the list are free)
  }

  uint64_t cut = 0;  // keys of kept tokens are at least this
  if (set.top_k > 0 && set.top_k < a.vocab)
    cut = border<false>(cluster, s, row, weigh, 0, set.top_k, 0.f);
  if (set.min_p > 0.f && !greedy) {
    const float least =
        __double2float_ru((double)weigh.top + (double)set.temperature * log((double)set.min_p));
    const uint64_t other = key_of(fminf(least, weigh.top), INT_MAX) & ~0xffffffffull;
    cut = other > cut ? other : cut;
  }
  if (set.top_p < 1.f && !greedy) {
    const uint64_t other = border<true>(cluster, s, row, weigh, cut, 0, set.top_p);
    cut = other > cut ? other : cut;
  }

  // Kept mass of every warp's run and of its parts, and the sum of exp(x - M) over
  // all tokens.
  const Cut keep(cut);
  const int begin = row.begin(warp), stop = row.begin(warp + 1);
  const int rounds = ((row.each + 31) / 32 + kBlocks - 1) / kBlocks;  // of a part
  unsigned long long mass = 0;
  Odds total = make_float2(0.f, 0.f);
  auto weigh_all = [&](auto add) {
    uint4 next = make_uint4(0, 0, 0, 0);
    if (begin + lane < stop) next = row.load(begin + lane);
    for (int v0 = begin, part = 0; v0 < stop; ++part) {
      unsigned long long sum = 0;
#pragma unroll 1
      for (int k = 0; k < rounds && v0 < stop; ++k, v0 += 32) {
        const int v = v0 + lane;
        const uint32_t none = Row<T>::lowest();
        const uint4 w = v < stop ? Row<T>::without_nan(next) : make_uint4(none, none, none, none);
        if (v + 32 < stop) next = row.load(v + 32);
        float x[kVector];
        Row<T>::unpack(w, x);
        const int i = row.index(v, 0);
        add(sum, x, i);
      }
      __syncwarp();
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s.blocks[warp][part] = sum;
      mass += sum;
    }
  };
  if (cut == 0 && weigh.top < kInf)
    weigh_all([&](unsigned long long& sum, const float (&x)[kVector], int) {
#pragma unroll
      for (int e = 0; e < kVector; ++e) sum = weigh.add(sum, x[e]);
      if (!want) return;
      float odds = 0.f;
#pragma unroll
      for (int e = 0; e < kVector; ++e) odds += weigh.odds(x[e]);
      if (odds < 1.f) {  // (M is not among them)
        total.y += odds;
      } else {
#pragma unroll
        for (int e = 0; e < kVector; ++e) weigh.add_odds(x[e], total);
      }
    });
  else
    weigh_all([&](unsigned long long& sum, const float (&x)[kVector], int i) {
#pragma unroll
      for (int e = 0; e < kVector; ++e) {
        if (keep.keeps(x[e], i + e)) sum += weigh.weight(x[e]);
        if (want) weigh.add_odds(x[e], total);
      }
    });
  __syncwarp();
  if (want) total = block_sum(s, total);
  unsigned long long all;
  const unsigned long long ahead = block_scan(s, lane == 0 ? mass : 0, &all);
  if (lane == 0) s.spans[warp] = ahead;
  if (threadIdx.x == 0) {
    s.odds = total;
    s.mass = all;
  }
  cluster.sync();
  const Shared* const other = cluster.map_shared_rank(&s, min(lane, ctas - 1));
  unsigned long long kept_mass;
  unsigned long long before = lanes_before(lane < ctas ? other->mass : 0, &kept_mass);
  before = __shfl_sync(0xffffffffu, before, rank);
  if (want) total = cluster_odds(cluster, s);
  cluster.sync();  // (the sums have been read)
  const float log_total = log_of(total);

  // A warp for each draw that falls into this CTA.
  for (int d = warp; d < a.draws; d += kWarps) {
    unsigned long long at = place_of(a, draws + d, kept_mass);
    if (at < before || at >= before + all) continue;
    at -= before;
    // The run it falls into: the last that begins at or before it and has any.
    const bool in = lane < kWarps && s.spans[min(lane, kWarps - 1)] <= at &&
                    at < (lane + 1 < kWarps ? s.spans[lane + 1] : all);
    const int w = __ffs(__ballot_sync(0xffffffffu, in)) - 1;
    at -= s.spans[w];
    // The part of the run: four a lane.
    static_assert(kBlocks == 4 * 32, "four parts a lane");
    const int its_begin = row.begin(w), its_stop = row.begin(w + 1);
    const int parts = (its_stop - its_begin + 32 * rounds - 1) / (32 * rounds);
    unsigned long long four[4], sum4 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      four[e] = 4 * lane + e < parts ? s.blocks[w][4 * lane + e] : 0;
      sum4 += four[e];
    }
    unsigned long long to4 = sum4;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, to4, o);
      if (lane >= o) to4 += up;
    }
    int part = 0;
    unsigned long long rest = at - (to4 - sum4);
    const unsigned holds = __ballot_sync(0xffffffffu, at < to4 && at >= to4 - sum4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (part == e && rest >= four[e]) rest -= four[e], ++part;
    }
    const int owner = __ffs(holds) - 1;
    at = __shfl_sync(0xffffffffu, rest, owner);
    const int its_part = 4 * owner + __shfl_sync(0xffffffffu, part, owner);
    const int from = its_begin + its_part * 32 * rounds, to_v = min(its_stop, from + 32 * rounds);
    // Four bytes a lane at a time.
    constexpr int kPair = 4 / sizeof(T);
#pragma unroll 1
    for (int u0 = 4 * from; u0 < 4 * to_v; u0 += 32) {
      const int u = u0 + lane;
      const uint4 vector = Row<T>::without_nan(row.load(min(u / 4, to_v - 1)));
      alignas(4) T y[kPair];
      *reinterpret_cast<uint32_t*>(y) = u % 4 == 0 ? vector.x : u % 4 == 1 ? vector.y
                                      : u % 4 == 2 ? vector.z : vector.w;
      unsigned long long weights[kPair], sum = 0;
      float x[kPair];
#pragma unroll
      for (int e = 0; e < kPair; ++e) {
        x[e] = to_float(y[e]);
        const bool in = u < 4 * to_v && keep.keeps(x[e], row.index(0, u * kPair + e));
        weights[e] = in ? weigh.weight(x[e]) : 0;
        sum += weights[e];
      }
      unsigned long long to = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, to, o);
        if (lane >= o) to += up;
      }
      const unsigned long long chunk = __shfl_sync(0xffffffffu, to, 31);
      if (at >= chunk) {
        at -= chunk;
        continue;
      }
      if (at < to && at >= to - sum) {
        unsigned long long left = at - (to - sum);
#pragma unroll
        for (int e = 0; e < kPair; ++e) {
          if (left < weights[e]) {
            a.tokens[draws + d] = row.index(0, u * kPair + e);
            if (want)
              a.logprobs[draws + d] = (x[e] == weigh.top ? 0.f : x[e] - weigh.top) - log_total;
            break;
          }
          left -= weights[e];
        }
      }
      break;
    }
  }
}

// CTAs of a row's cluster: as many as still have an SM each and kLeast values.
// Measured for 1, 2, 4, 8 and 16 of them (us, in a graph, with log-probabilities):
// few rows, bf16, top_k 50 and top_p of 4000 tokens 9.8 / 10.7 / 10.7 / 10.9 / 12.2, of
// 8000 10.9 / 10.0 / 10.6 / 10.9 / 12.1, of 16000 12.1 / 11.2 / 10.0 / 10.9 / 12.2, of
// 32000 14.7 / 12.8 / 11.1 / 10.5 / 12.4, of 64000 20.6 / 15.2 / 12.4 / 11.5 / 11.7
// (top_p alone 89 / 52 / 34 / 26 / 24); 64 rows of 32000 14.8 / 13.1 / 14.5 / 25 / 54, 8
// rows of 131071 (fp32, top_p) 184 / 101 / 59 / 38 / 36, 256 rows of 128000 70 / 77 / 89 /
// 122 / 248.
int ctas_of(const cxs_sample_call& a) {
  constexpr int kAtOnce = 148, kLeast = 3000;
  int ctas = 1;
  while (ctas < kMostCtas && (long long)a.rows * ctas * 2 <= kAtOnce && a.vocab >= 2 * kLeast * ctas)
    ctas *= 2;
  return ctas;
}

template <typename T>
int launch(const cxs_sample_call& a, cudaStream_t stream) {
  static cxs_host::OncePerDevice ready;
  const int status = ready.run([] {
    CXS_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kSliceBytes));
    CXS_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return (int)CXS_OK;
  });
  if (status != CXS_OK) return status;
  const int ctas = ctas_of(a);
  // (A row may begin inside a vector, and vectors are shared out whole.)
  const long long vectors = ((long long)a.vocab * sizeof(T) + 15) / 16 + 1;
  const long long bytes = (vectors + ctas - 1) / ctas * 16;
  const int slice = bytes <= kSliceBytes ? (int)bytes : 0;
  return cxs_host::launch_early("sample", sample_kernel<T>, dim3(a.rows * ctas), kThreads, slice,
                                ctas, stream, a, slice);
}

}  // namespace

extern "C" int cxs_sample(const cxs_sample_call* call, void* stream) {
  if (!call) return set_error(CXS_ERR_INVALID, "sample: null call");
  const cxs_sample_call& a = *call;
  if (a.rows < 0 || a.draws < 0 || a.vocab < 1)
    return set_error(CXS_ERR_INVALID, "sample: rows and draws must not be negative, vocab positive");
  if (a.type < CXS_TYPE_BF16 || a.type > CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "sample: unknown type");
  if (a.vocab > 1 << 24 || a.rows > 1 << 24 || (long long)a.rows * a.draws > INT_MAX)
    return set_error(CXS_ERR_CAPACITY, "sample: more than 2^24 tokens or rows, or 2^31 draws");
  if (!a.temperature && !(a.temperature_all >= 0.f && a.temperature_all < INFINITY))
    return set_error(CXS_ERR_INVALID, "sample: temperature must be finite and not negative");
  if (!a.top_k && a.top_k_all < 0) return set_error(CXS_ERR_INVALID, "sample: negative top_k");
  if (!a.top_p && !(a.top_p_all >= 0.f)) return set_error(CXS_ERR_INVALID, "sample: negative top_p");
  if (!a.min_p && !(a.min_p_all >= 0.f && a.min_p_all <= 1.f))
    return set_error(CXS_ERR_INVALID, "sample: min_p must be 0 .. 1");
  if (a.rows == 0 || a.draws == 0) return CXS_OK;
  if (!a.logits || !a.uniforms || !a.tokens)
    return set_error(CXS_ERR_INVALID, "sample: null logits, uniforms or tokens");
  const int size = a.type == CXS_TYPE_F32 ? 4 : 2;
  if ((uintptr_t)a.logits % size) return set_error(CXS_ERR_INVALID, "sample: unaligned logits");
  CXS_CACHE_TYPE(a.type, T, return launch<T>(a, (cudaStream_t)stream));
}
