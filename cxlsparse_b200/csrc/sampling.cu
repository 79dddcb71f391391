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
// weight is a 64-bit integer, 2^-t in fp64 (to 2^-42 of itself) times 2^S with S as
// large as the sum over the vocabulary allows (45 bits for 2^17 tokens). Sums of
// integers do not depend on their order, so neither does a result.
//
// A row is worked on by a cluster of CTAs, each with a run of the vocabulary and
// in it a run for each warp. The border token of a cut is found in a histogram of
// 2048 bins of log2 w (counts for top-k, masses for top-p), then among the
// tokens of one bin: by rank if they are few, by histograms of their order's
// key (logit and index, 64 bits) until they are.
#include <cooperative_groups.h>
#include <limits.h>

#include "cache8.cuh"

using cxs_host::set_error;

namespace {

using cxs::cache8::to_float;
namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kBinsPerOctave = 32;   // of the weight: 64 octaves in all
constexpr int kFew = 512;            // tokens whose ranks are counted one by one
constexpr float kInf = INFINITY;
constexpr double kLog2e = 1.4426950408889634;

// Order's key: larger comes first.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 as 0)
  const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)k << 32 | (0xffffffffu - (uint32_t)index);
}
// Its logit.
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^-t, t in [0, 64), times 2^bits as an integer: Taylor's polynomial of 2^-f
// for |f| <= 1/2 (the next term is below 2^-42), rounded at the last place.
__device__ __forceinline__ uint64_t fixed_exp2(double t, int bits) {
  const double shift = 6755399441055744.0;  // 1.5 * 2^52: t rounded in the low bits
  const double n = t + shift;
  const double g = (t - (n - shift)) * -0.6931471805599453;
  double p = 1.0 / 3628800;
  p = fma(p, g, 1.0 / 362880);
  p = fma(p, g, 1.0 / 40320);
  p = fma(p, g, 1.0 / 5040);
  p = fma(p, g, 1.0 / 720);
  p = fma(p, g, 1.0 / 120);
  p = fma(p, g, 1.0 / 24);
  p = fma(p, g, 1.0 / 6);
  p = fma(p, g, 0.5);
  p = fma(p, g, 1.0);
  p = fma(p, g, 1.0);
  const int e = bits - __double2loint(n);
  p = __hiloint2double(__double2hiint(p) + (e << 20), __double2loint(p));
  return (uint64_t)__double_as_longlong(p + 4503599627370496.0) & 0xfffffffffffffull;
}

struct Settings {  // of a row
  float temperature, top_p, min_p;
  int top_k;
};

struct Shared {
  uint32_t counts[kBins];
  unsigned long long masses[kBins];
  uint64_t list[kFew];                         // this CTA's
  uint64_t all[kFew];                          // the cluster's
  unsigned long long weights[kFew];
  unsigned long long sums[kWarps];             // of a scan
  unsigned long long spans[kWarps];            // kept mass before each warp's tokens
  uint64_t exchanged;                          // read by the cluster: largest key,
  unsigned long long mass;                     // kept mass of this CTA,
  float total;                                 // its sum of exp(x - M),
  int listed;                                  // and what it has listed
  int bin, count;
  unsigned long long before;
  uint64_t cut;
  float warp_totals[kWarps];
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
  unsigned long long all = s.sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const unsigned long long before = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);
  return sum - v + (warp > 0 ? before : 0);
}

template <typename T>
struct Row {
  static constexpr int kVector = 16 / sizeof(T);
  const T* base;       // the 16-byte vector that the row begins in
  int skip;            // values of it before the row
  int vocab;
  int first, last;     // vectors of this warp
  // f(logit, index, there) for this warp's tokens, vector by vector: all lanes call it.
  // NaN counts as -infinity.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x % 32;
    constexpr int kAtOnce = 4;
    for (int v0 = first; v0 < last; v0 += 32 * kAtOnce) {
      alignas(16) T x[kAtOnce][kVector];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int v = v0 + 32 * j + lane;
        if (v < last) load(v, x[j]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (v0 + 32 * j >= last) break;
        const int v = v0 + 32 * j + lane;
#pragma unroll
        for (int e = 0; e < kVector; ++e) {
          const int i = v * kVector + e - skip;
          const bool there = v < last && i >= 0 && i < vocab;
          const float y = there ? to_float(x[j][e]) : -kInf;
          f(y == y ? y : -kInf, i, there);
        }
      }
    }
  }
  __device__ __forceinline__ void load(int v, T (&x)[kVector]) const {
    const int i = v * kVector - skip;
    if (i >= 0 && i + kVector <= vocab) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(base + (long long)v * kVector);
    } else {
#pragma unroll
      for (int e = 0; e < kVector; ++e)
        if (i + e >= 0 && i + e < vocab) x[e] = base[(long long)v * kVector + e];
    }
  }
};

// What a row's tokens are weighed by.
struct Weigh {
  float top;       // largest logit
  float rate32;    // log2(e) / T, and in fp64
  double rate;
  int bits;
  __device__ __forceinline__ float octaves(float x) const {
    return x == top ? 0.f : (top - x) * rate32;
  }
  __device__ __forceinline__ int bin(float x) const {
    const float t = octaves(x) * kBinsPerOctave;
    return t < kBins - 1 ? (int)t : kBins - 1;  // (what is not a number, too)
  }
  __device__ __forceinline__ unsigned long long weight(float x) const {
    if (!(octaves(x) < 60.f)) return 0;
    return fixed_exp2(x == top ? 0.0 : ((double)top - (double)x) * rate, bits);
  }
};

// The key of the first token (in the order) at which what is counted, 1 or the
// weight of every token with a key of at least `cut`, reaches `target` (at least
// 1); 0 where all of it does not. MASS: target is the part `share` of the mass.
template <bool MASS, typename T>
__device__ uint64_t border(cg::cluster_group& cluster, Shared& s, const Row<T>& row,
                           const Weigh& weigh, uint64_t cut, unsigned long long target,
                           float share) {
  const int lane = threadIdx.x % 32, ctas = cluster.num_blocks();
  uint64_t low = 0, high = 0;          // keys still looked at, from the second round on
  int shift = 0, coarse_bin = -1;
  unsigned long long before = 0;       // of the tokens ahead of them
  for (int round = 0;; ++round) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.counts[i] = 0, s.masses[i] = 0;
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    row.each([&](float x, int i, bool there) {
      const uint64_t key = key_of(x, i);
      int bin = -1;
      if (there && x > -kInf && key >= cut) {
        if (round == 0)
          bin = weigh.bin(x);
        else if (key >= low && key <= high && weigh.bin(x) == coarse_bin)
          bin = (int)((high - key) >> shift);
      }
      if (!__any_sync(0xffffffffu, bin >= 0)) return;
      unsigned long long w = 0;
      if (MASS && bin >= 0) w = weigh.weight(x);
      if (bin >= 0) {
        atomicAdd(&s.counts[bin], 1u);
        if (MASS) atomicAdd(&s.masses[bin], w);
      }
    });
    cluster.sync();
    // The cluster's bins: two to a thread.
    constexpr int kEach = kBins / kThreads;
    uint32_t count[kEach] = {};
    unsigned long long amount[kEach] = {}, sum = 0;
    for (int c = 0; c < ctas; ++c) {
      const Shared* from = cluster.map_shared_rank(&s, c);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        count[e] += from->counts[threadIdx.x * kEach + e];
        if (MASS) amount[e] += from->masses[threadIdx.x * kEach + e];
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (!MASS) amount[e] = count[e];
      sum += amount[e];
    }
    unsigned long long all, at = before + block_scan(s, sum, &all);
    if (MASS && round == 0) {
      const double part = ceil((double)share * (double)all);
      target = part < 1.0 ? 1 : (unsigned long long)part;
      if (target > all) target = all;
    }
    if (before + all < target) {
      cluster.sync();  // (the bins have been read)
      return 0;
    }
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (at < target && at + amount[e] >= target) {
        s.bin = threadIdx.x * kEach + e;
        s.count = (int)count[e];
        s.before = at;
      }
      at += amount[e];
    }
    __syncthreads();
    const int bin = s.bin, found = s.count;
    before = s.before;
    if (round == 0) {
      coarse_bin = bin;
      low = cut;
      high = ~0ull;
    } else {
      high -= (uint64_t)bin << shift;
      const uint64_t width = (1ull << shift) - 1;
      if (high - low > width) low = high - width;
    }
    if (found <= kFew) break;
    if (round == 0) {
      // Keys of the bin: the bounds of what is there.
      uint64_t least = ~0ull, most = 0;
      row.each([&](float x, int i, bool there) {
        const uint64_t key = key_of(x, i);
        if (there && x > -kInf && key >= cut && weigh.bin(x) == coarse_bin) {
          least = key < least ? key : least;
          most = key > most ? key : most;
        }
      });
      for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(0xffffffffu, least, o);
        const uint64_t b = __shfl_xor_sync(0xffffffffu, most, o);
        least = a < least ? a : least;
        most = b > most ? b : most;
      }
      if (threadIdx.x == 0) s.list[0] = ~0ull, s.list[1] = 0;
      __syncthreads();
      if (lane == 0) {
        atomicMin((unsigned long long*)&s.list[0], (unsigned long long)least);
        atomicMax((unsigned long long*)&s.list[1], (unsigned long long)most);
      }
      cluster.sync();
      low = ~0ull, high = 0;
      for (int c = 0; c < ctas; ++c) {
        const Shared* from = cluster.map_shared_rank(&s, c);
        low = from->list[0] < low ? from->list[0] : low;
        high = from->list[1] > high ? from->list[1] : high;
      }
    }
    shift = 0;
    while ((high - low) >> shift >= kBins) ++shift;
    cluster.sync();  // (the bins and bounds have been read)
  }
  // Few enough: a list of them all, the rank of each.
  row.each([&](float x, int i, bool there) {
    const uint64_t key = key_of(x, i);
    if (there && x > -kInf && key >= low && key <= high && weigh.bin(x) == coarse_bin)
      s.list[atomicAdd(&s.listed, 1)] = key;
  });
  cluster.sync();
  int n = 0;
  for (int c = 0; c < ctas; ++c) {
    const Shared* from = cluster.map_shared_rank(&s, c);
    const int some = from->listed;
    for (int i = threadIdx.x; i < some; i += kThreads) {
      const uint64_t key = from->list[i];
      s.all[n + i] = key;
      s.weights[n + i] = MASS ? weigh.weight(logit_of(key)) : 1;
    }
    n += some;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = s.all[i];
    unsigned long long ahead = before;
    for (int j = 0; j < n; ++j) ahead += s.all[j] > key ? s.weights[j] : 0;
    if (ahead < target && ahead + s.weights[i] >= target) s.cut = key;
  }
  cluster.sync();  // (the lists have been read)
  return s.cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const cxs_sample_call a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ Shared s;
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int r = blockIdx.x / ctas, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const T* const values = (const T*)a.logits + r * a.row_stride;
  Row<T> row;
  row.vocab = a.vocab;
  row.skip = (int)((uintptr_t)values % 16 / sizeof(T));
  row.base = values - row.skip;
  {
    const int vectors = (int)(((long long)a.vocab + row.skip + row.kVector - 1) / row.kVector);
    const int each = (vectors + ctas - 1) / ctas, first = min(each * rank, vectors);
    const int here = min(each, vectors - first), mine = (here + kWarps - 1) / kWarps;
    row.first = first + min(mine * warp, here);
    row.last = first + min(mine * (warp + 1), here);
  }
  Settings set{a.temperature ? a.temperature[r] : a.temperature_all,
               a.top_p ? a.top_p[r] : a.top_p_all, a.min_p ? a.min_p[r] : a.min_p_all,
               a.top_k ? a.top_k[r] : a.top_k_all};
  const bool wrong = !(set.temperature >= 0.f && set.temperature < kInf) || !(set.top_p >= 0.f) ||
                     !(set.min_p >= 0.f && set.min_p <= 1.f) || set.top_k < 0;

  // The largest logit.
  uint64_t key = 0;
  row.each([&](float x, int i, bool there) {
    const uint64_t k = key_of(x, i);
    if (there && x > -kInf && k > key) key = k;
  });
  for (int o = 16; o; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  if (threadIdx.x == 0) s.exchanged = 0;
  __syncthreads();
  if (lane == 0) atomicMax((unsigned long long*)&s.exchanged, (unsigned long long)key);
  cluster.sync();
  key = 0;
  for (int c = 0; c < ctas; ++c) {
    const uint64_t other = cluster.map_shared_rank(&s, c)->exchanged;
    key = other > key ? other : key;
  }
  const long long draws = (long long)r * a.draws;
  if (wrong || key == 0) {  // no answer
    if (rank == 0)
      for (int d = threadIdx.x; d < a.draws; d += kThreads) {
        a.tokens[draws + d] = -1;
        if (a.logprobs) a.logprobs[draws + d] = -kInf;
      }
    cluster.sync();
    return;
  }

  Weigh weigh;
  weigh.top = logit_of(key);
  const bool greedy = set.temperature == 0.f || set.top_k == 1;
  weigh.rate = greedy ? 0.0 : kLog2e / set.temperature;
  weigh.rate32 = fminf((float)weigh.rate, 1e30f);
  weigh.bits = min(51, 62 - (32 - __clz(a.vocab)));
  uint64_t cut = 0;  // keys of kept tokens are at least this
  if (greedy) {
    cut = key;
  } else {
    if (set.top_k > 0 && set.top_k < a.vocab)
      cut = border<false>(cluster, s, row, weigh, 0, set.top_k, 0.f);
    if (set.min_p > 0.f) {
      const float least =
          __double2float_ru((double)weigh.top + (double)set.temperature * log((double)set.min_p));
      const uint64_t other = key_of(fminf(least, weigh.top), INT_MAX) & ~0xffffffffull;
      cut = other > cut ? other : cut;
    }
    if (set.top_p < 1.f) {
      const uint64_t other = border<true>(cluster, s, row, weigh, cut, 0, set.top_p);
      cut = other > cut ? other : cut;
    }
  }

  // Kept mass of every warp's run, and the sum of exp(x - M) over all tokens.
  unsigned long long mass = 0;
  float total = 0.f;
  const bool want = a.logprobs != nullptr;
  row.each([&](float x, int i, bool there) {
    const bool kept = there && x > -kInf && key_of(x, i) >= cut;
    if (__any_sync(0xffffffffu, kept) && kept) mass += weigh.weight(x);
    if (want) total += x == weigh.top ? 1.f : exp2f((x - weigh.top) * (float)kLog2e);
  });
  for (int o = 16; o; o >>= 1) {
    mass += __shfl_xor_sync(0xffffffffu, mass, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) s.warp_totals[warp] = total;
  unsigned long long all;
  const unsigned long long ahead = block_scan(s, lane == 0 ? mass : 0, &all);
  if (lane == 0) s.spans[warp] = ahead;
  if (threadIdx.x == 0) {
    total = 0.f;
    for (int w = 0; w < kWarps; ++w) total += s.warp_totals[w];
    s.total = total;
    s.mass = all;
  }
  cluster.sync();
  unsigned long long before = 0, kept_mass = 0;
  total = 0.f;
  for (int c = 0; c < ctas; ++c) {
    const Shared* from = cluster.map_shared_rank(&s, c);
    if (c == rank) before = kept_mass;
    kept_mass += from->mass;
    total += from->total;
  }
  const float log_total = logf(total);

  // A warp for each draw that falls into this CTA.
  for (int d = warp; d < a.draws; d += kWarps) {
    double u = a.wide_uniforms ? ((const double*)a.uniforms)[draws + d]
                               : (double)((const float*)a.uniforms)[draws + d];
    u = u > 0.0 ? u : 0.0;  // (NaN, too)
    const double part = u * (double)kept_mass;
    unsigned long long at = part < (double)kept_mass ? (unsigned long long)part : kept_mass - 1;
    if (at >= kept_mass) at = kept_mass - 1;
    if (at < before || at >= before + all) continue;
    at -= before;
    // The run it falls into: the last that begins at or before it and has any.
    const unsigned run =
        __ballot_sync(0xffffffffu, s.spans[lane] <= at &&
                                       at < (lane + 1 < kWarps ? s.spans[lane + 1] : all));
    const int w = __ffs(run) - 1;
    at -= s.spans[w];
    Row<T> its = row;
    {
      const int vectors = (int)(((long long)a.vocab + row.skip + row.kVector - 1) / row.kVector);
      const int each = (vectors + ctas - 1) / ctas, first = min(each * rank, vectors);
      const int here = min(each, vectors - first), mine = (here + kWarps - 1) / kWarps;
      its.first = first + min(mine * w, here);
      its.last = first + min(mine * (w + 1), here);
    }
    for (int v0 = its.first; v0 < its.last; v0 += 32) {
      const int v = v0 + lane;
      T x[Row<T>::kVector];
      if (v < its.last) its.load(v, x);
      unsigned long long weights[Row<T>::kVector], sum = 0;
#pragma unroll
      for (int e = 0; e < Row<T>::kVector; ++e) {
        const int i = v * Row<T>::kVector + e - its.skip;
        const bool there = v < its.last && i >= 0 && i < a.vocab;
        const float y = there ? to_float(x[e]) : -kInf;
        weights[e] = there && y > -kInf && key_of(y, i) >= cut ? weigh.weight(y) : 0;
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
        for (int e = 0; e < Row<T>::kVector; ++e) {
          if (left < weights[e]) {
            const float y = to_float(x[e]);
            a.tokens[draws + d] = v * Row<T>::kVector + e - its.skip;
            if (want) a.logprobs[draws + d] = (y == weigh.top ? 0.f : y - weigh.top) - log_total;
            break;
          }
          left -= weights[e];
        }
      }
      break;
    }
  }
  cluster.sync();  // (the sums have been read)
}

template <typename T>
int launch(const cxs_sample_call& a, int ctas, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(a.rows * ctas);
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  CXS_CUDA(cudaLaunchKernelEx(&config, sample_kernel<T>, a));
  CXS_LAUNCH_CHECK("sample");
  return CXS_OK;
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
  const int ctas = 1;
  cudaStream_t s = (cudaStream_t)stream;
  CXS_CACHE_TYPE(a.type, T, return launch<T>(a, ctas, s));
}
