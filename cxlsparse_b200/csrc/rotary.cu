// Rotary positions: layouts, part of the head, any frequencies, either direction.
#include "cache8.cuh"

using cxs_host::set_error;

namespace {

using cxs::cache8::from_float;
using cxs::cache8::to_float;

// Sine and cosine of a phase given as a 64-bit fraction of a turn: the top
// bits, centred on zero, go to sincospif as half turns.
__device__ __forceinline__ float2 turn(unsigned long long phase, float magnitude, int transpose) {
  const int top = (int)(phase >> 32);          // [-1/2, 1/2) turns in units of 2^-32
  float s, c;
  sincospif((float)top * 0x1p-31f, &s, &c);
  return make_float2(c * magnitude, (transpose ? -s : s) * magnitude);
}

struct alignas(16) Vec16 {
  uint32_t w[4];
};

// V consecutive channels: one 16-byte access, or (V of 1 or 2) V plain ones.
template <typename T, int V>
__device__ __forceinline__ void load(T (&to)[V], const T* from) {
  if constexpr (V * sizeof(T) == 16) {
    *reinterpret_cast<Vec16*>(to) = *reinterpret_cast<const Vec16*>(from);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = from[e];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* to, const T (&from)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    *reinterpret_cast<Vec16*>(to) = *reinterpret_cast<const Vec16*>(from);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = from[e];
  }
}

// How a head is cut: a thread's unit is two vectors of V channels. Half
// layout: channels [u V, u V + V) and the same of the second half; interleaved:
// neighbouring vectors. Units past the rotated channels copy two vectors.
struct Cut {
  int units;   // of a head; threadIdx.x
  int turned;  // units that rotate (half layout)
  int tokens;  // of a CTA
  int step_token, step_head;  // blockDim.y rows further: this many tokens and heads
};

// Memory-bound: every channel is read and written once; the angles of a CTA's
// tokens are computed once, into shared memory, for all their heads, while
// the first kRows rows of every thread are already being loaded (a row is one
// head of one token). 2 x kRows vectors a thread in flight. Measured: 19,188
// tokens of 40 heads of 128 in fp16, 393 MB in 65 us (6.1 TB/s); a token each of
// 8 users in 2.6 us.
constexpr int kRows = 4;

template <typename T, int LAYOUT, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const cxs_rotary_call r, const Cut cut) {
  extern __shared__ float2 angles[];  // [tokens of the CTA][pairs]
  const int pairs = r.rotary_dim / 2, heads = r.heads + r.kv_heads;
  const int token0 = blockIdx.x * cut.tokens;
  const int tokens = min(cut.tokens, r.tokens - token0);
  const int u = threadIdx.x;

  // The unit's channels: offsets of its vectors (-1: none) and first pairs.
  int at0, at1, pair0, pair1;  // pair -1: copied
  if (LAYOUT == CXS_ROTARY_HALF) {
    if (u < cut.turned) {
      at0 = u * V, at1 = at0 + pairs, pair0 = pair1 = at0;
    } else {
      at0 = r.rotary_dim + 2 * (u - cut.turned) * V, at1 = at0 + V, pair0 = pair1 = -1;
    }
  } else {
    at0 = 2 * u * V, at1 = at0 + V;
    pair0 = at0 < r.rotary_dim ? at0 / 2 : -1;
    pair1 = at1 < r.rotary_dim ? at1 / 2 : -1;
  }
  if (at1 >= r.dim) at1 = -1;

  int token = threadIdx.y / heads, head = threadIdx.y % heads;
  const T* src[kRows];
  T x[kRows][2][V];
  int rows_token[kRows], rows_head[kRows];
  auto advance = [&](int n) {  // the thread's next rows: loads
#pragma unroll
    for (int i = 0; i < n; ++i) {
      rows_token[i] = token < tokens ? token : -1;
      rows_head[i] = head;
      if (token < tokens) {
        const long long t = token0 + token;
        src[i] = head < r.heads
                     ? (const T*)r.q + t * r.q_token_stride + head * r.q_head_stride
                     : (const T*)r.k + t * r.k_token_stride + (head - r.heads) * r.k_head_stride;
        load<T, V>(x[i][0], src[i] + at0);
        if (at1 >= 0) load<T, V>(x[i][1], src[i] + at1);
      }
      token += cut.step_token;
      head += cut.step_head;
      if (head >= heads) head -= heads, ++token;
    }
  };
  advance(kRows);
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < tokens * pairs;
       i += blockDim.x * blockDim.y) {
    const int pair = i % pairs;
    const long long t = token0 + i / pairs;
    const long long position =
        r.wide_positions ? ((const long long*)r.positions)[t] : ((const int*)r.positions)[t];
    angles[i] = turn((unsigned long long)position * (unsigned long long)r.steps[pair], r.magnitude,
                     r.transpose);
  }
  __syncthreads();
  while (true) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (rows_token[i] < 0) continue;
      const long long t = token0 + rows_token[i];
      const int h = rows_head[i];
      T* dst = h < r.heads
                   ? (T*)r.q_out + t * r.q_out_token_stride + h * r.q_out_head_stride
                   : (T*)r.k_out + t * r.k_out_token_stride + (h - r.heads) * r.k_out_head_stride;
      const float2* turns = angles + rows_token[i] * pairs;
      if (LAYOUT == CXS_ROTARY_HALF) {
        if (pair0 >= 0) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float a = to_float(x[i][0][e]), b = to_float(x[i][1][e]);
            const float2 c = turns[pair0 + e];
            x[i][0][e] = from_float<T>(a * c.x - b * c.y);
            x[i][1][e] = from_float<T>(b * c.x + a * c.y);
          }
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int pair = half ? pair1 : pair0;
          if (pair < 0) continue;
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float a = to_float(x[i][half][e]), b = to_float(x[i][half][e + 1]);
            const float2 c = turns[pair + e / 2];
            x[i][half][e] = from_float<T>(a * c.x - b * c.y);
            x[i][half][e + 1] = from_float<T>(b * c.x + a * c.y);
          }
        }
      }
      store<T, V>(dst + at0, x[i][0]);
      if (at1 >= 0) store<T, V>(dst + at1, x[i][1]);
    }
    if (token >= tokens) return;
    advance(kRows);
  }
}

template <typename T, int LAYOUT, int V>
int launch(const cxs_rotary_call& r, cudaStream_t stream) {
  Cut cut = {};
  const int heads = r.heads + r.kv_heads;
  if (LAYOUT == CXS_ROTARY_HALF) {
    cut.turned = r.rotary_dim / 2 / V;
    cut.units = cut.turned + ((r.dim - r.rotary_dim) / V + 1) / 2;
  } else {
    cut.units = (r.dim / V + 1) / 2;
  }
  const int rows = cut.units < 256 ? 256 / cut.units : 1;  // at a time
  cut.step_token = rows / heads;
  cut.step_head = rows % heads;
  // As many tokens as give every thread kRows rows, while that leaves CTAs
  // for the GPU (600: four on each SM) and the angles fit 16 KB.
  int tokens = (kRows * rows + heads - 1) / heads;
  const int spread = (r.tokens + 599) / 600, fit = 16384 / (r.rotary_dim / 2 * (int)sizeof(float2));
  if (tokens > spread) tokens = spread;
  if (tokens > fit) tokens = fit;
  if (tokens < 1) tokens = 1;
  cut.tokens = tokens;
  const int smem = tokens * (r.rotary_dim / 2) * sizeof(float2);
  rotary_kernel<T, LAYOUT, V><<<(r.tokens + tokens - 1) / tokens, dim3(cut.units, rows), smem,
                                stream>>>(r, cut);
  CXS_LAUNCH_CHECK("rotary");
  return CXS_OK;
}

// 16-byte vectors where every pointer and stride allows them and no vector
// holds both rotated and other channels, or straddles the half layout's
// halves; else single channels (pairs, interleaved).
template <typename T, int LAYOUT>
int dispatch(const cxs_rotary_call& r, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  unsigned long long bits = 0;
  if (r.heads)
    bits |= (uintptr_t)r.q | (uintptr_t)r.q_out |
            sizeof(T) * (r.q_token_stride | r.q_head_stride | r.q_out_token_stride |
                         r.q_out_head_stride);
  if (r.kv_heads)
    bits |= (uintptr_t)r.k | (uintptr_t)r.k_out |
            sizeof(T) * (r.k_token_stride | r.k_head_stride | r.k_out_token_stride |
                         r.k_out_head_stride);
  const int run = LAYOUT == CXS_ROTARY_HALF ? r.rotary_dim / 2 : r.rotary_dim;
  if (bits % 16 == 0 && r.dim % V == 0 && run % V == 0) return launch<T, LAYOUT, V>(r, stream);
  return launch<T, LAYOUT, LAYOUT == CXS_ROTARY_HALF ? 1 : 2>(r, stream);
}

}  // namespace

extern "C" int cxs_rotary(const cxs_rotary_call* call, void* stream) {
  if (!call) return set_error(CXS_ERR_INVALID, "rotary: null call");
  const cxs_rotary_call& r = *call;
  if (r.tokens < 0 || r.heads < 0 || r.kv_heads < 0)
    return set_error(CXS_ERR_INVALID, "rotary: negative sizes");
  if (r.dim < 2 || r.dim % 2 || r.dim > 512)
    return set_error(CXS_ERR_INVALID, "rotary: dim must be even and at most 512");
  if (r.rotary_dim < 2 || r.rotary_dim % 2 || r.rotary_dim > r.dim)
    return set_error(CXS_ERR_INVALID, "rotary: rotary_dim must be even and at most dim");
  if (r.layout != CXS_ROTARY_HALF && r.layout != CXS_ROTARY_INTERLEAVED)
    return set_error(CXS_ERR_INVALID, "rotary: unknown layout");
  if (r.type < CXS_TYPE_BF16 || r.type > CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "rotary: unknown type");
  if (r.heads > 65535 || r.kv_heads > 65535)
    return set_error(CXS_ERR_CAPACITY, "rotary: at most 65535 heads");
  if (r.tokens == 0 || r.heads + r.kv_heads == 0) return CXS_OK;
  if (!r.positions || !r.steps || (r.heads && (!r.q || !r.q_out)) ||
      (r.kv_heads && (!r.k || !r.k_out)))
    return set_error(CXS_ERR_INVALID, "rotary: null buffer");
  CXS_CACHE_TYPE(r.type, T, {
    if (r.layout == CXS_ROTARY_HALF)
      return dispatch<T, CXS_ROTARY_HALF>(r, (cudaStream_t)stream);
    return dispatch<T, CXS_ROTARY_INTERLEAVED>(r, (cudaStream_t)stream);
  });
}
