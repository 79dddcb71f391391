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

// One CTA per token, one thread per channel pair of a head.
template <typename T>
__global__ void rotary_kernel(const cxs_rotary_call r) {
  extern __shared__ float2 angles[];
  const long long token = blockIdx.x;
  const long long position = r.wide_positions ? ((const long long*)r.positions)[token]
                                              : ((const int*)r.positions)[token];
  const int pairs = r.rotary_dim / 2;
  for (int i = threadIdx.x; i < pairs; i += blockDim.x)
    angles[i] = turn((unsigned long long)position * (unsigned long long)r.steps[i], r.magnitude,
                     r.transpose);
  __syncthreads();
  const int half = r.dim / 2;
  for (int n = threadIdx.x; n < (r.heads + r.kv_heads) * half; n += blockDim.x) {
    int head = n / half, i = n % half;
    const T* x;
    T* y;
    if (head < r.heads) {
      x = (const T*)r.q + token * r.q_token_stride + head * r.q_head_stride;
      y = (T*)r.q_out + token * r.q_out_token_stride + head * r.q_out_head_stride;
    } else {
      head -= r.heads;
      x = (const T*)r.k + token * r.k_token_stride + head * r.k_head_stride;
      y = (T*)r.k_out + token * r.k_out_token_stride + head * r.k_out_head_stride;
    }
    if (i < pairs) {
      const int ia = r.layout == CXS_ROTARY_HALF ? i : 2 * i;
      const int ib = r.layout == CXS_ROTARY_HALF ? i + pairs : 2 * i + 1;
      const float a = to_float(x[ia]), b = to_float(x[ib]);
      const float2 t = angles[i];
      y[ia] = from_float<T>(a * t.x - b * t.y);
      y[ib] = from_float<T>(b * t.x + a * t.y);
    } else {
      y[2 * i] = x[2 * i];
      y[2 * i + 1] = x[2 * i + 1];
    }
  }
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
  const int smem = r.rotary_dim / 2 * sizeof(float2);
  CXS_CACHE_TYPE(r.type, T,
                 (rotary_kernel<T><<<r.tokens, 256, smem, (cudaStream_t)stream>>>(r)));
  CXS_LAUNCH_CHECK("rotary");
  return CXS_OK;
}
