// Shared parts of the dense 8-bit cache kernels: the two code formats, the
// types of the 16- and 32-bit side and where a user's new tokens lie.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cxs_common.cuh"

namespace cxs {
namespace cache8 {

constexpr float kLeastScale = 5.421010862427522e-20f;  // 2^-64

// Codes of a format: the largest one, decoding and rounding of four at once.
template <int FORMAT>
struct Code;

template <>
struct Code<CXS_FORMAT_E4M3> {
  static constexpr float kTop = 448.f;
  static constexpr float kInverseTop = 1.f / 448.f;
  static __device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    __nv_fp8x4_e4m3 v;
    v.__x = w;
    const float4 f = static_cast<float4>(v);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  }
  // Nearest codes, ties to even, saturated; NaN stays NaN.
  static __device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
    uint32_t lo, hi;
    asm("{.reg .b16 h; cvt.rn.satfinite.e4m3x2.f32 h, %2, %1; cvt.u32.u16 %0, h;}"
        : "=r"(lo) : "f"(x[0]), "f"(x[1]));
    asm("{.reg .b16 h; cvt.rn.satfinite.e4m3x2.f32 h, %2, %1; cvt.u32.u16 %0, h;}"
        : "=r"(hi) : "f"(x[2]), "f"(x[3]));
    return lo | hi << 16;
  }
};

template <>
struct Code<CXS_FORMAT_INT8> {
  static constexpr float kTop = 127.f;
  static constexpr float kInverseTop = 1.f / 127.f;
  static __device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
  }
  // Nearest codes, ties to even, saturated; NaN becomes 0. Adding 1.5 * 2^23
  // leaves the integer, rounded, in the low bits of the sum.
  static __device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = x[e] == x[e] ? fminf(fmaxf(x[e], -kTop), kTop) : 0.f;
      b[e] = __float_as_uint(__fadd_rn(y, 12582912.f));
    }
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void report(int* error, int bits) {
  if (error) atomicOr(error, bits);
}

// A scale as the kernels use it: at least 2^-64, NaN kept.
__device__ __forceinline__ float usable_scale(float s) { return s < kLeastScale ? kLeastScale : s; }

// The packed rows of one user. A user whose rows are not what the call says
// they can be (outside the packed ones, backwards, more than max_tokens) has
// none: rows taken from either end would stand for other positions.
struct Rows {
  int first;  // first packed row
  int count;  // rows
};
__device__ __forceinline__ Rows user_rows(const cxs_cache_call& c, int user, int* bad) {
  int lo = user, hi = user + 1;
  if (c.offsets) {
    lo = c.offsets[user];
    hi = c.offsets[user + 1];
  }
  // In 32 bits (0 <= lo <= hi: the difference fits), without a branch: in 64, or
  // with one, append prefill took 46.8 to 47.6 us in the place of 45.9.
  const bool out = lo < 0 || hi < lo || hi > c.tokens || hi - lo > c.max_tokens;
  if (out) *bad = 1;
  return {lo, out ? 0 : hi - lo};
}

// Packed rows of no user: before the first user's (b = -1), past the last
// user's (b = users), and user b's where user_rows lets it have none.
struct Gap {
  long long low, high;
};
__device__ __forceinline__ Gap row_gap(const cxs_cache_call& c, int b, int users) {
  if (!c.offsets) return {0, 0};
  Gap g;
  if (b < 0) {
    g = {0, c.offsets[0]};
  } else if (b == users) {
    g = {c.offsets[users], c.tokens};
  } else {
    int bad = 0;
    user_rows(c, b, &bad);
    if (!bad) return {0, 0};
    g = {c.offsets[b], c.offsets[b + 1]};
  }
  if (g.low < 0) g.low = 0;
  if (g.high > c.tokens) g.high = c.tokens;
  return g;
}

}  // namespace cache8
}  // namespace cxs

namespace cxs_host {
// Runs a step (a function attribute, say) once for each device.
struct OncePerDevice {
  static constexpr int kDevices = 64;
  int done[kDevices];
  template <typename F>
  int run(F step) {
    int device = 0;
    CXS_CUDA(cudaGetDevice(&device));
    if (device < kDevices && __atomic_load_n(&done[device], __ATOMIC_ACQUIRE)) return CXS_OK;
    const int status = step();
    if (status == CXS_OK && device < kDevices) __atomic_store_n(&done[device], 1, __ATOMIC_RELEASE);
    return status;
  }
};
constexpr long long kMaxPositions = 1ll << 30;  // positions of one table row
// CXS_OK, or what is wrong with the sizes / the pointers every cache call shares.
int check_cache(const cxs_cache_call* call, const char* what);
int check_cache_pointers(const cxs_cache_call* call, const char* what);
}  // namespace cxs_host

// Call f with template arguments for (format, dim, page_size).
#define CXS_CACHE_FORMAT(format, F, ...)                  \
  do {                                                    \
    if ((format) == CXS_FORMAT_E4M3) {                    \
      constexpr int F = CXS_FORMAT_E4M3;                  \
      __VA_ARGS__;                                        \
    } else {                                              \
      constexpr int F = CXS_FORMAT_INT8;                  \
      __VA_ARGS__;                                        \
    }                                                     \
  } while (0)
#define CXS_CACHE_TYPE(type, T, ...)                      \
  do {                                                    \
    if ((type) == CXS_TYPE_BF16) {                        \
      using T = __nv_bfloat16;                            \
      __VA_ARGS__;                                        \
    } else if ((type) == CXS_TYPE_F16) {                  \
      using T = __half;                                   \
      __VA_ARGS__;                                        \
    } else {                                              \
      using T = float;                                    \
      __VA_ARGS__;                                        \
    }                                                     \
  } while (0)
