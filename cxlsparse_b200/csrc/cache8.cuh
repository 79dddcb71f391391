// Shared parts of the dense 8-bit cache kernels: the two code formats, the
// types of the 16- and 32-bit side and where a user's new tokens lie.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cxs_common.cuh"

namespace cxs {
namespace cache8 {

constexpr float kLeastScale = 5.421010862427522e-20f;  // 2^-64

// Codes of a format: the largest one, decoding and rounding.
template <int FORMAT>
struct Code;

template <>
struct Code<CXS_FORMAT_E4M3> {
  static constexpr float kTop = 448.f;
  static constexpr float kInverseTop = 1.f / 448.f;
  static __device__ __forceinline__ float decode(uint8_t c) {
    __nv_fp8_e4m3 v;
    v.__x = c;
    return static_cast<float>(v);
  }
  // Nearest code, ties to even, saturated; NaN stays NaN.
  static __device__ __forceinline__ uint8_t encode(float x) {
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
};

template <>
struct Code<CXS_FORMAT_INT8> {
  static constexpr float kTop = 127.f;
  static constexpr float kInverseTop = 1.f / 127.f;
  static __device__ __forceinline__ float decode(uint8_t c) {
    return static_cast<float>(static_cast<int8_t>(c));
  }
  // Nearest code, ties to even, saturated; NaN becomes 0.
  static __device__ __forceinline__ uint8_t encode(float x) {
    if (!(x == x)) return 0;
    return static_cast<uint8_t>(
        static_cast<int8_t>(__float2int_rn(fminf(fmaxf(x, -kTop), kTop))));
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

// The packed rows of one user, cut to what the call says they can be.
struct Rows {
  int first;  // first packed row
  int count;  // rows
};
__device__ __forceinline__ Rows user_rows(const cxs_cache_call& c, int user, int* bad) {
  long long lo = user, hi = user + 1;
  if (c.offsets) {
    lo = c.offsets[user];
    hi = c.offsets[user + 1];
  }
  if (lo < 0 || hi < lo || hi > c.tokens || hi - lo > c.max_tokens) {
    *bad = 1;
    if (hi > c.tokens) hi = c.tokens;
    if (lo < 0 || hi < lo) return {kInt32Max, 0};
    if (hi - lo > c.max_tokens) hi = lo + c.max_tokens;
  }
  return {static_cast<int>(lo), static_cast<int>(hi - lo)};
}

}  // namespace cache8
}  // namespace cxs

namespace cxs_host {
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
