// Writing tokens into the dense 8-bit cache and reading them back.
#include "cache8.cuh"

using cxs_host::set_error;

namespace cxs_host {

int check_cache(const cxs_cache_call* c, const char* what) {
  if (!c) return set_error(CXS_ERR_INVALID, "%s: null call", what);
  if (c->pages < 1 || c->kv_heads < 1 || c->users < 0 || c->width < 1 || c->tokens < 0 ||
      c->max_tokens < 0)
    return set_error(CXS_ERR_INVALID, "%s: invalid sizes", what);
  if (c->dim != 64 && c->dim != 128)
    return set_error(CXS_ERR_INVALID, "%s: dim must be 64 or 128", what);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64)
    return set_error(CXS_ERR_INVALID, "%s: page_size must be 16, 32 or 64", what);
  if (c->format != CXS_FORMAT_E4M3 && c->format != CXS_FORMAT_INT8)
    return set_error(CXS_ERR_INVALID, "%s: unknown format", what);
  if (c->type < CXS_TYPE_BF16 || c->type > CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "%s: unknown type", what);
  if (c->table_stride < 0 || (c->users > 1 && c->table_stride < c->width))
    return set_error(CXS_ERR_INVALID, "%s: table rows overlap", what);
  if ((long long)c->width * c->page_size > kMaxPositions)
    return set_error(CXS_ERR_CAPACITY, "%s: more than 2^30 positions in a table row", what);
  if (c->users > 65535 || c->kv_heads > 32767)
    return set_error(CXS_ERR_CAPACITY, "%s: at most 65535 users and 32767 heads", what);
  if (!c->offsets && c->tokens != c->users)
    return set_error(CXS_ERR_INVALID, "%s: without offsets every user has one token", what);
  if (!c->offsets && c->tokens > 0 && c->max_tokens < 1)
    return set_error(CXS_ERR_INVALID, "%s: without offsets max_tokens must not be 0", what);
  return CXS_OK;
}

int check_cache_pointers(const cxs_cache_call* c, const char* what) {
  if (!c->codes || !c->scales || !c->table || !c->lengths)
    return set_error(CXS_ERR_INVALID, "%s: null cache buffer", what);
  if ((uintptr_t)c->codes % 16)
    return set_error(CXS_ERR_INVALID, "%s: codes must be 16-byte aligned", what);
  return CXS_OK;
}

}  // namespace cxs_host

namespace {

using namespace cxs::cache8;

// Sixteen consecutive values, 16 bytes at a time where `wide` allows it.
template <typename T>
__device__ __forceinline__ void load16(float (&x)[16], const T* from, bool wide) {
  alignas(16) T in[16];
  if (wide) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i)
      reinterpret_cast<uint4*>(in)[i] = reinterpret_cast<const uint4*>(from)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) in[e] = from[e];
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = to_float(in[e]);
}

// Pages that a user's new tokens reach at most, wherever they start: a user has
// no more rows than there are, whatever max_tokens says.
int most_pages(const cxs_cache_call& c) {
  const long long most = c.max_tokens < c.tokens ? c.max_tokens : c.tokens;
  return (int)((most + c.page_size - 2) / c.page_size) + 1;
}

// One page, head and part (K or V) per CTA, 16 channels of a slot per thread:
// the values are read once, kept in registers while the CTA finds the largest
// magnitude, then written as codes, 16 bytes a thread. Memory-bound (2 or 4
// bytes in, 1 out): a page's CTA has all its loads in flight at once, and
// several CTAs share an SM, so one's reduction hides under the others' loads.
// Older codes are touched only where the page's scale grows. Measured: 4 x 8192
// tokens of 8 heads of 128, bf16 to e4m3, 201 MB in 46 us (4.4 TB/s), a token
// each of 8 users in 2.2 us.
template <int FORMAT, typename T>
__global__ void __launch_bounds__(512, 4)  // four of the largest CTAs on an SM (three: 51 us)
    append_kernel(const cxs_cache_call c, const T* __restrict__ k, long long k_token,
                  long long k_head, const T* __restrict__ v, long long v_token, long long v_head,
                  int page_bits) {
  using C = Code<FORMAT>;
  const int step = blockIdx.x, head = blockIdx.y >> 1, part = blockIdx.y & 1, user = blockIdx.z;
  int bad = 0;
  const Rows rows = user_rows(c, user, &bad);
  const int most = c.width << page_bits;
  const int length = c.lengths[user];
  const long long start = (long long)length - rows.count;  // of the new tokens
  if (start < 0 || length > most) bad = 1;
  if (bad && step == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
  const int from = start > 0 ? (int)start : 0, to = min(length, most);
  // Position of slot 0; unsigned, as a page past the last may lie past 2^31.
  const int block = (from >> page_bits) + step;
  if (rows.count == 0 || from >= to || (unsigned)block << page_bits >= (unsigned)to) return;
  const int low = block << page_bits;
  const int fill = max(from - low, 0);                 // slots of older tokens
  const int stop = min(to - low, 1 << page_bits);
  const int chunk_bits = c.dim == 64 ? 2 : 3;
  const int slot = threadIdx.x >> chunk_bits;
  const int channel = (threadIdx.x & ((1 << chunk_bits) - 1)) * 16;
  const bool fresh = slot >= fill && slot < stop, old = slot < fill;
  const int page = c.table[user * c.table_stride + block];

  float x[16];
  float size = 0.f;
  if (fresh) {
    const T* row = part ? v + head * v_head : k + head * k_head;
    row += (rows.first + (low - start) + slot) * (part ? v_token : k_token) + channel;
    load16(x, row, ((uintptr_t)row & 15) == 0);
#pragma unroll
    for (int e = 0; e < 16; ++e) size = fmaxf(size, fabsf(x[e]));  // (passes over NaN)
  }
  if (page < 0 || page >= c.pages) {
    if (blockIdx.y == 0 && threadIdx.x == 0) report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
    return;
  }
  const long long cell = ((long long)page * c.kv_heads + head) * 2 + part;
  uint4* codes = (uint4*)((uint8_t*)c.codes + cell * c.page_size * c.dim) + threadIdx.x;
  const float before = fill ? c.scales[cell] : 0.f;
  __shared__ float partial[2][16];
  auto largest = [&](float mine, float* slots) {
    for (int o = 16; o; o >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (threadIdx.x % 32 == 0) slots[threadIdx.x / 32] = mine;
    __syncthreads();
    for (int w = 0; w < blockDim.x / 32; ++w) mine = fmaxf(mine, slots[w]);
    return mine;
  };
  size = largest(size, partial[0]);  // (and every thread has read the older scale)
  if (size == INFINITY) {            // rare: the largest finite magnitude
    size = 0.f;
    if (fresh)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (fabsf(x[e]) < INFINITY) size = fmaxf(size, fabsf(x[e]));
    size = largest(size, partial[1]);
  }
  const float scale = fmaxf(fmaxf(size * C::kInverseTop, kLeastScale), before);
  if (threadIdx.x == 0) c.scales[cell] = scale;
  float factor;
  if (fresh) {
    factor = 1.f / scale;
  } else if (old && scale > before) {
    factor = before / scale;
    const uint4 w = *codes;
    float y[4];
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      C::decode4(in[i], y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
    }
  } else {
    return;
  }
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y[4] = {x[4 * i] * factor, x[4 * i + 1] * factor, x[4 * i + 2] * factor,
                        x[4 * i + 3] * factor};
    out[i] = C::encode4(y);
  }
  *codes = make_uint4(out[0], out[1], out[2], out[3]);
}

// One page and head per CTA: K and V of a page are one run of bytes. A thread
// reads as many codes as make 16 bytes of the result (a warp's stores are then
// whole lines), kUnroll times at once. Memory-bound: 1 byte in, 2 or 4 out.
// Measured: four histories to 16K, 8 heads of 128, int8 to fp16, 262 MB in 46 us
// (5.7 TB/s; 52 us with 32 bytes of the result a thread). Rows of no user are
// cleared by the CTAs of a user beside them.
constexpr int kReadThreads = 128, kUnroll = 8;

template <int FORMAT, typename T>
__global__ void __launch_bounds__(kReadThreads)
    read_kernel(const cxs_cache_call c, T* __restrict__ k, T* __restrict__ v, int page_bits) {
  using C = Code<FORMAT>;
  const int step = blockIdx.x, head = blockIdx.y, user = blockIdx.z;
  int bad = 0;
  const Rows rows = user_rows(c, user, &bad);
  const int start = c.lengths[user], most = c.width << page_bits;
  const long long end = (long long)start + rows.count;
  if (start < 0 || end > most) bad = 1;
  if (bad && step == 0 && head == 0 && threadIdx.x == 0)
    report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
  constexpr int kCodes = 16 / sizeof(T), kCodeBits = kCodes == 8 ? 3 : 2;  // of a unit
  const int unit_bits = (c.dim == 64 ? 6 : 7) - kCodeBits;               // units of a row
  const auto clear = [&](const Gap& gap) {  // every gridDim.x-th row of it
    for (long long row = gap.low + step; row < gap.high; row += gridDim.x)
      for (int n = threadIdx.x; n < 2 << unit_bits; n += kReadThreads) {
        const int channel = (n & ((1 << unit_bits) - 1)) << kCodeBits;
        T* const to = (n >> unit_bits ? v : k) + (row * c.kv_heads + head) * c.dim + channel;
        *(uint4*)to = make_uint4(0, 0, 0, 0);
      }
  };
  if (user == 0) clear(row_gap(c, -1, c.users));
  if (bad) clear(row_gap(c, user, c.users));
  if (user == c.users - 1) clear(row_gap(c, c.users, c.users));
  // Pages are counted from the one (possibly before the first) that holds `start`.
  const int block = (start >> page_bits) + step;
  const long long low = (long long)block << page_bits;
  if (low >= end) return;
  const int fill = start > low ? (int)(start - low) : 0;
  const int stop = end - low < c.page_size ? (int)(end - low) : c.page_size;
  int page = -1;
  if (low >= 0 && low < most) {
    page = c.table[user * c.table_stride + block];
    if (page < 0 || page >= c.pages) {
      page = -1;
      if (head == 0 && threadIdx.x == 0) report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
    }
  }
  const long long cell = ((long long)(page < 0 ? 0 : page) * c.kv_heads + head) * 2;
  const float scale_k = page < 0 ? 0.f : c.scales[cell];
  const float scale_v = page < 0 ? 0.f : c.scales[cell + 1];
  const uint8_t* codes = (const uint8_t*)c.codes + cell * c.page_size * c.dim;
  const int half = 1 << (page_bits + unit_bits);
  const long long row0 = rows.first + (low - start);
  for (int base = threadIdx.x; base < 2 * half; base += kReadThreads * kUnroll) {
    uint32_t w[kUnroll][kCodes / 4];
    bool live[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int n = base + i * kReadThreads, slot = (n & (half - 1)) >> unit_bits;
      live[i] = n < 2 * half && slot >= fill && slot < stop;
#pragma unroll
      for (int j = 0; j < kCodes / 4; ++j) w[i][j] = 0;
      if (live[i] && page >= 0) {
        if constexpr (kCodes == 8) {
          const uint2 in = __ldcs(reinterpret_cast<const uint2*>(codes) + n);
          w[i][0] = in.x;
          w[i][1] = in.y;
        } else {
          w[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(codes) + n);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (!live[i]) continue;
      const int n = base + i * kReadThreads;
      const bool second = n >= half;
      const int slot = (n & (half - 1)) >> unit_bits;
      const int channel = (n & ((1 << unit_bits) - 1)) << kCodeBits;
      const float scale = second ? scale_v : scale_k;
      alignas(16) T out[kCodes];
#pragma unroll
      for (int j = 0; j < kCodes / 4; ++j) {
        float x[4];
        C::decode4(w[i][j], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * j + e] = from_float<T>(x[e] * scale);
      }
      *(uint4*)((second ? v : k) + ((row0 + slot) * c.kv_heads + head) * c.dim + channel) =
          *reinterpret_cast<const uint4*>(out);
    }
  }
}

}  // namespace

extern "C" int cxs_cache_append(const cxs_cache_call* call, const void* k, int64_t k_token_stride,
                                int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                int64_t v_head_stride, void* stream) {
  int status = cxs_host::check_cache(call, "cache append");
  if (status != CXS_OK) return status;
  if (call->users == 0 || call->tokens == 0) return CXS_OK;
  status = cxs_host::check_cache_pointers(call, "cache append");
  if (status != CXS_OK) return status;
  if (!k || !v) return set_error(CXS_ERR_INVALID, "cache append: null keys or values");
  const dim3 grid(most_pages(*call), call->kv_heads * 2, call->users);
  const int page_bits = call->page_size == 16 ? 4 : call->page_size == 32 ? 5 : 6;
  const int threads = call->page_size * call->dim / 16;
  CXS_CACHE_FORMAT(call->format, F,
                   CXS_CACHE_TYPE(call->type, T,
                                  (append_kernel<F, T><<<grid, threads, 0, (cudaStream_t)stream>>>(
                                      *call, (const T*)k, k_token_stride, k_head_stride,
                                      (const T*)v, v_token_stride, v_head_stride, page_bits))));
  CXS_LAUNCH_CHECK("cache append");
  return CXS_OK;
}

extern "C" int cxs_cache_read(const cxs_cache_call* call, void* k, void* v, void* stream) {
  int status = cxs_host::check_cache(call, "cache read");
  if (status != CXS_OK) return status;
  if (call->tokens == 0) return CXS_OK;
  if (!k || !v) return set_error(CXS_ERR_INVALID, "cache read: null output");
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16)
    return set_error(CXS_ERR_INVALID, "cache read: outputs must be 16-byte aligned");
  if (call->users == 0) {  // rows of no user
    const size_t bytes = (size_t)call->tokens * call->kv_heads * call->dim *
                         (call->type == CXS_TYPE_F32 ? 4 : 2);
    CXS_CUDA(cudaMemsetAsync(k, 0, bytes, (cudaStream_t)stream));
    CXS_CUDA(cudaMemsetAsync(v, 0, bytes, (cudaStream_t)stream));
    return CXS_OK;
  }
  status = cxs_host::check_cache_pointers(call, "cache read");
  if (status != CXS_OK) return status;
  const dim3 grid(most_pages(*call), call->kv_heads, call->users);
  const int page_bits = call->page_size == 16 ? 4 : call->page_size == 32 ? 5 : 6;
  CXS_CACHE_FORMAT(
      call->format, F,
      CXS_CACHE_TYPE(call->type, T,
                     (read_kernel<F, T><<<grid, kReadThreads, 0, (cudaStream_t)stream>>>(
                         *call, (T*)k, (T*)v, page_bits))));
  CXS_LAUNCH_CHECK("cache read");
  return CXS_OK;
}
