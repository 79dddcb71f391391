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

// One page, head and part (K or V) per CTA: the page's new tokens' largest
// magnitude, the scale, and one pass that writes codes.
template <int FORMAT, typename T>
__global__ void append_kernel(const cxs_cache_call c, const T* __restrict__ k,
                              long long k_token, long long k_head, const T* __restrict__ v,
                              long long v_token, long long v_head, int reach) {
  using C = Code<FORMAT>;
  const int user = blockIdx.x / reach, step = blockIdx.x % reach;
  const int head = blockIdx.y, part = blockIdx.z;
  int bad = 0;
  const Rows rows = user_rows(c, user, &bad);
  long long start = (long long)c.lengths[user] - rows.count;
  const long long end = start + rows.count;
  const long long most = (long long)c.width * c.page_size;
  if (start < 0 || end > most) bad = 1;
  if (bad && step == 0 && head == 0 && part == 0 && threadIdx.x == 0)
    report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
  const long long from = start > 0 ? start : 0, to = end < most ? end : most;
  const long long low = (from / c.page_size + step) * c.page_size;  // position of slot 0
  if (from >= to || low >= to) return;
  const int page = c.table[user * c.table_stride + low / c.page_size];
  if (page < 0 || page >= c.pages) {
    if (head == 0 && part == 0 && threadIdx.x == 0) report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
    return;
  }
  const int fill = from > low ? (int)(from - low) : 0;  // slots of older tokens
  const int stop = to - low < c.page_size ? (int)(to - low) : c.page_size;
  const T* x = part ? v + head * v_head : k + head * k_head;
  const long long x_token = part ? v_token : k_token;
  x += (rows.first + low - start) * x_token;  // slot 0's row (slots below `fill` are not read)
  const long long cell = ((long long)page * c.kv_heads + head) * 2 + part;
  uint8_t* codes = (uint8_t*)c.codes + cell * c.page_size * c.dim;

  __shared__ float partial[32];
  float size = 0.f;
  for (int i = fill * c.dim + threadIdx.x; i < stop * c.dim; i += blockDim.x) {
    const float a = fabsf(to_float(x[(i / c.dim) * x_token + i % c.dim]));
    if (a < INFINITY) size = fmaxf(size, a);  // neither infinity nor NaN
  }
  for (int o = 16; o; o >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, o));
  if (threadIdx.x % 32 == 0) partial[threadIdx.x / 32] = size;
  __syncthreads();
  for (int w = 0; w < blockDim.x / 32; ++w) size = fmaxf(size, partial[w]);
  const float before = fill ? c.scales[cell] : 0.f;
  const float scale = fmaxf(fmaxf(size * C::kInverseTop, kLeastScale), before);
  const float inverse = 1.f / scale;
  for (int i = fill * c.dim + threadIdx.x; i < stop * c.dim; i += blockDim.x)
    codes[i] = C::encode(to_float(x[(i / c.dim) * x_token + i % c.dim]) * inverse);
  if (fill && scale > before) {
    const float ratio = before / scale;
    for (int i = threadIdx.x; i < fill * c.dim; i += blockDim.x)
      codes[i] = C::encode(C::decode(codes[i]) * ratio);
  }
  __syncthreads();  // every thread has read the older scale
  if (threadIdx.x == 0) c.scales[cell] = scale;
}

// One page and head per CTA.
template <int FORMAT, typename T>
__global__ void read_kernel(const cxs_cache_call c, T* __restrict__ k, T* __restrict__ v,
                            int reach) {
  using C = Code<FORMAT>;
  const int user = blockIdx.x / reach, step = blockIdx.x % reach, head = blockIdx.y;
  int bad = 0;
  const Rows rows = user_rows(c, user, &bad);
  const long long start = c.lengths[user], end = start + rows.count;
  const long long most = (long long)c.width * c.page_size;
  if (start < 0 || end > most) bad = 1;
  if (bad && step == 0 && head == 0 && threadIdx.x == 0)
    report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
  // Pages are counted from the one (possibly before the first) that holds `start`.
  const long long block = (start >= 0 ? start / c.page_size
                                      : -((-start + c.page_size - 1) / c.page_size)) + step;
  const long long low = block * c.page_size;
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
  for (int part = 0; part < 2; ++part) {
    const long long cell = ((long long)page * c.kv_heads + head) * 2 + part;
    const uint8_t* codes = (const uint8_t*)c.codes + cell * c.page_size * c.dim;
    const float scale = page < 0 ? 0.f : c.scales[cell];
    T* out = part ? v : k;
    for (int i = fill * c.dim + threadIdx.x; i < stop * c.dim; i += blockDim.x) {
      const long long row = rows.first + low + i / c.dim - start;
      out[(row * c.kv_heads + head) * c.dim + i % c.dim] =
          from_float<T>(page < 0 ? 0.f : C::decode(codes[i]) * scale);
    }
  }
}

}  // namespace

extern "C" int cxs_cache_append(const cxs_cache_call* call, const void* k, int64_t k_token_stride,
                                int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                int64_t v_head_stride, void* stream) {
  int status = cxs_host::check_cache(call, "cache append");
  if (status != CXS_OK) return status;
  if (call->users == 0 || call->tokens == 0 || call->max_tokens == 0) return CXS_OK;
  status = cxs_host::check_cache_pointers(call, "cache append");
  if (status != CXS_OK) return status;
  if (!k || !v) return set_error(CXS_ERR_INVALID, "cache append: null keys or values");
  const int reach = (call->max_tokens + call->page_size - 2) / call->page_size + 1;
  if ((long long)call->users * reach > 0x7fffffffll)
    return set_error(CXS_ERR_CAPACITY, "cache append: too many pages in one call");
  const dim3 grid(call->users * reach, call->kv_heads, 2);
  CXS_CACHE_FORMAT(call->format, F,
                   CXS_CACHE_TYPE(call->type, T,
                                  (append_kernel<F, T><<<grid, 256, 0, (cudaStream_t)stream>>>(
                                      *call, (const T*)k, k_token_stride, k_head_stride,
                                      (const T*)v, v_token_stride, v_head_stride, reach))));
  CXS_LAUNCH_CHECK("cache append");
  return CXS_OK;
}

extern "C" int cxs_cache_read(const cxs_cache_call* call, void* k, void* v, void* stream) {
  int status = cxs_host::check_cache(call, "cache read");
  if (status != CXS_OK) return status;
  if (call->users == 0 || call->tokens == 0 || call->max_tokens == 0) return CXS_OK;
  status = cxs_host::check_cache_pointers(call, "cache read");
  if (status != CXS_OK) return status;
  if (!k || !v) return set_error(CXS_ERR_INVALID, "cache read: null output");
  const int reach = (call->max_tokens + call->page_size - 2) / call->page_size + 1;
  if ((long long)call->users * reach > 0x7fffffffll)
    return set_error(CXS_ERR_CAPACITY, "cache read: too many pages in one call");
  const dim3 grid(call->users * reach, call->kv_heads);
  CXS_CACHE_FORMAT(
      call->format, F,
      CXS_CACHE_TYPE(call->type, T,
                     (read_kernel<F, T><<<grid, 256, 0, (cudaStream_t)stream>>>(
                         *call, (T*)k, (T*)v, reach))));
  CXS_LAUNCH_CHECK("cache read");
  return CXS_OK;
}
