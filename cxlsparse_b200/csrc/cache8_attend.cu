// Attention over the dense 8-bit cache.
#include "cache8.cuh"

using cxs_host::set_error;

namespace {

using namespace cxs::cache8;

constexpr float kLog2e = 1.4426950408889634f;

// One warp per packed row and query head: lanes take 32 keys at a time for
// the scores, then D / 32 channels each for the sum of values.
template <int FORMAT, typename T, int D>
__global__ void attend_kernel(const cxs_cache_attend_call a) {
  using C = Code<FORMAT>;
  const cxs_cache_call& c = a.cache;
  __shared__ float q_rows[4][D];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int head = blockIdx.y * 4 + warp;
  if (head >= a.heads) return;
  const int row = blockIdx.x;
  // The row's user: the last one whose rows start at or before it.
  int user = row;
  if (c.offsets) {
    int lo = 0, hi = c.users - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (c.offsets[mid] <= row) lo = mid; else hi = mid - 1;
    }
    user = lo;
  }
  int bad = 0;
  const Rows rows = user_rows(c, user, &bad);
  const long long most = (long long)c.width * c.page_size;
  long long length = c.lengths[user];
  const long long position = length - rows.count + (row - rows.first);
  if (length > most) { bad = 1; length = most; }
  if (bad && lane == 0) report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
  long long end = a.causal && position + 1 < length ? position + 1 : length;
  long long begin = a.window > 0 && position - a.window + 1 > 0 ? position - a.window + 1 : 0;
  if (row < rows.first || row >= rows.first + rows.count) end = 0;
  const int kv_head = head / (a.heads / c.kv_heads);
  const T* q = (const T*)a.query + row * a.q_token_stride + head * a.q_head_stride;
  for (int d = lane; d < D; d += 32) q_rows[warp][d] = to_float(q[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  for (long long base = begin; base < end; base += 32) {
    const long long key = base + lane;
    float s = -INFINITY, sv = 0.f;
    const uint8_t* values = nullptr;
    if (key < end) {
      const int page = c.table[user * c.table_stride + key / c.page_size];
      if (page < 0 || page >= c.pages) {
        report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
      } else {
        const long long cell = ((long long)page * c.kv_heads + kv_head) * 2;
        const uint8_t* keys = (const uint8_t*)c.codes + (cell * c.page_size + key % c.page_size) * D;
        values = keys + c.page_size * D;
        float dot = 0.f;
        for (int d = 0; d < D; ++d) dot = fmaf(q_rows[warp][d], C::decode(keys[d]), dot);
        s = dot * (usable_scale(c.scales[cell]) * a.scale);
        sv = usable_scale(c.scales[cell + 1]);
      }
    }
    float top = s;
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    top = fmaxf(top, m);
    const float base_m = top == -INFINITY ? 0.f : top;
    const float p = values ? exp2f((s - base_m) * kLog2e) : 0.f;
    const float factor = exp2f((m - base_m) * kLog2e);
    float sum = p;
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * factor + sum;
    m = top;
    for (int e = 0; e < D / 32; ++e) o[e] *= factor;
    for (int j = 0; j < 32; ++j) {
      const unsigned long long at =
          __shfl_sync(0xffffffffu, (unsigned long long)values, j);
      const float w = __shfl_sync(0xffffffffu, p * sv, j);
      if (!at) continue;
      for (int e = 0; e < D / 32; ++e)
        o[e] = fmaf(w, C::decode(((const uint8_t*)at)[e * 32 + lane]), o[e]);
    }
  }
  const bool some = !(l == 0.f);
  T* out = (T*)a.out + ((long long)row * a.heads + head) * D;
  for (int e = 0; e < D / 32; ++e) out[e * 32 + lane] = from_float<T>(some ? o[e] / l : 0.f);
  if (a.lse && lane == 0)
    a.lse[(long long)row * a.heads + head] = some ? m + logf(l) : -INFINITY;
}

int check_attend(const cxs_cache_attend_call* a) {
  if (!a) return set_error(CXS_ERR_INVALID, "cache attend: null call");
  const int status = cxs_host::check_cache(&a->cache, "cache attend");
  if (status != CXS_OK) return status;
  if (a->cache.type == CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "cache attend: queries must be bf16 or fp16");
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return set_error(CXS_ERR_INVALID, "cache attend: heads must be a multiple of kv_heads");
  if (a->window < 0) return set_error(CXS_ERR_INVALID, "cache attend: negative window");
  return CXS_OK;
}

}  // namespace

extern "C" int cxs_cache_attend_workspace(const cxs_cache_attend_call* call, int64_t* bytes) {
  const int status = check_attend(call);
  if (status != CXS_OK) return status;
  if (!bytes) return set_error(CXS_ERR_INVALID, "cache attend: null result");
  *bytes = 0;
  return CXS_OK;
}

extern "C" int cxs_cache_attend(const cxs_cache_attend_call* call, void* stream) {
  int status = check_attend(call);
  if (status != CXS_OK) return status;
  const cxs_cache_call& c = call->cache;
  if (c.tokens == 0) return CXS_OK;
  if (c.users == 0) return set_error(CXS_ERR_INVALID, "cache attend: rows without users");
  status = cxs_host::check_cache_pointers(&c, "cache attend");
  if (status != CXS_OK) return status;
  if (!call->query || !call->out) return set_error(CXS_ERR_INVALID, "cache attend: null query or out");
  const dim3 grid(c.tokens, (call->heads + 3) / 4);
  CXS_CACHE_FORMAT(c.format, F, CXS_CACHE_TYPE(c.type, T, if (c.dim == 64) {
                     attend_kernel<F, T, 64><<<grid, 128, 0, (cudaStream_t)stream>>>(*call);
                   } else {
                     attend_kernel<F, T, 128><<<grid, 128, 0, (cudaStream_t)stream>>>(*call);
                   }));
  CXS_LAUNCH_CHECK("cache attend");
  return CXS_OK;
}
