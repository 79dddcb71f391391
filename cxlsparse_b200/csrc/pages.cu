// Sequences over the pages of a dense 8-bit cache: extending, forking, freeing
// and compacting them on the device.
//
// State: table [sequences, width] page ids (-1: none), lengths, references
// (table entries that name a page; 0: free) and lowest, below which no page is
// free. Pages are handed out lowest id first, in the order of the sequences (or
// children), so results do not depend on timing. What decides a call runs in one
// CTA (validation, a scan over the sequences, a search for free pages from
// `lowest` on) and changes nothing where the call cannot be carried out; rows
// and page contents, of all layers at once, are then copied by a second launch
// over the whole device.
#include <limits.h>

#include "cache8.cuh"

using cxs_host::set_error;

namespace {

using cxs::cache8::report;

constexpr int kPlanThreads = 1024, kWarps = kPlanThreads / 32;
constexpr int kScan = 16;           // pages a thread looks at in one round
constexpr int kApplyThreads = 256;
constexpr int kRowChunk = 128;      // table entries a warp copies at a time

// Workspace: int32 arrays.
struct Work {
  int* copies;   // [1] pages to copy
  int* source;   // [slots] of each copy
  int* target;
  int* fill;     // [slots] slots of the page to copy
  int* first;    // [sequences + 1] pages handed out before each sequence or child
  int* size;     // [sequences] tokens of each child
  int* claim;    // [sequences]
  int* moved;    // [pages] new id of a page
};
__host__ __device__ inline long long slots_of(const cxs_pages_call& c) {
  return c.pages > c.sequences ? c.pages : c.sequences;
}
__host__ __device__ inline long long work_ints(const cxs_pages_call& c) {
  return 4 + 3 * slots_of(c) + 3ll * c.sequences + 1 + c.pages;
}
__device__ inline Work work_of(const cxs_pages_call& c) {
  Work w;
  const long long n = slots_of(c);
  w.copies = (int*)c.workspace;
  w.source = w.copies + 4;
  w.target = w.source + n;
  w.fill = w.target + n;
  w.first = w.fill + n;
  w.size = w.first + c.sequences + 1;
  w.claim = w.size + c.sequences;
  w.moved = w.claim + c.sequences;
  return w;
}

// Sum of v over the threads before this one, and over all of them.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int sums[kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();  // (the sums of the scan before have been read)
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  int all = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const int before = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);
  return sum - v + (warp > 0 ? before : 0);
}

// Calls found(page, rank) for the pages of [low, high) that are free (or, with
// `used`, not), ranks counted from 0 in the order of the ids, until `most` have
// been found. Returns how many there were. For the whole CTA.
template <typename F>
__device__ int find_pages(const int* references, int low, int high, bool used, int most, F found) {
  int count = 0;
  for (long long base = low; base < high && count < most; base += kPlanThreads * kScan) {
    const long long at = base + (long long)threadIdx.x * kScan;
    unsigned hit = 0;
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      const int r = at + e < high ? references[at + e] : used ? 0 : 1;
      hit |= (unsigned)((r > 0) == used) << e;
    }
    int all;
    int rank = count + block_scan(__popc(hit), &all);
    for (; hit; hit &= hit - 1, ++rank)
      if (rank < most) found((int)at + __ffs(hit) - 1, rank);
    count += all;
  }
  return count;
}

// Takes the `total` lowest free pages into `fresh`; false (and reported): there
// are not that many.
__device__ bool take_pages(const cxs_pages_call& c, int total, int* fresh) {
  if (total == 0) return true;
  const int n = find_pages(c.references, max(*c.lowest, 0), c.pages, false, total,
                           [&](int page, int rank) { fresh[rank] = page; });
  if (n < total) {
    if (threadIdx.x == 0) report(c.error, CXS_DEVICE_ERR_NO_PAGES);
    return false;
  }
  __syncthreads();
  return true;
}

__device__ __forceinline__ int pages_for(long long tokens, int page_bits) {
  return (int)((tokens + (1 << page_bits) - 1) >> page_bits);
}

// Room for counts[b] more tokens of every sequence (null: one each). Latency:
// a chain of loads and four barriers a scan: 2 us in a graph for 10 to 260 sequences,
// 3 for 2000.
__global__ void __launch_bounds__(kPlanThreads)
    extend_kernel(const cxs_pages_call c, const int* counts, int page_bits) {
  const Work w = work_of(c);
  cxs::after_earlier();
  cxs::next_may_come();
  const long long most = (long long)c.width << page_bits;
  int total = 0, bad = 0;
  for (int b0 = 0; b0 < c.sequences; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int need = 0;
    if (b < c.sequences) {
      const int length = c.lengths[b], more = counts ? counts[b] : 1;
      if (more < 0 || length < 0 || (long long)length + more > most) {
        bad |= CXS_DEVICE_ERR_BAD_LENGTH;
      } else if (more > 0) {
        need = pages_for((long long)length + more, page_bits) - pages_for(length, page_bits);
        if (length & ((1 << page_bits) - 1)) {  // the page that the tokens go on in
          const int page = c.table[(long long)b * c.width + (length >> page_bits)];
          if (page < 0 || page >= c.pages)
            bad |= CXS_DEVICE_ERR_BAD_BLOCK;
          else if (c.references[page] > 1)
            bad |= CXS_DEVICE_ERR_SHARED_PAGE;
        }
      }
    }
    int all;
    const int before = block_scan(need, &all);
    if (b < c.sequences) w.first[b] = total + before;
    total += all;
  }
  if (bad) report(c.error, bad);
  if (__syncthreads_or(bad)) return;
  if (!take_pages(c, total, w.target)) return;
  for (int r = threadIdx.x; r < total; r += kPlanThreads) {
    int l = 0, h = c.sequences - 1;  // the last sequence with first <= r
    while (l < h) {
      const int m = (l + h + 1) / 2;
      if (w.first[m] <= r) l = m; else h = m - 1;
    }
    const int page = w.target[r];
    c.table[(long long)l * c.width + pages_for(c.lengths[l], page_bits) + r - w.first[l]] = page;
    c.references[page] = 1;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < c.sequences; b += kPlanThreads) {
    const int more = counts ? counts[b] : 1;
    if (more > 0) c.lengths[b] += more;
  }
  if (threadIdx.x == 0 && total > 0) *c.lowest = w.target[total - 1] + 1;
}

// What forking does: a fresh page for each child whose parent ends inside a page.
// With the launch that copies, in a graph: 8 children of 16 layers (2 heads of 64
// channels) 9 us, 256 of 4 layers (8 of 128) 13, 2000 of one 19. (In one CTA because
// the lowest free ids, which every child's page depends on, are a scan over all.)
__global__ void __launch_bounds__(kPlanThreads)
    fork_kernel(const cxs_pages_call c, const int* parents, const int* children, int n,
                int page_bits) {
  const Work w = work_of(c);
  cxs::after_earlier();
  cxs::next_may_come();
  if (threadIdx.x == 0) w.copies[0] = w.copies[1] = 0;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int child = children[i];
    if (child >= 0 && child < c.sequences) w.claim[child] = 0;
  }
  __syncthreads();
  int total = 0, bad = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int parent = parents[i], child = children[i];
      int length = 0;
      if (parent < 0 || parent >= c.sequences || child < 0 || child >= c.sequences) {
        bad |= CXS_DEVICE_ERR_BAD_SEQUENCE;
      } else if (c.lengths[child] != 0 || atomicAdd(&w.claim[child], 1) > 0) {
        bad |= CXS_DEVICE_ERR_BAD_SEQUENCE;  // holds tokens, or is there twice
      } else {
        length = c.lengths[parent];
        if (length < 0 || length > (long long)c.width << page_bits) {
          bad |= CXS_DEVICE_ERR_BAD_LENGTH;
          length = 0;
        }
        need = (length & ((1 << page_bits) - 1)) != 0;
        if (need) {
          const int page = c.table[(long long)parent * c.width + (length >> page_bits)];
          if (page < 0 || page >= c.pages) bad |= CXS_DEVICE_ERR_BAD_BLOCK;
        }
      }
      w.size[i] = length;
    }
    int all;
    const int before = block_scan(need, &all);
    if (i < n) w.first[i] = total + before;
    total += all;
  }
  if (bad) report(c.error, bad);
  if (__syncthreads_or(bad)) return;
  if (!take_pages(c, total, w.target)) return;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int length = w.size[i], fill = length & ((1 << page_bits) - 1);
    if (fill) {
      const int k = w.first[i], page = w.target[k], at = length >> page_bits;
      w.source[k] = c.table[(long long)parents[i] * c.width + at];
      w.fill[k] = fill;
      c.table[(long long)children[i] * c.width + at] = page;
      c.references[page] = 1;
    }
    c.lengths[children[i]] = length;
  }
  if (threadIdx.x == 0) {
    if (total > 0) *c.lowest = w.target[total - 1] + 1;
    w.copies[0] = total;
    w.copies[1] = n;
  }
}

// The live pages past the first `live` ids go to the free ones among those. 16384
// references a round of each search; nothing to move: 5 us with the second launch.
__global__ void __launch_bounds__(kPlanThreads)
    compact_kernel(const cxs_pages_call c, int* live_out) {
  const Work w = work_of(c);
  cxs::after_earlier();
  cxs::next_may_come();
  const int live = find_pages(c.references, 0, c.pages, true, INT_MAX, [](int, int) {});
  const int moves = find_pages(c.references, 0, live, false, INT_MAX,
                               [&](int page, int rank) { w.target[rank] = page; });
  find_pages(c.references, live, c.pages, true, moves, [&](int page, int rank) {
    w.source[rank] = page;
    w.fill[rank] = c.page_size;
  });
  __syncthreads();
  for (int k = threadIdx.x; k < moves; k += kPlanThreads) {
    const int source = w.source[k], target = w.target[k];
    w.moved[source] = target;
    c.references[target] = c.references[source];
    c.references[source] = 0;
  }
  if (threadIdx.x == 0) {
    w.copies[0] = moves;
    w.copies[1] = live;
    *c.lowest = live;
    if (live_out) *live_out = live;
  }
}

// Page contents of all layers, a warp for each page's K or V of a head; then the
// rows: of the children (their parents' full pages), or all, with new ids. Bound by
// HBM: eight 16-byte loads a lane in flight, 570 MB of a pool in 88 us, 0.98 of the
// copy rate.
template <bool COMPACT>
__global__ void __launch_bounds__(kApplyThreads)
    apply_kernel(const cxs_pages_call c, const int* parents, const int* children, int page_bits) {
  const Work w = work_of(c);
  const int lane = threadIdx.x % 32;
  const int warp = (blockIdx.x * kApplyThreads + threadIdx.x) / 32;
  const int warps = gridDim.x * (kApplyThreads / 32);
  cxs::after_earlier();
  cxs::next_may_come();
  const int copies = w.copies[0], count = w.copies[1];
  const int parts = 2 * c.kv_heads;
  const long long part_bytes = (long long)c.page_size * c.dim;
  for (long long run = warp; run < (long long)copies * parts * c.layers; run += warps) {
    const long long page = run / parts;
    const int part = (int)(run - page * parts);
    const int layer = (int)(page / copies), k = (int)(page - (long long)layer * copies);
    const long long from = (long long)w.source[k] * parts + part;
    const long long to = (long long)w.target[k] * parts + part;
    uint8_t* const codes = (uint8_t*)c.layer_buffers[2 * layer];
    float* const scales = (float*)c.layer_buffers[2 * layer + 1];
    const uint4* const in = (const uint4*)(codes + from * part_bytes);
    uint4* const out = (uint4*)(codes + to * part_bytes);
    const int vectors = w.fill[k] * c.dim / 16;
    constexpr int kAtOnce = 8;
    for (int v0 = lane; v0 < vectors; v0 += 32 * kAtOnce) {
      uint4 x[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (v0 + 32 * j < vectors) x[j] = in[v0 + 32 * j];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (v0 + 32 * j < vectors) out[v0 + 32 * j] = x[j];
    }
    if (lane == 0) scales[to] = scales[from];
  }
  if (COMPACT) {
    const long long entries = (long long)c.sequences * c.width;
    for (long long i = (long long)warp * 32 + lane; i < entries; i += (long long)warps * 32) {
      const int page = c.table[i];
      if (page >= count && page < c.pages) c.table[i] = w.moved[page];
    }
  } else {
    const int chunks = (c.width + kRowChunk - 1) / kRowChunk;
    for (long long unit = warp; unit < (long long)count * chunks; unit += warps) {
      const int i = (int)(unit / chunks), j0 = (int)(unit - (long long)i * chunks) * kRowChunk;
      const int full = w.size[i] >> page_bits;
      if (j0 >= full) continue;
      const int* const in = c.table + (long long)parents[i] * c.width;
      int* const out = c.table + (long long)children[i] * c.width;
      for (int j = j0 + lane; j < min(full, j0 + kRowChunk); j += 32) {
        const int page = in[j];
        out[j] = page;
        if (page >= 0 && page < c.pages) atomicAdd(c.references + page, 1);
      }
    }
  }
}

// Each entry is taken out once, so a sequence that is there twice is freed once.
__global__ void __launch_bounds__(kApplyThreads)
    free_kernel(const cxs_pages_call c, const int* sequences, int n) {
  cxs::after_earlier();
  cxs::next_may_come();
  const int chunks = (c.width + kApplyThreads - 1) / kApplyThreads;
  for (long long unit = blockIdx.x; unit < (long long)n * chunks; unit += gridDim.x) {
    const int i = (int)(unit / chunks), chunk = (int)(unit - (long long)i * chunks);
    const int b = sequences[i], j = chunk * kApplyThreads + threadIdx.x;
    if (b < 0 || b >= c.sequences) {
      if (j == 0) report(c.error, CXS_DEVICE_ERR_BAD_SEQUENCE);
      continue;
    }
    if (j == 0) c.lengths[b] = 0;
    if (j >= c.width) continue;
    const int page = atomicExch(c.table + (long long)b * c.width + j, -1);
    if (page >= 0 && page < c.pages && atomicSub(c.references + page, 1) == 1)
      atomicMin(c.lowest, page);
  }
}

// The table and lengths that a program held, references counted anew (they are
// 0 before). Entries past a sequence's length are not looked at.
__global__ void __launch_bounds__(kApplyThreads)
    adopt_kernel(const cxs_pages_call c, const int* table, long long stride, int width,
                 const int* lengths, int page_bits) {
  const int chunks = (c.width + kApplyThreads - 1) / kApplyThreads;
  for (long long unit = blockIdx.x; unit < (long long)c.sequences * chunks; unit += gridDim.x) {
    const int b = (int)(unit / chunks), j = (int)(unit - (long long)b * chunks) * kApplyThreads + threadIdx.x;
    int length = lengths[b];
    if (length < 0 || length > (long long)width << page_bits) {
      if (j == 0) report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
      length = 0;
    }
    if (j == 0) c.lengths[b] = length;
    if (j >= c.width) continue;
    int page = j < pages_for(length, page_bits) ? table[b * stride + j] : -1;
    if (j < pages_for(length, page_bits) && (page < 0 || page >= c.pages)) {
      report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
      page = -1;
    }
    c.table[(long long)b * c.width + j] = page;
    if (page >= 0) atomicAdd(c.references + page, 1);
  }
}

// ------------------------------------------------------------------ host ---

int check_pages(const cxs_pages_call* c, const char* what) {
  if (!c) return set_error(CXS_ERR_INVALID, "%s: null call", what);
  if (c->pages < 1 || c->layers < 1 || c->sequences < 1 || c->width < 1 || c->kv_heads < 1)
    return set_error(CXS_ERR_INVALID, "%s: pages, layers, sequences, width and kv_heads must be positive", what);
  if (c->dim != 64 && c->dim != 128) return set_error(CXS_ERR_INVALID, "%s: dim must be 64 or 128", what);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64)
    return set_error(CXS_ERR_INVALID, "%s: page_size must be 16, 32 or 64", what);
  if ((long long)c->width * c->page_size > cxs_host::kMaxPositions)
    return set_error(CXS_ERR_CAPACITY, "%s: more than 2^30 positions in a row", what);
  if ((long long)c->width * c->sequences > 0x7fffffffll)
    return set_error(CXS_ERR_CAPACITY, "%s: a table of 2^31 or more entries", what);
  if (c->pages > 0x40000000 || c->kv_heads > 32767 || c->layers > 65535)
    return set_error(CXS_ERR_CAPACITY, "%s: too many pages, heads or layers", what);
  return CXS_OK;
}

int check_pointers(const cxs_pages_call* c, const char* what) {
  if (!c->layer_buffers || !c->table || !c->lengths || !c->references || !c->lowest)
    return set_error(CXS_ERR_INVALID, "%s: null buffers, table, lengths, references or lowest", what);
  if (!c->workspace || (uintptr_t)c->workspace % 4 ||
      c->workspace_bytes < work_ints(*c) * (long long)sizeof(int))
    return set_error(CXS_ERR_INVALID, "%s: workspace missing, unaligned or too small", what);
  return CXS_OK;
}

int page_bits_of(const cxs_pages_call& c) { return c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : 6; }

constexpr int kMostBlocks = 148 * 8;  // CTAs of 256 threads that an SM of a B200 holds, all SMs

int blocks_for(long long units) {
  return (int)(units < 1 ? 1 : units < kMostBlocks ? units : kMostBlocks);
}

// `work`: warps that have something to do, at most.
template <bool COMPACT>
int launch_apply(const cxs_pages_call& c, const int* parents, const int* children, long long work,
                 cudaStream_t stream) {
  const int blocks = blocks_for((work + kApplyThreads / 32 - 1) / (kApplyThreads / 32));
  return cxs_host::launch_early("pages apply", apply_kernel<COMPACT>, blocks, kApplyThreads, 0, 0,
                                stream, c, parents, children, page_bits_of(c));
}

}  // namespace

extern "C" int cxs_pages_workspace(const cxs_pages_call* call, int64_t* bytes) {
  const int status = check_pages(call, "pages");
  if (status != CXS_OK) return status;
  if (!bytes) return set_error(CXS_ERR_INVALID, "pages: null result");
  *bytes = work_ints(*call) * (int64_t)sizeof(int);
  return CXS_OK;
}

extern "C" int cxs_pages_extend(const cxs_pages_call* call, const int32_t* counts, void* stream) {
  int status = check_pages(call, "pages extend");
  if (status == CXS_OK) status = check_pointers(call, "pages extend");
  if (status != CXS_OK) return status;
  return cxs_host::launch_early("pages extend", extend_kernel, 1, kPlanThreads, 0, 0,
                                (cudaStream_t)stream, *call, counts, page_bits_of(*call));
}

extern "C" int cxs_pages_fork(const cxs_pages_call* call, const int32_t* parents,
                              const int32_t* children, int32_t count, void* stream) {
  int status = check_pages(call, "pages fork");
  if (status != CXS_OK) return status;
  if (count < 0 || count > call->sequences)
    return set_error(CXS_ERR_INVALID, "pages fork: count must be 0 .. sequences");
  if (count == 0) return CXS_OK;
  status = check_pointers(call, "pages fork");
  if (status != CXS_OK) return status;
  if (!parents || !children) return set_error(CXS_ERR_INVALID, "pages fork: null parents or children");
  status = cxs_host::launch_early("pages fork", fork_kernel, 1, kPlanThreads, 0, 0,
                                  (cudaStream_t)stream, *call, parents, children, count,
                                  page_bits_of(*call));
  if (status != CXS_OK) return status;
  const long long chunks = (call->width + kRowChunk - 1) / kRowChunk;
  const long long runs = (long long)count * call->layers * call->kv_heads * 2;
  return launch_apply<false>(*call, parents, children, runs > count * chunks ? runs : count * chunks,
                             (cudaStream_t)stream);
}

extern "C" int cxs_pages_free(const cxs_pages_call* call, const int32_t* sequences, int32_t count,
                              void* stream) {
  int status = check_pages(call, "pages free");
  if (status != CXS_OK) return status;
  if (count < 0) return set_error(CXS_ERR_INVALID, "pages free: negative count");
  if (count == 0) return CXS_OK;
  status = check_pointers(call, "pages free");
  if (status != CXS_OK) return status;
  if (!sequences) return set_error(CXS_ERR_INVALID, "pages free: null sequences");
  const long long chunks = (call->width + kApplyThreads - 1) / kApplyThreads;
  return cxs_host::launch_early("pages free", free_kernel, blocks_for(count * chunks), kApplyThreads,
                                0, 0, (cudaStream_t)stream, *call, sequences, count);
}

extern "C" int cxs_pages_adopt(const cxs_pages_call* call, const int32_t* table,
                               int64_t table_stride, int32_t width, const int32_t* lengths,
                               void* stream) {
  int status = check_pages(call, "pages adopt");
  if (status == CXS_OK) status = check_pointers(call, "pages adopt");
  if (status != CXS_OK) return status;
  if (!table || !lengths) return set_error(CXS_ERR_INVALID, "pages adopt: null table or lengths");
  if (width < 1 || width > call->width || table_stride < width)
    return set_error(CXS_ERR_INVALID, "pages adopt: width must be 1 .. the table's, table_stride at least width");
  cudaStream_t s = (cudaStream_t)stream;
  const bool next = call->lowest == call->references + call->pages;  // one run of bytes
  CXS_CUDA(cudaMemsetAsync(call->references, 0, ((size_t)call->pages + next) * sizeof(int32_t), s));
  if (!next) CXS_CUDA(cudaMemsetAsync(call->lowest, 0, sizeof(int32_t), s));
  const long long chunks = (call->width + kApplyThreads - 1) / kApplyThreads;
  adopt_kernel<<<blocks_for(call->sequences * chunks), kApplyThreads, 0, s>>>(
      *call, table, table_stride, width, lengths, page_bits_of(*call));
  CXS_LAUNCH_CHECK("pages adopt");
  return CXS_OK;
}

extern "C" int cxs_pages_compact(const cxs_pages_call* call, int32_t* live, void* stream) {
  int status = check_pages(call, "pages compact");
  if (status == CXS_OK) status = check_pointers(call, "pages compact");
  if (status != CXS_OK) return status;
  status = cxs_host::launch_early("pages compact", compact_kernel, 1, kPlanThreads, 0, 0,
                                  (cudaStream_t)stream, *call, live);
  if (status != CXS_OK) return status;
  return launch_apply<true>(*call, nullptr, nullptr, 1ll << 30, (cudaStream_t)stream);
}
