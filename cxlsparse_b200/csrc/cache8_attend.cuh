// Attention over the dense 8-bit cache: what its kernels share.
//
// Mathematics. With codes c and scales s_k, s_v constant over a page, a score
// in base-2 units is x = scale log2(e) s_k (q . c_k), and
//   out = sum 2^x s_v c_v / sum 2^x = sum p c_v / sum p / s_v,
//   p = 2^(x + log2 s_v - M + 13),  M = running max of x + log2 s_v, moved when
//   a score passes it by 2: p <= 2^15.
// p is rounded to fp16 and multiplied with the codes themselves, which fp16
// holds exactly (e4m3 and integers to 128); the denominator divides each page's
// sum of p by its s_v in fp32. fp16 keeps 11 bits down to 2^-14: of every key
// whose 2^x s_v is within 2^-27 of the row's largest, and of smaller ones what
// is left above 2^-38 of it. The top of fp16's range is used because keys far
// below the largest are not always negligible: its V may be 0 (a first token
// that takes 0.999 of the softmax before 64K others, each 2^-26 of it; a page
// whose scale a hidden outlier has set). With M at the largest p itself such
// rows were off by a half. 2^ and log2 are
// the approximate instructions (2^-22 of the result, 2 units of the last place):
// far below the rounding of p. Queries are scaled by a power of two per row so
// that fp16 holds them: exact for fp16 inputs, and for bf16 (8 bits of
// mantissa) but for parts 2^-28 below the row's largest element, which lose
// less than 2^-39 of it.
#pragma once

#include <limits.h>

#include "cache8.cuh"

namespace cxs {
namespace cache8 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = INFINITY;
// M moves when a score passes it by kLag, and a score of M weighs 2^kHead:
// most tiles leave O as it is, and fp16 has the room above and below. Measured
// for lags of 8 / 4 / 2 / 1 (weights to 2^15 in each): prefill chunk 603 / 606 /
// 609 / 611 us, suffixes and decode steps the same; beside a dominant key of
// V = 0 over 64K tokens the error of out is 2e-2, 2.3e-3, below 1e-3, below 1e-3.
constexpr float kLag = 2.f, kHead = 13.f;
constexpr long long kSpinLimit = 1ll << 32;  // clock cycles before a wait gives up

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------ code conversion ---

// Two codes (the low or high half of `w`) as fp16, exact.
template <int FORMAT>
__device__ __forceinline__ uint32_t half2_of(uint32_t w, int high);
template <>
__device__ __forceinline__ uint32_t half2_of<CXS_FORMAT_E4M3>(uint32_t w, int high) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
      : "=r"(r)
      : "h"((unsigned short)(high ? w >> 16 : w & 0xffffu)));
  return r;
}
// An integer v as 1024 + 128 + v (its bits in an fp16 mantissa), minus 1152.
template <>
__device__ __forceinline__ uint32_t half2_of<CXS_FORMAT_INT8>(uint32_t w, int high) {
  const uint32_t biased = __byte_perm(w ^ 0x80808080u, 0x64646464u, high ? 0x4342 : 0x4140);
  __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// ----------------------------------------------------------------- items ---
//
// An item is one user's tile of query rows (a row is a new token and one of
// the KV head's query heads: row r is token r / group, head r % group) with
// one KV head. Its work is a run of key tiles. All items' tiles, in order,
// are cut into equal shares, one for each worker (a warp of the kernel for few
// rows, a CTA of the other), whatever the users' lengths; an item whose tiles
// fall into several shares leaves a partial result (O, M, l) in each. They are
// joined in the order of the keys: those of a CTA's warps at its end, those of
// CTAs by combine_kernel.

constexpr int kSlice = 2048;  // users of one launch (their tile counts sit in shared memory)

struct Shape {
  int group;      // query heads of a KV head
  int user0;      // first user of this launch (table, lengths and offsets point at it)
  int users;
  int last;       // the launch holds the last user
  int grid;       // CTAs
  int workers;    // most shares: warps or CTAs of the grid
  int min_tiles;  // fewest tiles worth a share,
  int few_tiles;  // but of no more tiles in all than this, each is one
};

// One user's positions. Visible to some row: [begin, end).
struct Span {
  int first, count;     // packed rows
  int start;            // position of the first row (negative: more rows than tokens)
  int length;           // tokens, cut to the table
  int begin;
};

__device__ __forceinline__ Span user_span(const cxs_cache_attend_call& a, const Shape& z, int user,
                                          int* bad) {
  const cxs_cache_call& c = a.cache;
  Span s;
  Rows rows;
  if (c.offsets) {
    rows = user_rows(c, user, bad);
  } else {
    rows = {z.user0 + user, 1};
  }
  const int most = c.width * c.page_size;
  s.first = rows.first;
  s.count = rows.count;
  s.length = c.lengths[user];
  if (s.length < 0) s.length = 0, *bad = 1;
  s.start = s.length - rows.count;
  if (s.length > most) s.length = most, *bad = 1;
  s.begin = a.window > 0 && s.start >= a.window ? min(s.start - a.window + 1, s.length) : 0;
  return s;
}

// Row r of a user sees positions [x, y).
__device__ __forceinline__ int2 row_range(const cxs_cache_attend_call& a, const Span& s,
                                          int token) {
  const int position = s.start + token;
  int hi = s.length, lo = 0;
  if (a.causal && position + 1 < hi) hi = position + 1;
  if (a.window > 0 && position >= a.window) lo = position - a.window + 1;
  return make_int2(lo, hi);
}

// a / b of a >= 0, b > 0: in 32 bits, where a fits, at a fifth of the cost.
__device__ __forceinline__ long long divide(long long a, int b) {
  if (a >> 32 == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// The tiles cut into `count` shares: of `each` tiles, the first `more` of them
// of one more.
struct Shares {
  int count;
  long long each;
  int more;
  __device__ __forceinline__ Shares(long long total, const Shape& z) {
    const long long wanted =
        total <= z.few_tiles ? total : divide(total + z.min_tiles - 1, z.min_tiles);
    count = wanted < z.workers ? (int)wanted : z.workers;
    each = count > 0 ? divide(total, count) : 0;
    more = (int)(total - each * count);
  }
  __device__ __forceinline__ long long begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int of(long long tile) const {  // the share that has it
    const long long wide = (each + 1) * more;
    if (tile < wide || each == 0) return (int)(each + 1 > INT_MAX ? tile / (each + 1) : divide(tile, (int)each + 1));
    return more + (int)(each > INT_MAX ? (tile - wide) / each : divide(tile - wide, (int)each));
  }
};

struct alignas(16) Partial {  // the item that starts in a share and goes on past it
  int parts;      // shares it falls into; 0: none
  int first, rows, row0, kv_head;  // the item's packed first row, user's rows, first row, head
};

// Rows of no user (see row_gap): zero, and nothing in the sum. Shared out among the
// workers, each of `threads` threads.
template <typename T, int D>
__device__ void clear_rows(const cxs_cache_attend_call& a, const Shape& z, int worker, int workers,
                           int thread, int threads) {
  const cxs_cache_call& c = a.cache;
  if (!c.offsets) return;
  for (int b = worker - 1; b <= z.users; b += workers) {
    if ((b < 0 && z.user0 > 0) || (b == z.users && !z.last)) continue;  // (another launch's)
    const Gap gap = row_gap(c, b, z.users);
    for (long long i = gap.low * a.heads * D + thread; i < gap.high * a.heads * D; i += threads)
      ((T*)a.out)[i] = from_float<T>(0.f);
    if (a.lse)
      for (long long i = gap.low * a.heads + thread; i < gap.high * a.heads; i += threads)
        a.lse[i] = -kInf;
  }
}

// A probability of 0 times a NaN would be NaN, so V of a tile with keys that
// some row does not see has its NaN codes (e4m3 only) replaced by 0 before the
// product. The rows that do see such a key get their NaN once the item's result
// is written, from the codes themselves: few tiles can have any, and hardly one
// does, so this stays out of the loops (in them it cost 4 %).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {  // 0x80 in each NaN byte's place
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t w, uint32_t* found) {
  const uint32_t n = nan_codes(w);
  *found |= n;
  return w & ~(n | (n - (n >> 7)));
}
__device__ __forceinline__ uint4 without_nan(uint4 w, uint32_t* found) {
  return make_uint4(without_nan(w.x, found), without_nan(w.y, found), without_nan(w.z, found),
                    without_nan(w.w, found));
}
// The keys [lo, hi) that all rows of an item see; tiles beyond are hidden in part.
__device__ __forceinline__ int2 seen_by_all(const cxs_cache_attend_call& a, const Shape& z,
                                            const Span& s, int row0, int row1) {
  return make_int2(row_range(a, s, row1 / z.group).x, row_range(a, s, row0 / z.group).y);
}
// Makes NaN the channels d .. d + count - 1 of a row's result (out, or its part
// where that is not null) in which V of some key of [lo, hi), but for the keys
// [skip.x, skip.y), is NaN. `codes` are the KV head's V of page 0, pages
// page_bytes apart, `table` the user's.
template <typename T, int D>
__device__ __noinline__ void mark_nans(const uint8_t* codes, long long page_bytes, int pages,
                                       const int* table, int page_size, int lo, int hi, int2 skip,
                                       T* out, float* part, int d, int count) {
  for (int w = d; w < d + count; w += 4) {
    uint32_t nans = 0;
    for (int t = lo; t < hi; ++t) {
      if (t >= skip.x && t < skip.y) {
        t = skip.y - 1;
        continue;
      }
      const int page = table[t / page_size];
      if (page < 0 || page >= pages) continue;
      nans |= nan_codes(*reinterpret_cast<const uint32_t*>(codes + page * page_bytes +
                                                           t % page_size * D + w));
    }
    for (int e = 0; e < 4; ++e) {
      if (!(nans >> (8 * e + 7) & 1)) continue;
      if (part)
        part[w + e] = __uint_as_float(0x7fffffffu);
      else
        out[w + e] = from_float<T>(__uint_as_float(0x7fffffffu));
    }
  }
}

constexpr int kTileRows = 256;  // query rows of an item of the tile kernel

// What attention over shared tokens works out beforehand (cache8_shared.cu).
struct GroupPlan {
  int first, count;   // packed rows
  int shared;         // common tokens that all rows see
  int user0;          // whose pages they are in
};
struct ItemPlan {     // kTileRows query rows of a group, for every KV head
  long long before;   // cost of the items before it
  int group, tile_row;
  int tiles, common_tiles;
  int user_a, user_b; // its rows' users
  GroupPlan of;
};
struct SharePlan {    // a CTA's tiles and the item they begin in (all in one place: a CTA
  long long low, high;    // begins with reading it)
  long long total;    // cost of all items
  int id, kv_head;
  int solo;           // no group has more than half of kTileRows rows
  ItemPlan item;
};
struct PlanHead {
  int gaps;
};
struct SharedPlan {
  PlanHead* head;
  GroupPlan* groups;
  ItemPlan* items;
  SharePlan* shares;
  long long* runs;    // [users + groups]: runs of 16 own keys of the group's users
                      // before user u of group g at [u + g], of all of them after the last
  Gap* gaps;          // packed rows of no group
};

// One launch of the tile kernel over z.users users (cache8_tile.cu).
int launch_tile(const cxs_cache_attend_call& a, const Shape& z, cudaStream_t stream);
// The launch that joins what was left in parts (cache8_attend.cu).
// `spread`: items fall into many parts, read by several groups of threads.
int launch_join(const cxs_cache_attend_call& a, const Shape& z, bool few, bool spread,
                cudaStream_t stream);
int check_attend(const cxs_cache_attend_call* a, const char* what);
int check_attend_pointers(const cxs_cache_attend_call* a, long long workspace, const char* what);
int sm_count(int* sms);
bool few_rows(const cxs_cache_attend_call& a);
// Bytes that the kernels of few or many rows leave their partial results in.
long long partial_bytes(const cxs_cache_attend_call& a, bool few);
constexpr int kMostCtas = 148;  // largest grid of a call: one CTA per SM of a B200. (A
                                // constant: the workspace does not depend on the device.)

}  // namespace cache8
}  // namespace cxs
