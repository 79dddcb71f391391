// Attention over the dense 8-bit cache: many query rows a KV head (suffixes,
// prefills), on tcgen05 with TMEM accumulators.
//
// An item is 256 query rows (two groups of 128) of one user and KV head; its
// keys come in tiles of 128. One CTA per SM, 16 warps:
//   warps 0-3, 4-7  softmax of group 0 and 1, one row a thread: reads S from
//                   TMEM, writes p as fp16 (for D = 128 over S), rescales O when
//                   M moves
//   warps 8-11      conversion of K and V codes to fp16 operand tiles in shared
//                   memory, which both groups use
//   warp 12         one thread issues every MMA: S = Q K^T (Q, K in shared
//                   memory), O += P V (P in TMEM, V in shared memory)
//   warp 13         loads: bulk copies of the tiles' pages into shared memory,
//                   their scales, and what the others need to know of a tile
// While one group's softmax runs, the tensor core works for the other. For D =
// 64 P has columns of its own, and S of the next tile is computed as soon as
// this one's has been read. For D = 128 it has not: the MMAs of one thread
// complete in order, so S of the next tile may be issued over P right after
// the P V that reads it, and a commit after S also tells that the group's
// previous P V is done (O may be rescaled).
// Waits are bounded: a wait that runs out sets the error word and an abort
// flag that ends every role.
// Measured: 256 tokens of 32 query and 2 KV heads of 64 over 16K keys (e4m3) in
// 79 us, 438 TFLOP/s; 3 users' prefill chunks, 32 / 8 heads of 128 (int8), in
// 595 us, 796 TFLOP/s of the 1650 that cuBLAS reaches in bf16. No unit is full
// (special functions 41 and 38 % of the time, tensor core 20 and 38 %): a row's
// softmax is a chain (read S, maximum, exponentials) that two warps a scheduler
// do not cover, S and P V wait for it at 128 channels, where TMEM holds only one
// S of each group, and registers are short (188 to 396 bytes spilled a thread).
//
// SHARED: the item's rows are those of several users that have their first tokens
// in common. Its tiles are first those of the common tokens, from the first
// user's pages, then tiles made up of runs of 16 of each user's own keys, of
// which a row sees its own user's only. What the users' sizes come to is worked
// out by a launch before (cache8_shared.cu).
#pragma once

#include "cache8_attend.cuh"
#include "tile_tc.cuh"

namespace {

using namespace cxs::cache8;
namespace tc = cxs::tc;

constexpr int kKeys = 128;              // of a tile
constexpr int kThreads = 16 * 32;  // the last two warps only share the setup
constexpr int kConvertWarp = 8, kMmaWarp = 12, kLoadWarp = 13;
constexpr int kPanel = 128 * 128;       // bytes: 128 rows (queries or keys) of 64 channels, swizzled
constexpr int kRuns = kKeys / 16;       // runs of 16 keys: each within one page
constexpr int kRing = 8;                // tiles whose Tile is kept: more than are ever in work
// Tiles that an item's queries and results cost (measured: about 20,000 cycles
// an item, 5,000 to 6,000 a tile; shares of tiles alone ended 30 % apart).
constexpr int kItemCost = 4;
constexpr int kTmem = 512;              // columns: all; see Layout

// Registers a thread by role: twice the softmax's, the conversion's and the
// rest's, times 128, are the 64 K that 512 threads of 128 are launched with.
constexpr int kSoftmaxRegs = 184, kConvertRegs = 80, kOtherRegs = 64;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kOtherRegs == 4 * 128, "the block's registers");
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// First and last of its item here; rows for group 1; keys that some row does not see.
constexpr int kFirst = 1, kLast = 2, kTwo = 4, kHidden = 8;
constexpr unsigned kWild = 1u << kRuns;  // a scale of the tile is infinite or NaN

struct Tile {                // what the roles need of a tile of keys
  float4 runs[kRuns];        // of 16 keys: |scale| log2(e) s_k, log2 s_v, 1 / s_v, and (SHARED)
                             // how many of a user's own keys hold tokens
  unsigned missing;          // bit u: run u has no page, no row sees it; (SHARED) kWild
  int left;                  // keys of the tile that hold tokens (may be negative or above kKeys)
  int flags;
  int unused;
};

// Shared memory. K has one operand stage where two do not fit (D = 128): the
// next K is converted while the softmax of this tile runs.
template <int D>
struct Layout {
  static constexpr int kPanels = D / 64;
  // TMEM columns: S of two groups, P (over S where nothing else is left), O.
  static constexpr bool kApart = D == 64;  // P has its own columns
  static constexpr int kP = kApart ? 256 : 0, kPStep = kApart ? 64 : 128;
  static constexpr int kO = kApart ? 384 : 256;
  static constexpr int kKStages = D == 64 ? 2 : 1, kVStages = 2, kRawStages = D == 64 ? 2 : 1;
  static constexpr int kRawPart = kKeys * D;                     // bytes of K or V codes
  static constexpr int kQ = 0;                                   // [2 groups][panels]
  static constexpr int kK = kQ + 2 * kPanels * kPanel;           // [stages][panels]
  static constexpr int kV = kK + kKStages * kPanels * kPanel;    // [stages][panels]
  static constexpr int kRaw = kV + kVStages * kPanels * kPanel;  // [stages][K, V]
  static constexpr int kTiles = kRaw + kRawStages * 2 * kRawPart;  // [kRing]
  static constexpr int kBars = kTiles + kRing * (int)sizeof(Tile);
  static constexpr int kPrefix = kBars + 320;
  static constexpr int kCounts = kPrefix + (kSlice + 1) * 8;
  static constexpr int kBytes = kCounts + (kSlice + 1) * 4 + 1024;  // and the 1024-byte alignment
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

struct Bars {
  uint64_t raw_full[2][2], raw_free[2][2];          // by raw stage and part
  uint64_t k_full[2], v_full[2], k_free[2], v_free[2];  // by operand stage
  uint64_t s_full[2], s_free[2], p_full[2], q_full[2], o_done[2], o_free[2];  // by group
  uint64_t turn[2][4];  // (SHARED) of a group's warps to take their exponentials
  uint64_t drain[2];
  int abort;
  int nans;  // V had NaN codes where keys are hidden
  uint32_t tmem;
};
static_assert(sizeof(Bars) <= 320, "barrier block");

// Stage of use n of a ring of N and the parity of its n-th phase.
template <int N>
__device__ __forceinline__ int stage_of(int n) { return N == 1 ? 0 : n & 1; }
template <int N>
__device__ __forceinline__ int phase_of(int n) { return N == 1 ? n : n >> 1; }

// Whether a barrier's phase has completed, without waiting.
__device__ __forceinline__ bool test_wait(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(cxs::smem_addr(bar)), "r"(phase)
      : "memory");
  return ok != 0;
}

// Bounded wait on a barrier phase; false: some role of the CTA gave up.
__device__ __forceinline__ bool wait(uint64_t* bar, int phase, Bars* b, int* error) {
  if (cxs::mbar_try_wait(bar, phase & 1)) return true;
  const long long start = clock64();
  while (!cxs::mbar_try_wait(bar, phase & 1)) {
    if (*(volatile int*)&b->abort) return false;
    if (clock64() - start > kSpinLimit) {
      report(error, CXS_DEVICE_ERR_COPY_TIMEOUT);
      *(volatile int*)&b->abort = 1;
      return false;
    }
  }
  return true;
}

// The same for a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, int phase, Bars* b, int* error) {
  return __all_sync(0xffffffffu, wait(bar, phase, b, error));
}

// Arrive for a warp whose lanes have all written what the barrier guards.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) cxs::mbar_arrive(bar);
}

// kind::f16 with fp16 operands and fp32 accumulation.
__device__ __forceinline__ uint32_t idesc_f16(int m, int n, int b_mn_major) {
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// D (+)= A B; A in shared memory, or (mma_ts) in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((int)accumulate));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((int)accumulate));
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one;
}

// 64 fp32 columns of this warp's 32 lanes (the wait is part of the statement:
// nothing can use, move or spill the registers before they are written).
__device__ __forceinline__ void ld64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,"
      "%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]),
        "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]),
        "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}

// 32 of them.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;"
      : "=f"(d)
      : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

// (No memory clobber: loads of what a tile's next columns need move ahead.)
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}

// An item and where its tiles lie among all tiles of the launch.
struct Item {
  int user, tile_row, kv_head;   // rows kTileRows * tile_row .. (SHARED: of the group; the
                                 // common tokens are in that user's pages)
  long long begin, end;
  long long index;               // among all items
  Span span;
  int rows;                      // of the user with this KV head
  int first;                     // its first tile of keys
  int id, group, common_tiles;   // SHARED: its plan, its group and the common keys' tiles;
  int user_a, user_b;            // users that its rows belong to
};

// Tiles of keys that some row of a row tile sees; at least one, so that rows
// that see nothing are written.
__device__ __forceinline__ int key_tiles(const cxs_cache_attend_call& a, const Shape& z,
                                         const Span& s, int rows, int tile_row, int* first) {
  const int row0 = tile_row * kTileRows, row1 = min(rows, row0 + kTileRows) - 1;
  const int lo = row_range(a, s, row0 / z.group).x, hi = row_range(a, s, row1 / z.group).y;
  *first = lo / kKeys;
  const int n = (hi + kKeys - 1) / kKeys - *first;
  return hi > 0 && n > 0 ? n : 1;
}

// --------------------------------------------------------------- SHARED ---

// The item of plan `id` and KV head, its tiles and its group's span: `length`
// common tokens, the packed rows of the group.
__device__ __forceinline__ void plan_item(const ItemPlan& item, const Shape& z, int id,
                                          int kv_head, int kv_heads, Item& p) {
  p.id = id;
  p.group = item.group;
  p.tile_row = item.tile_row;
  p.kv_head = kv_head;
  p.index = (long long)id * kv_heads + kv_head;
  p.begin = item.before + (long long)kv_head * (item.tiles + kItemCost) - kItemCost * p.index;
  p.end = p.begin + item.tiles;
  p.common_tiles = item.common_tiles;
  p.user_a = item.user_a;
  p.user_b = item.user_b;
  p.user = item.of.user0;
  p.rows = item.of.count * z.group;
  p.first = 0;
  p.span = Span{item.of.first, item.of.count, 0, item.of.shared, 0};
}

// The last of users [lo, hi] whose packed rows begin at or before `row`. (No
// offsets: each has one.)
__device__ __forceinline__ int user_of(const int* offsets, int row, int lo, int hi) {
  if (!offsets) return row;
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if (offsets[m] <= row) lo = m; else hi = m - 1;
  }
  return lo;
}

// A row's user and the end of the keys it sees; returns where the user's runs
// begin, in keys, among the own keys of the item.
__device__ __forceinline__ int own_range(const cxs_cache_attend_call& a, const SharedPlan& plan,
                                         const Shape& z, const Item& p, int row, int* user,
                                         int* end) {
  const cxs_cache_call& c = a.cache;
  const int packed = p.span.first + row / z.group;
  const int u = user_of(c.offsets, packed, p.user_a, p.user_b);
  const int next = c.offsets ? __ldg(c.offsets + u + 1) : packed + 1;  // row past the user's
  const int most = c.width * c.page_size, length = max(__ldg(c.lengths + u), 0);
  int hi = min(length, most);
  if (a.causal) hi = min(hi, length - (next - packed) + 1);
  *user = u;
  *end = max(hi, p.span.length);
  const long long* const runs = plan.runs + p.group;
  return (int)(runs[u] - runs[p.user_a]) * 16;
}

// The page of the item's own run `n` (for lanes of the first kRuns), where in it
// the run begins and how many of its keys hold tokens; -2: there is none.
__device__ __forceinline__ int own_run(const cxs_cache_attend_call& a, const SharedPlan& plan,
                                       const Item& p, long long n, int lane, int* slot, int* held) {
  const cxs_cache_call& c = a.cache;
  const long long* const runs = plan.runs + p.group;
  *held = *slot = 0;
  const long long at = runs[p.user_a] + n;
  if (lane >= kRuns || at >= runs[p.user_b + 1]) return -2;
  int lo = p.user_a, hi = p.user_b;  // the last user whose runs begin at or before `at`
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if (runs[m] <= at) lo = m; else hi = m - 1;
  }
  const int key = p.span.length / 16 * 16 + (int)(at - runs[lo]) * 16;
  const int length = min(max(__ldg(c.lengths + lo), 0), c.width * c.page_size);
  *held = min(length - key, 16);
  *slot = key % c.page_size;
  return __ldg(c.table + lo * c.table_stride + key / c.page_size);
}

// Rows of no user, or of a group that has none: zero, and nothing in the sum.
template <typename T, int D>
__device__ void clear_shared(const cxs_cache_attend_call& a, const SharedPlan& plan) {
  for (int n = blockIdx.x; n < plan.head->gaps; n += gridDim.x) {
    const Gap gap = plan.gaps[n];
    for (long long i = gap.low * a.heads * D + threadIdx.x; i < gap.high * a.heads * D; i += kThreads)
      ((T*)a.out)[i] = from_float<T>(0.f);
    if (a.lse)
      for (long long i = gap.low * a.heads + threadIdx.x; i < gap.high * a.heads; i += kThreads)
        a.lse[i] = -kInf;
  }
}

template <int FORMAT, typename T, int D, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const cxs_cache_attend_call a, const Shape z, const SharedPlan plan) {
  using L = Layout<D>;
  const cxs_cache_call& c = a.cache;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem =
      (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Bars* const bars = (Bars*)(smem + L::kBars);
  Tile* const ring = (Tile*)(smem + L::kTiles);
  long long* const prefix = (long long*)(smem + L::kPrefix);
  int* const counts = (int*)(smem + L::kCounts);
  // (Broadcast: uniform across the warp also for the compiler.)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int part = 0; part < 2; ++part) {
        cxs::mbar_init(&bars->raw_full[i][part], 1);
        cxs::mbar_init(&bars->raw_free[i][part], 4);
      }
      cxs::mbar_init(&bars->k_full[i], 4);
      cxs::mbar_init(&bars->v_full[i], 4);
      cxs::mbar_init(&bars->k_free[i], SHARED ? 2 : 1);  // (by the last group, or each)
      cxs::mbar_init(&bars->v_free[i], SHARED ? 2 : 1);
      cxs::mbar_init(&bars->s_full[i], 1);
      cxs::mbar_init(&bars->s_free[i], 4);
      cxs::mbar_init(&bars->p_full[i], 4);
      cxs::mbar_init(&bars->q_full[i], 4);
      cxs::mbar_init(&bars->o_done[i], 1);
      cxs::mbar_init(&bars->o_free[i], 4);
    }
    for (int w = 0; w < 8; ++w) cxs::mbar_init(&bars->turn[w / 4][w % 4], 1);
    for (int i = 0; i < 2; ++i) cxs::mbar_init(&bars->drain[i], 1);
    bars->abort = 0;
    bars->nans = 0;
    cxs::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     cxs::smem_addr(&bars->tmem)),
                 "r"(kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (SHARED) asm volatile("griddepcontrol.wait;" ::: "memory");
  // Costs (tiles, and kItemCost for each item) and items before each user: a
  // warp adds up a user's row tiles, one warp scans.
  for (int b = warp; !SHARED && b < z.users; b += kThreads / 32) {
    int bad = 0;
    const Span s = user_span(a, z, b, &bad);
    const int rows = s.count * z.group, row_tiles = (rows + kTileRows - 1) / kTileRows;
    long long n = 0;
    for (int r = lane; r < row_tiles; r += 32) {
      int first;
      n += key_tiles(a, z, s, rows, r, &first) + kItemCost;
    }
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) {
      prefix[b + 1] = n * c.kv_heads;
      counts[b + 1] = row_tiles * c.kv_heads;
      if (bad && blockIdx.x == 0) report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
    }
  }
  __syncthreads();
  if (!SHARED && warp == 0) {
    long long base = 0;
    int items = 0;
    if (lane == 0) prefix[0] = 0, counts[0] = 0;
    for (int b0 = 0; b0 < z.users; b0 += 32) {
      const int b = b0 + lane;
      long long sum = b < z.users ? prefix[b + 1] : 0;
      int count = b < z.users ? counts[b + 1] : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        const int more = __shfl_up_sync(0xffffffffu, count, o);
        if (lane >= o) sum += up, count += more;
      }
      if (b < z.users) prefix[b + 1] = base + sum, counts[b + 1] = items + count;
      base += __shfl_sync(0xffffffffu, sum, 31);
      items += __shfl_sync(0xffffffffu, count, 31);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
  const long long total = SHARED ? plan.shares[blockIdx.x].total : prefix[z.users];
  const Shares shares(total, z);
  Partial* const partials = reinterpret_cast<Partial*>(a.workspace);
  Partial& mine = partials[blockIdx.x];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) mine.parts = 0;
  float* const scratch = reinterpret_cast<float*>(partials + z.grid) +
                         (long long)blockIdx.x * 2 * kTileRows * (D + 2);

  // The item that place `at` among all costs falls into; returns the tile there
  // (the item's first one, if `at` is in the item's own cost). Every warp
  // looks for itself.
  auto locate = [&](long long at, Item& p) -> long long {
    int l = 0, h = z.users - 1;
    while (l < h) {
      const int m = (l + h) / 2;
      if (prefix[m + 1] > at) h = m; else l = m + 1;
    }
    int bad = 0;
    p.user = l;
    p.span = user_span(a, z, l, &bad);
    p.rows = p.span.count * z.group;
    long long before = prefix[l];  // cost before row tile r0
    for (int r0 = 0;; r0 += 32) {
      const int r = r0 + lane;
      int first = 0, n = 0;
      if ((long long)r * kTileRows < p.rows) n = key_tiles(a, z, p.span, p.rows, r, &first) + kItemCost;
      long long sum = (long long)n * c.kv_heads;
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > at);
      if (past) {
        const int in = __ffs(past) - 1, cost = __shfl_sync(0xffffffffu, n, in);
        const long long start = before + __shfl_sync(0xffffffffu, sum, in) - (long long)cost * c.kv_heads;
        p.tile_row = r0 + in;
        p.first = __shfl_sync(0xffffffffu, first, in);
        p.kv_head = (int)divide(at - start, cost);
        p.index = counts[l] + (long long)p.tile_row * c.kv_heads + p.kv_head;
        const long long begin = start + (long long)p.kv_head * cost;
        p.begin = begin - kItemCost * p.index;
        p.end = p.begin + cost - kItemCost;
        return p.begin + max(at - begin - kItemCost, 0ll);
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
      if ((r0 + 32) * (long long)kTileRows >= p.rows) return 0;  // (not reached)
    }
  };
  long long lo = 0, hi = 0;
  Item item = {};
  if constexpr (SHARED) {
    const SharePlan share = plan.shares[blockIdx.x];
    if ((int)blockIdx.x < shares.count) {
      lo = share.low;
      hi = share.high;
      plan_item(share.item, z, share.id, share.kv_head, c.kv_heads, item);
    }
  } else if ((int)blockIdx.x < shares.count) {
    hi = (int)blockIdx.x + 1 < shares.count ? locate(shares.begin(blockIdx.x + 1), item)
                                            : total - (long long)kItemCost * counts[z.users];
    lo = locate(shares.begin(blockIdx.x), item);
  }
  // The item after `p` (there is one: its tiles end before the share does).
  auto next = [&](Item& p) {
    const long long n = p.end - p.begin;
    p.begin = p.end;
    ++p.index;
    if (++p.kv_head < c.kv_heads) {
      p.end = p.begin + n;
      return;
    }
    p.kv_head = 0;
    if constexpr (SHARED) {
      plan_item(plan.items[p.id + 1], z, p.id + 1, 0, c.kv_heads, p);
      return;
    }
    ++p.tile_row;
    if ((long long)p.tile_row * kTileRows >= p.rows) {
      do ++p.user;
      while (counts[p.user + 1] == counts[p.user]);
      int bad = 0;
      p.span = user_span(a, z, p.user, &bad);
      p.rows = p.span.count * z.group;
      p.tile_row = 0;
    }
    p.end = p.begin + key_tiles(a, z, p.span, p.rows, p.tile_row, &p.first);
  };
  // SHARED, P over S, and no item of the call has rows for group 1: its columns are
  // a second S, so that the next tile's S need not wait for this one's P V (8 users'
  // 32 candidates, 8 KV heads of 128: 110 us against 100).
  const bool solo = SHARED && !L::kApart && plan.shares[blockIdx.x].solo;
  // Whether the item has rows for group g.
  auto active = [&](const Item& p, int g) { return p.rows - p.tile_row * kTileRows > 128 * g; };

  if (warp < kConvertWarp) {
    // ------------------------------------------------------------ softmax ---
    more_registers<kSoftmaxRegs>();
    const int g = warp / 4, r = threadIdx.x % 128;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t s_of = tmem + lanes + 128 * g, p_of = tmem + lanes + L::kP + L::kPStep * g;
    const uint32_t o_at = tmem + lanes + L::kO + D * g;
    uint8_t* const q_panels = smem + L::kQ + g * L::kPanels * kPanel;
    int tiles = 0;    // of the share
    int mine_s = 0;   // tiles of this group
    int turns = 0;    // tiles that both groups have had
    float m = -kInf, l = 0.f, back = 1.f;
    // The P V of this group's last tile. (solo: two may be on their way, each with a
    // barrier of its own, for a barrier's parity tells two phases apart, not three.)
    const auto last_o = [&]() {
      const int n = mine_s - 1;
      return warp_wait(&bars->o_done[solo ? n & 1 : g], solo ? n >> 1 : n, bars, c.error);
    };
    bool pending = false;  // an item whose O is still in TMEM:
    Item ended = {};
    long long started = lo;
    long long tile = lo;
    while (true) {
      for (; tile < hi && !active(item, g);) {  // items without rows for this group
        const long long until = item.end < hi ? item.end : hi;
        tiles += (int)(until - tile);
        tile = until;
        if (until < hi) next(item);
      }
      if (tile < hi) {
        // The warp's 32 rows of queries, scaled by a power of two each (and the
        // scale's sign), into the group's Q panels, before the last item's O
        // is written: S of this item may start meanwhile. D / 8 lanes read a
        // row together (a lane for each row would touch 32 lines at once).
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kBatch = 8;  // rows
        int row = item.tile_row * kTileRows + 32 * (warp % 8) + lane / kLanes;
        int token = row / z.group, head = row - token * z.group;
#pragma unroll 1
        for (int b0 = 0; b0 < 32; b0 += kAtOnce * kBatch) {
          uint4 in[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            in[j] = make_uint4(0, 0, 0, 0);
            if (row < item.rows) {
              const T* const from =
                  (const T*)a.query + (long long)(item.span.first + token) * a.q_token_stride +
                  (long long)(item.kv_head * z.group + head) * a.q_head_stride + 8 * (lane % kLanes);
              if (((uintptr_t)from & 15) == 0) {
                in[j] = *reinterpret_cast<const uint4*>(from);
              } else {
                alignas(16) T x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = from[e];
                in[j] = *reinterpret_cast<const uint4*>(x);
              }
            }
            row += kAtOnce;
            for (head += kAtOnce; head >= z.group; head -= z.group) ++token;
          }
          // (Two copies of a long loop that runs from a cold instruction cache: 8 cost 5 us.)
#pragma unroll 2
          for (int j = 0; j < kBatch; ++j) {
            const int r32 = b0 + j * kAtOnce + lane / kLanes, r128 = 32 * (warp % 4) + r32;
            alignas(16) T x[8];
            *reinterpret_cast<uint4*>(x) = in[0];
#pragma unroll
            for (int k = 1; k < kBatch; ++k) in[k - 1] = in[k];
            float v[8], top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[e] = to_float(x[e]);
              if (fabsf(v[e]) < kInf) top = fmaxf(top, fabsf(v[e]));
            }
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1)
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            if (e < -100) e = -100;
            if (top == 0.f) e = 14;
            float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            if (a.scale < 0.f) up = -up;
            if (a.scale == 0.f) up = 0.f;  // every score is 0
            const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
            // The inverse goes to the row's own lane.
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
              const float its = __shfl_sync(0xffffffffu, down, k * kLanes);
              if (lane == b0 + j * kAtOnce + k) back = its;
            }
            const int chunk = lane % kLanes;
            *reinterpret_cast<uint4*>(q_panels + chunk / 8 * kPanel +
                                      tc::sw128_chunk(r128, chunk % 8)) =
                make_uint4(pack_half2(v[0] * up, v[1] * up), pack_half2(v[2] * up, v[3] * up),
                           pack_half2(v[4] * up, v[5] * up), pack_half2(v[6] * up, v[7] * up));
          }
        }
        cxs::fence_proxy_async_shared();
        warp_arrive(&bars->q_full[g], lane);
      }
      if (pending) {
        // The ended item's O: the result, or this share's part of it.
        if (!last_o()) goto done;
        tc::fence_after();
        const long long until = ended.end < hi ? ended.end : hi;
        const bool complete = started == ended.begin && until == ended.end;
        float* const part = scratch + (started == ended.begin ? kTileRows * (D + 2) : 0);
        const bool some = !(l == 0.f);
        const float inv = some ? 1.f / l : 0.f;
        const int row = ended.tile_row * kTileRows + 128 * g + r;
        const bool live = row < ended.rows;
        const long long head = (long long)(ended.span.first + row / z.group) * a.heads +
                               ended.kv_head * z.group + row % z.group;
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          float o[32];
          __syncwarp();
          tc::ld32(o_at + 32 * q, o);
          if (live && complete) {
            alignas(16) T y[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = from_float<T>(some ? o[e] * inv : 0.f);
            uint4* out = reinterpret_cast<uint4*>((T*)a.out + head * D + 32 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = reinterpret_cast<const uint4*>(y)[e];
          } else if (live) {
            float4* out = reinterpret_cast<float4*>(part + (128 * g + r) * D + 32 * q);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              out[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        tc::fence_before();
        warp_arrive(&bars->o_free[g], lane);
        if (live && complete) {
          if (a.lse) a.lse[head] = some ? (m - kHead + log2f(l)) * kLn2 : -kInf;
        } else if (live) {
          part[kTileRows * D + 2 * (128 * g + r)] = m - kHead;  // what O and l are relative to
          part[kTileRows * D + 2 * (128 * g + r) + 1] = l;
        }
        // (Set before the last of these V was ready, or by an earlier item.)
        if (FORMAT == CXS_FORMAT_E4M3 && *(volatile int*)&bars->nans && live) {
          const long long half_page = (long long)c.page_size * D;
          const uint8_t* const v_codes =
              (const uint8_t*)c.codes + (2 * ended.kv_head + 1) * half_page;
          float* const its_part = complete ? nullptr : part + (128 * g + r) * D;
          if constexpr (SHARED) {
            // (Of a user's own keys all, whichever share has them: a NaN stays.)
            int user, end;
            own_range(a, plan, z, ended, row, &user, &end);
            mark_nans<T, D>(v_codes, 2 * c.kv_heads * half_page, c.pages,
                            c.table + user * c.table_stride, c.page_size, ended.span.length, end,
                            make_int2(0, 0), (T*)a.out + head * D, its_part, 0, D);
          } else {
            const int2 see = row_range(a, ended.span, row / z.group);
            const int2 all = seen_by_all(a, z, ended.span, ended.tile_row * kTileRows,
                                         min(ended.rows, (ended.tile_row + 1) * kTileRows) - 1);
            const int key = (ended.first + (int)(started - ended.begin)) * kKeys;
            // (Tiles that every row sees whole went as they are.)
            mark_nans<T, D>(v_codes, 2 * c.kv_heads * half_page, c.pages,
                            c.table + ended.user * c.table_stride, c.page_size, max(see.x, key),
                            min(see.y, key + (int)(until - started) * kKeys),
                            make_int2((all.x + kKeys - 1) / kKeys * kKeys, all.y / kKeys * kKeys),
                            (T*)a.out + head * D, its_part, 0, D);
          }
        }
        __syncwarp();
        if (!complete && started == ended.begin && g == 0 && r == 0) {
          const int last = shares.of(ended.end - 1 + kItemCost * (ended.index + 1));
          mine.first = ended.span.first;
          mine.rows = ended.rows;
          mine.row0 = ended.tile_row * kTileRows;
          mine.kv_head = ended.kv_head;
          mine.parts = last - (int)blockIdx.x + 1;
        }
      }
      if (tile >= hi) break;

      const long long until = item.end < hi ? item.end : hi;
      const int count = (int)(until - tile);
      const int row = item.tile_row * kTileRows + 128 * g + r;
      int2 see, own = make_int2(0, 0);  // keys of the item's tiles that the row sees
      if constexpr (SHARED) {
        see = make_int2(0, item.span.length);
        if (row < item.rows) {
          int user, end;
          const int at = item.common_tiles * kKeys + own_range(a, plan, z, item, row, &user, &end);
          own = make_int2(at + item.span.length % 16, at + end - item.span.length / 16 * 16);
        }
      } else {
        see = row < item.rows ? row_range(a, item.span, row / z.group)
                              : make_int2(0, item.span.length);
      }
      m = -kInf;
      l = 0.f;
      int key0 = (item.first + (int)(tile - item.begin)) * kKeys;
#pragma unroll 1
      for (int i = 0; i < count; ++i, ++tiles, ++mine_s, key0 += kKeys) {
        // (Tile t was described before the K that S was computed from came.)
        // (solo: two S on their way at once, each with a barrier of its own.)
        if (!warp_wait(&bars->s_full[solo ? mine_s & 1 : g], solo ? mine_s >> 1 : mine_s, bars, c.error))
          goto done;
        tc::fence_after();
        const Tile& tile_info = ring[tiles % kRing];
        const uint32_t second = solo && (mine_s & 1) ? 128 : 0;
        const uint32_t s_at = s_of + second, p_at = p_of + second;
        int from = see.x - key0, to = see.y - key0;  // visible columns
        if (SHARED && key0 >= item.common_tiles * kKeys) from = own.x - key0, to = own.y - key0;
        const unsigned missing = tile_info.missing;
        // A run's factor; never 0, which times a hidden score would be NaN
        // (scores that small are 0 either way); NaN stays NaN.
        auto factor_of = [&](float run) {
          const float f = run * back;
          return f < 1.2e-38f ? 1.2e-38f : f;
        };
        if constexpr (SHARED) {
          // Half of the columns in registers at a time: the second half first, for the
          // maximum alone, then the first for both, then the second again. (With all
          // of them there are no registers left to have loads and exponentials in
          // flight: the suffix case 160 us against 155.)
          uint32_t x[kKeys / 2];
          const bool edge = !__all_sync(0xffffffffu, from <= 0 && to >= kKeys && missing == 0);
          auto load = [&](int half) {
            ld64(s_at + 64 * half, x);
            if (!edge) return;
            // What the row does not see becomes -infinity.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int q = 2 * half + h;
              const int low = min(max(from - 32 * q, 0), 32), high = min(max(to - 32 * q, 0), 32);
              unsigned seen =
                  (high == 32 ? ~0u : (1u << high) - 1) & ~(low == 32 ? ~0u : (1u << low) - 1);
              if (missing >> (2 * q) & 1) seen &= 0xffff0000u;
              if (missing >> (2 * q + 1) & 1) seen &= 0x0000ffffu;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                x[32 * h + e] = seen >> e & 1 ? x[32 * h + e] : 0xff800000u;
            }
          };
          float top = -kInf, factor[kRuns], lift[kRuns];
#pragma unroll
          for (int half = 1; half >= 0; --half) {
            load(half);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int u = 4 * half + h;
              const float2 run = *reinterpret_cast<const float2*>(&tile_info.runs[u]);
              factor[u] = factor_of(run.x);
              lift[u] = run.y;
              float t = max3(x[16 * h], x[16 * h + 1], x[16 * h + 2]);
#pragma unroll
              for (int e = 3; e < 15; e += 2) t = max3(__float_as_uint(t), x[16 * h + e], x[16 * h + e + 1]);
              t = fmaxf(t, __uint_as_float(x[16 * h + 15]));
              top = fmaxf(top, fmaf(t, factor[u], lift[u]));
            }
          }
          // (Another user's runs count for nothing, whatever their scales are. The
          // maximum passes over the NaN that comes of one times -infinity.)
          if (missing & kWild) {
#pragma unroll
            for (int u = 0; u < kRuns; ++u)
              if (from >= 16 * u + 16 || to <= 16 * u) factor[u] = 1.f, lift[u] = 0.f;
          }
          const bool grows = top > m + kLag;
          // The last tile's P V is done: O may be rescaled and P overwritten.
          // (With P over S, S of this tile came after it.)
          if (L::kApart && mine_s > 0) {
            if (!warp_wait(&bars->o_done[g], mine_s - 1, bars, c.error)) goto done;
            tc::fence_after();
          }
          if (__any_sync(0xffffffffu, grows)) {
            if (solo && mine_s > 0) {
              if (!last_o()) goto done;
              tc::fence_after();
            }
            const float f = !grows ? 1.f : m == -kInf ? 0.f : ex2(m - top);
            if (grows) m = top;
            l *= f;
            if (i > 0) {
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                float o[16];
                tc::ld16(o_at + d, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f;
                tc::st16(o_at + d, o);
              }
            }
          }
          const float base = m == -kInf ? 0.f : m - kHead;
          // The groups' exponentials in turn, half a tile apart: one's wait for S, its
          // maximum and its stores then lie beside the other's: 139 us against 143.
          const bool two = active(item, 1);
          if (two && (g == 1 || turns > 0)) {
            if (!warp_wait(&bars->turn[g][warp % 4], turns - (g == 0), bars, c.error)) goto done;
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 1) {
              load(1);
              if (L::kApart) {  // S of the next tile may come
                tc::fence_before();
                warp_arrive(&bars->s_free[g], lane);
              }
              if (two) warp_arrive(&bars->turn[1 - g][warp % 4], lane);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t p[16];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int u = 4 * half + 2 * q + h;
                const float shift = lift[u] - base;
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const uint32_t* const s2 = x + 32 * q + 16 * h + e;
                  float2 y = __ffma2_rn(make_float2(__uint_as_float(s2[0]), __uint_as_float(s2[1])),
                                        make_float2(factor[u], factor[u]), make_float2(shift, shift));
                  y = make_float2(ex2(y.x), ex2(y.y));
                  sum = __fadd2_rn(sum, y);
                  p[8 * h + e / 2] = pack_half2(y.x, y.y);
                }
                l = fmaf(sum.x + sum.y, tile_info.runs[u].z, l);
              }
              st16(p_at + 32 * half + 16 * q, p);
            }
          }
          turns += two;
        } else {
          uint32_t x[kKeys];
          ld64(s_at, x);
          ld64(s_at + 64, x + 64);
          if (L::kApart) {  // S of the next tile may come
            tc::fence_before();
            warp_arrive(&bars->s_free[g], lane);
          }
          if (!__all_sync(0xffffffffu, from <= 0 && to >= kKeys && missing == 0)) {
            // What the row does not see becomes -infinity.
#pragma unroll
            for (int q = 0; q < kKeys / 32; ++q) {
              const int low = min(max(from - 32 * q, 0), 32), high = min(max(to - 32 * q, 0), 32);
              unsigned seen =
                  (high == 32 ? ~0u : (1u << high) - 1) & ~(low == 32 ? ~0u : (1u << low) - 1);
              if (missing >> (2 * q) & 1) seen &= 0xffff0000u;
              if (missing >> (2 * q + 1) & 1) seen &= 0x0000ffffu;
#pragma unroll
              for (int e = 0; e < 32; ++e) x[32 * q + e] = seen >> e & 1 ? x[32 * q + e] : 0xff800000u;
            }
          }
          float top = -kInf;
#pragma unroll
          for (int u = 0; u < kRuns; ++u) {
            const float2 run = *reinterpret_cast<const float2*>(&tile_info.runs[u]);
            float t0 = __uint_as_float(x[16 * u]), t1 = __uint_as_float(x[16 * u + 1]);
#pragma unroll
            for (int e = 2; e < 16; e += 2) {
              t0 = fmaxf(t0, __uint_as_float(x[16 * u + e]));
              t1 = fmaxf(t1, __uint_as_float(x[16 * u + e + 1]));
            }
            top = fmaxf(top, fmaf(fmaxf(t0, t1), factor_of(run.x), run.y));
          }
          const bool grows = top > m + kLag;
          // The last tile's P V is done: O may be rescaled and P overwritten.
          // (With P over S, S of this tile came after it.)
          if (L::kApart && mine_s > 0) {
            if (!warp_wait(&bars->o_done[g], mine_s - 1, bars, c.error)) goto done;
            tc::fence_after();
          }
          if (__any_sync(0xffffffffu, grows)) {
            const float f = !grows ? 1.f : m == -kInf ? 0.f : ex2(m - top);
            if (grows) m = top;
            l *= f;
            if (i > 0) {
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                float o[16];
                tc::ld16(o_at + d, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f;
                tc::st16(o_at + d, o);
              }
            }
          }
          const float base = m == -kInf ? 0.f : m - kHead;
#pragma unroll
          for (int q = 0; q < kKeys / 32; ++q) {
            uint32_t p[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 run = tile_info.runs[2 * q + h];
              const float factor = factor_of(run.x), shift = run.y - base;
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const uint32_t* const s2 = x + 32 * q + 16 * h + e;
                float2 y = __ffma2_rn(make_float2(__uint_as_float(s2[0]), __uint_as_float(s2[1])),
                                      make_float2(factor, factor), make_float2(shift, shift));
                y = make_float2(ex2(y.x), ex2(y.y));
                sum = __fadd2_rn(sum, y);
                p[8 * h + e / 2] = pack_half2(y.x, y.y);
              }
              l = fmaf(sum.x + sum.y, run.z, l);
            }
            st16(p_at + 16 * q, p);
          }
        }
        tc::wait_st();
        tc::fence_before();
        warp_arrive(&bars->p_full[solo ? mine_s & 1 : g], lane);
      }
      pending = true;
      ended = item;
      started = tile;
      tile = until;
      if (until < hi) next(item);
    }
  } else if (warp < kMmaWarp) {
    // --------------------------------------------------------- conversion ---
    fewer_registers<kConvertRegs>();
    // A thread's 16 codes: chunk `chunk` of 64 channels (a panel), key `key` of
    // each pass. Eight neighbouring lanes take four chunks of two keys, for
    // D = 128 of different panels: their reads and their writes then each
    // cover all banks.
    const int i = threadIdx.x - 32 * kConvertWarp, chunk = i % 4;
    const int panel = D == 64 ? 0 : (i / 8 % 2) ^ (i / 4 % 2);
    const int key = D == 64 ? i / 4 : i / 16 * 2 + i / 4 % 2;
    constexpr int kStep = 128 * 16 / D;         // keys of one pass of the 128 threads
    const int from = key * D + panel * 64 + chunk * 16;
    const int to0 = panel * kPanel + tc::sw128_chunk(key, 2 * chunk);
    const int to1 = panel * kPanel + tc::sw128_chunk(key, 2 * chunk + 1);
    // Codes -> fp16 in the operand's layout; keys without a token become 0 (a
    // probability of 0 times whatever their bytes hold could be NaN).
    // So do NaN codes of V in a tile that hides keys from some row.
    auto convert = [&](const uint8_t* raw, uint8_t* panels, const Tile& tile, int part) {
      const unsigned missing = tile.missing;
      const int left = tile.left;
      const bool hidden = FORMAT == CXS_FORMAT_E4M3 && part && tile.flags & kHidden;
      auto pass = [&](int at, uint4 w) {
        *reinterpret_cast<uint4*>(panels + to0 + at * 128) =
            make_uint4(half2_of<FORMAT>(w.x, 0), half2_of<FORMAT>(w.x, 1),
                       half2_of<FORMAT>(w.y, 0), half2_of<FORMAT>(w.y, 1));
        *reinterpret_cast<uint4*>(panels + to1 + at * 128) =
            make_uint4(half2_of<FORMAT>(w.z, 0), half2_of<FORMAT>(w.z, 1),
                       half2_of<FORMAT>(w.w, 0), half2_of<FORMAT>(w.w, 1));
      };
      if (left >= kKeys && missing == 0 && !hidden) {
#pragma unroll 4
        for (int at = 0; at < kKeys; at += kStep)
          pass(at, *reinterpret_cast<const uint4*>(raw + from + at * D));
      } else {
        uint32_t found = 0;
#pragma unroll 1
        for (int at = 0; at < kKeys; at += kStep) {
          bool here = key + at < left && !(missing >> ((key + at) / 16) & 1);
          if (SHARED) here &= (key + at) % 16 < (int)tile.runs[(key + at) / 16].w;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (here) w = *reinterpret_cast<const uint4*>(raw + from + at * D);
          if (hidden) w = without_nan(w, &found);
          pass(at, w);
        }
        if (found) *(volatile int*)&bars->nans = 1;
      }
    };
    const int n = (int)(hi - lo);
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        const int raw = stage_of<L::kRawStages>(t);
        const int to = part ? stage_of<L::kVStages>(t) : stage_of<L::kKStages>(t);
        const int use = part ? phase_of<L::kVStages>(t) : phase_of<L::kKStages>(t);
        if (!warp_wait(&bars->raw_full[raw][part], phase_of<L::kRawStages>(t), bars, c.error)) goto done;
        if (!warp_wait(part ? &bars->v_free[to] : &bars->k_free[to], use + 1, bars, c.error)) goto done;
        convert(smem + L::kRaw + (2 * raw + part) * L::kRawPart,
                smem + (part ? L::kV : L::kK) + to * L::kPanels * kPanel, ring[t % kRing], part);
        cxs::fence_proxy_async_shared();
        warp_arrive(part ? &bars->v_full[to] : &bars->k_full[to], lane);
        if (lane == 0) cxs::mbar_arrive(&bars->raw_free[raw][part]);
      }
    }
  } else {
    // ---------------------------------------------------------------- MMAs ---
    fewer_registers<kOtherRegs>();
    // The whole warp walks the tiles, so that what the MMAs need stays in
    // uniform registers; one elected lane issues them.
    if (!SHARED && warp == kMmaWarp && lo < hi) {
      const uint32_t base = cxs::smem_addr(smem);
      constexpr uint32_t kPanel16 = kPanel / 16;  // descriptors count 16-byte units
      const uint64_t dq = tc::desc_sw128(base + L::kQ, 16, 1024);
      const uint64_t dk = tc::desc_sw128(base + L::kK, 16, 1024);
      // V is read channel-major: 64-channel panels kPanel apart, 8 keys 1024.
      const uint64_t dv = tc::desc_sw128(base + L::kV, kPanel, 1024);
      const uint32_t id_s = idesc_f16(128, 128, 0), id_o = idesc_f16(128, D, 1);
      const int count = (int)(hi - lo);
      // Tiles whose K and V have come: seen in order, since a group that has no
      // rows for some tiles may ask for one long after the next has taken its
      // stage (the barrier's parity then says nothing).
      int k_ready = 0, v_ready = 0;
      auto ready = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, test_wait(bar, phase & 1));
      };
      auto have_k = [&](int n) {
        if (n == k_ready && ready(&bars->k_full[stage_of<L::kKStages>(n)], phase_of<L::kKStages>(n)))
          ++k_ready;
        return n < k_ready;
      };
      auto have_v = [&](int n) {
        if (n == v_ready && ready(&bars->v_full[n & 1], n >> 1)) ++v_ready;
        return n < v_ready;
      };
      // Next tile and uses of the barriers so far, by group.
      int s_next[2] = {0, 0}, s_items[2] = {0, 0}, s_tiles[2] = {0, 0};
      int o_next[2] = {0, 0}, o_items[2] = {0, 0}, o_tiles[2] = {0, 0};
      // S of group g's next tile, if what it needs is there: K, the item's
      // queries, and its columns (read, or with P over S: their P V issued).
      auto try_s = [&](int g) -> bool {
        const int n = s_next[g], stage = stage_of<L::kKStages>(n);
        if (n >= count || (!L::kApart && n > o_next[g]) || !have_k(n)) return false;
        const int flags = ring[n % kRing].flags;
        if (g == 1 && !(flags & kTwo)) {  // not for this group
          ++s_next[1];
          if (o_next[1] == n) ++o_next[1];
          return true;
        }
        if ((flags & kFirst) && !ready(&bars->q_full[g], s_items[g])) return false;
        if (L::kApart && s_tiles[g] > 0 && !ready(&bars->s_free[g], s_tiles[g] - 1)) return false;
        s_items[g] += flags & kFirst ? 1 : 0;
        ++s_tiles[g];
        ++s_next[g];
        tc::fence_after();
        const uint64_t q = dq + g * L::kPanels * kPanel16;
        const uint64_t k = dk + stage * L::kPanels * kPanel16;
        // The last to use this K: the other group has, or has no rows.
        const bool last = !(flags & kTwo) || s_next[1 - g] > n;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_ss(tmem + 128 * g, q + i / 4 * kPanel16 + 2 * (i % 4),
                   k + i / 4 * kPanel16 + 2 * (i % 4), id_s, i > 0);
          tc::commit(&bars->s_full[g]);
          if (last) tc::commit(&bars->k_free[stage]);
        }
        __syncwarp();
        return true;
      };
      // O of group g's next tile, if its P and V are there (and, for an item's
      // first tile, the last item's O has been read).
      auto try_o = [&](int g) -> bool {
        const int n = o_next[g];
        if (n >= s_next[g]) return false;
        const int flags = ring[n % kRing].flags;
        if (g == 1 && !(flags & kTwo)) {
          ++o_next[1];
          return true;
        }
        if (!ready(&bars->p_full[g], o_tiles[g])) return false;
        if (!have_v(n)) return false;
        if ((flags & kFirst) && o_items[g] > 0 && !ready(&bars->o_free[g], o_items[g] - 1))
          return false;
        o_items[g] += flags & kFirst ? 1 : 0;
        ++o_tiles[g];
        ++o_next[g];
        tc::fence_after();
        const uint64_t v = dv + (n & 1) * L::kPanels * kPanel16;
        const bool last = !(flags & kTwo) || o_next[1 - g] > n;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            mma_ts(tmem + L::kO + D * g, tmem + L::kP + L::kPStep * g + 8 * i, v + 128 * i, id_o,
                   !(flags & kFirst) || i > 0);
          tc::commit(&bars->o_done[g]);
          if (last) tc::commit(&bars->v_free[n & 1]);
        }
        __syncwarp();
        return true;
      };
      // Whatever is ready, a group's P V and then its next S: the groups then
      // run half a tile apart, and one's softmax hides the other's MMAs.
      bool fine = true;
      long long since = clock64();
      while (o_next[0] < count || o_next[1] < count) {
        bool some = try_o(0);
        some |= try_s(0);
        some |= try_o(1);
        some |= try_s(1);
        if (some) {
          since = clock64();
        } else if (__any_sync(0xffffffffu, *(volatile int*)&bars->abort ||
                                               clock64() - since > kSpinLimit)) {
          if (!*(volatile int*)&bars->abort) report(c.error, CXS_DEVICE_ERR_COPY_TIMEOUT);
          *(volatile int*)&bars->abort = 1;
          fine = false;
          break;
        }
      }
      if (!fine) {  // let the MMAs in flight end before TMEM is freed
        if (elect_one()) tc::commit(&bars->drain[0]);
        __syncwarp();
        const long long start = clock64();
        while (!cxs::mbar_try_wait(&bars->drain[0], 0) && clock64() - start < kSpinLimit) {
        }
      }
      // SHARED: a warp for each group, which sleeps on what must come next. (One that
      // looks for whatever is ready in both groups notices a P late: a tile took
      // 4200 cycles in the place of 3600. Without SHARED and for 128 channels it is
      // the other way round, 613 us against 650: the groups then stay in turn.)
    } else if (SHARED && (warp == kMmaWarp || warp == kMmaWarp + 2) && lo < hi) {
      const int g = warp != kMmaWarp;
      const uint32_t base = cxs::smem_addr(smem);
      constexpr uint32_t kPanel16 = kPanel / 16;  // descriptors count 16-byte units
      const uint64_t dq = tc::desc_sw128(base + L::kQ, 16, 1024) + g * L::kPanels * kPanel16;
      const uint64_t dk = tc::desc_sw128(base + L::kK, 16, 1024);
      // V is read channel-major: 64-channel panels kPanel apart, 8 keys 1024.
      const uint64_t dv = tc::desc_sw128(base + L::kV, kPanel, 1024);
      const uint32_t id_s = idesc_f16(128, 128, 0), id_o = idesc_f16(128, D, 1);
      const int count = (int)(hi - lo);
      int s_items = 0, s_tiles = 0, o_items = 0, o_tiles = 0;  // of this group, so far
      // S of tile n: K, the item's queries and (read, or with P over S: their P V
      // issued) its columns.
      auto issue_s = [&](int n) -> bool {
        const int stage = stage_of<L::kKStages>(n);
        if (!warp_wait(&bars->k_full[stage], phase_of<L::kKStages>(n), bars, c.error)) return false;
        const int flags = ring[n % kRing].flags;
        if (g == 1 && !(flags & kTwo)) {  // not for this group
          if (lane == 0) cxs::mbar_arrive(&bars->k_free[stage]);
          return true;
        }
        if ((flags & kFirst) && !warp_wait(&bars->q_full[g], s_items++, bars, c.error)) return false;
        if (L::kApart && s_tiles > 0 && !warp_wait(&bars->s_free[g], s_tiles - 1, bars, c.error))
          return false;
        ++s_tiles;
        tc::fence_after();
        const uint64_t k = dk + stage * L::kPanels * kPanel16;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_ss(tmem + 128 * (solo ? n & 1 : g), dq + i / 4 * kPanel16 + 2 * (i % 4),
                   k + i / 4 * kPanel16 + 2 * (i % 4), id_s, i > 0);
          tc::commit(&bars->s_full[solo ? n & 1 : g]);
          tc::commit(&bars->k_free[stage]);
        }
        __syncwarp();
        return true;
      };
      // O of tile n: its P and V and, for an item's first tile, the last item's O
      // read.
      auto issue_o = [&](int n) -> bool {
        if (!warp_wait(&bars->v_full[n & 1], n >> 1, bars, c.error)) return false;
        const int flags = ring[n % kRing].flags;
        if (g == 1 && !(flags & kTwo)) {
          if (lane == 0) cxs::mbar_arrive(&bars->v_free[n & 1]);
          return true;
        }
        if (!warp_wait(&bars->p_full[solo ? n & 1 : g], solo ? n >> 1 : o_tiles, bars, c.error))
          return false;
        ++o_tiles;
        if (flags & kFirst) {
          if (o_items > 0 && !warp_wait(&bars->o_free[g], o_items - 1, bars, c.error)) return false;
          ++o_items;
        }
        tc::fence_after();
        const uint64_t v = dv + (n & 1) * L::kPanels * kPanel16;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            mma_ts(tmem + L::kO + D * g, tmem + L::kP + (solo ? 128 * (n & 1) : L::kPStep * g) + 8 * i,
                   v + 128 * i, id_o,
                   !(flags & kFirst) || i > 0);
          tc::commit(&bars->o_done[solo ? n & 1 : g]);
          tc::commit(&bars->v_free[n & 1]);
        }
        __syncwarp();
        return true;
      };
      // Where P has its own columns S of the next tile goes before P V of this one,
      // but at an item's end: the next item's queries come later.
      bool fine = issue_s(0);
#pragma unroll 1
      for (int n = 0; fine && n < count; ++n) {
        const bool o_first = (!L::kApart && !solo) || (ring[n % kRing].flags & kLast);
        if (o_first) fine = issue_o(n);
        if (fine && n + 1 < count) fine = issue_s(n + 1);
        if (fine && !o_first) fine = issue_o(n);
      }
      if (!fine) {  // let the MMAs in flight end before TMEM is freed
        if (elect_one()) tc::commit(&bars->drain[g]);
        __syncwarp();
        const long long start = clock64();
        while (!cxs::mbar_try_wait(&bars->drain[g], 0) && clock64() - start < kSpinLimit) {
        }
      }
    } else if (warp == kLoadWarp) {
      // -------------------------------------------------------------- loads ---
      const int page_bits = __ffs(c.page_size) - 1, entries = kKeys >> page_bits;
      const int page_bytes = c.page_size * D;
      const float unit = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
      const int n = (int)(hi - lo);
      long long tile = lo;
      // Lane e: the id of the e-th page of the tile at `tile` (looked up one
      // tile early), -1 where it has no token or none that a row sees.
      // (SHARED, past the common keys: of its e-th run, with the run's place in the
      // page and keys.)
      int slot = 0, held = 0;
      auto look_up = [&]() {
        if constexpr (SHARED) {
          const long long in = tile - item.begin - item.common_tiles;
          if (in >= 0) return own_run(a, plan, item, in * kRuns + lane, lane, &slot, &held);
        }
        const int at = (item.first + (int)(tile - item.begin)) * kKeys + (lane << page_bits);
        const bool needed = lane < entries && at < item.span.length &&
                            at + c.page_size > item.span.begin;
        return needed ? __ldg(c.table + item.user * c.table_stride + (at >> page_bits)) : -2;
      };
      int id = n > 0 ? look_up() : -2;
      int2 all = make_int2(0, 0);  // keys that every row of the item sees
#pragma unroll 1
      for (int t = 0; t < n; ++t) {
        const bool own = SHARED && tile - item.begin >= item.common_tiles;
        if (id != -2 && (id < 0 || id >= c.pages)) report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
        if (id < 0 || id >= c.pages) id = -1;
        const long long cell = ((long long)id * c.kv_heads + item.kv_head) * 2;
        const unsigned pages = __ballot_sync(0xffffffffu, id >= 0);
        // Lane u: the scales of run u of 16 keys.
        const int e = own ? lane % kRuns : (lane % kRuns * 16) >> page_bits;
        const long long its = __shfl_sync(0xffffffffu, cell, e);
        const bool here = pages >> e & 1;
        float sk = 1.f, sv = 1.f;
        if (here && lane < kRuns) {
          sk = __ldg(c.scales + its);
          sv = __ldg(c.scales + its + 1);
        }
        unsigned missing = __ballot_sync(0xffffffffu, lane < kRuns && !here);
        if constexpr (SHARED)
          if (__any_sync(0xffffffffu, !(sk < kInf && sv < kInf))) missing |= kWild;
        const bool first = tile == item.begin || t == 0, last = tile + 1 == item.end || t + 1 == n;
        const int key0 = (item.first + (int)(tile - item.begin)) * kKeys;
        const int left = own ? kKeys : item.span.length - key0;
        const float keys_here = own ? (float)held : 16.f;
        const int copy_bytes = own ? 16 * D : page_bytes;
        if (!SHARED && FORMAT == CXS_FORMAT_E4M3 && first)
          all = seen_by_all(a, z, item.span, item.tile_row * kTileRows,
                            min(item.rows, (item.tile_row + 1) * kTileRows) - 1);
        const bool hidden =
            FORMAT == CXS_FORMAT_E4M3 &&
            (SHARED ? own : key0 < all.x || key0 + min(left, kKeys) > all.y);
        const int flags = (first ? kFirst : 0) | (last ? kLast : 0) | (active(item, 1) ? kTwo : 0) |
                          (hidden ? kHidden : 0);
        const uint8_t* from = (const uint8_t*)c.codes + cell * page_bytes + (own ? slot * D : 0);
        ++tile;
        if (t + 1 < n) {
          if (tile >= item.end) next(item);
          id = look_up();
        }
        const int raw = stage_of<L::kRawStages>(t);
        uint8_t* const to = smem + L::kRaw + 2 * raw * L::kRawPart + lane * copy_bytes;
        const uint32_t bytes = __popc(pages) * copy_bytes;
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          if (!warp_wait(&bars->raw_free[raw][part], phase_of<L::kRawStages>(t) + 1, bars, c.error)) {
            // Copies in flight end before the CTA does (of each barrier, the
            // last use issued: one that has ended is not waited for).
            for (int k = 0; k < 2 * L::kRawStages; ++k) {
              const int use = 2 * t + part - 1 - k;  // of K and V of all tiles, in order
              if (use < 0) break;
              const long long start = clock64();
              while (!cxs::mbar_try_wait(&bars->raw_full[stage_of<L::kRawStages>(use / 2)][use & 1],
                                         phase_of<L::kRawStages>(use / 2) & 1) &&
                     clock64() - start < kSpinLimit) {
              }
            }
            goto done;
          }
          if (part == 0) {
            // K's arrival also tells the other roles that the tile is described.
            Tile& about = ring[t % kRing];
            if (lane < kRuns)
              about.runs[lane] = make_float4(usable_scale(sk) * unit, __log2f(usable_scale(sv)),
                                             !SHARED || sv == sv ? __frcp_rn(usable_scale(sv)) : 1.f,
                                             keys_here);
            if (lane == 0) {
              about.missing = missing;
              about.left = left;
              about.flags = flags;
            }
          }
          __syncwarp();
          if (lane == 0) cxs::mbar_expect_tx(&bars->raw_full[raw][part], bytes);
          __syncwarp();
          if (pages >> lane & 1)
            cxs::bulk_g2s(to + part * L::kRawPart, from + part * page_bytes, copy_bytes,
                          &bars->raw_full[raw][part]);
        }
      }
    }
  }
done:
  __syncwarp();
  if constexpr (SHARED)
    clear_shared<T, D>(a, plan);
  else
    clear_rows<T, D>(a, z, blockIdx.x, gridDim.x, threadIdx.x, kThreads);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem));
}

template <int FORMAT, typename T, int D, bool SHARED>
int launch(const cxs_cache_attend_call& a, const Shape& z, const SharedPlan& plan,
           cudaStream_t stream) {
  static cxs_host::OncePerDevice ready;
  const int status = ready.run([] {
    CXS_CUDA(cudaFuncSetAttribute(tile_kernel<FORMAT, T, D, SHARED>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kBytes));
    return (int)CXS_OK;
  });
  if (status != CXS_OK) return status;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(z.grid);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = Layout<D>::kBytes;
  config.stream = stream;
  cudaLaunchAttribute early = {};  // its setup may run beside the plan's launch
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = SHARED;
  CXS_CUDA(cudaLaunchKernelEx(&config, tile_kernel<FORMAT, T, D, SHARED>, a, z, plan));
  CXS_LAUNCH_CHECK("cache attend");
  return CXS_OK;
}

template <bool SHARED>
int launch_of(const cxs_cache_attend_call& a, const Shape& z, const SharedPlan& plan,
              cudaStream_t stream) {
  CXS_CACHE_FORMAT(a.cache.format, F, {
    if (a.cache.type == CXS_TYPE_BF16)
      return a.cache.dim == 64 ? launch<F, __nv_bfloat16, 64, SHARED>(a, z, plan, stream)
                               : launch<F, __nv_bfloat16, 128, SHARED>(a, z, plan, stream);
    return a.cache.dim == 64 ? launch<F, __half, 64, SHARED>(a, z, plan, stream)
                             : launch<F, __half, 128, SHARED>(a, z, plan, stream);
  });
}

}  // namespace
