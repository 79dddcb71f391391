// Attention over the dense 8-bit cache: few query rows a KV head, the joining
// of partial results, and the entry points.
#include "cache8_attend.cuh"

using cxs_host::set_error;

namespace {

using namespace cxs::cache8;

// D += A B, 16x8x16, fp16 in, fp32 out.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^(x f + shift) of two scores.
__device__ __forceinline__ float2 exp2_pair(float x, float y, float f, float shift) {
  const float2 e =
      __ffma2_rn(make_float2(x, y), make_float2(f, f), make_float2(shift, shift));
  return make_float2(ex2(e.x), ex2(e.y));
}

// ------------------------------------------------- few rows: one warp, 16 ---

// One CTA of 12 warps per SM. Each warp works through its own share; the CTA's
// warps meet once, at the end, to join what they hold of the same items (a
// meeting at every item cost as much as the tiles of a ragged decode batch). A
// warp takes a tile of keys at a time with all
// 16 rows: the tile's runs of K and V codes come by bulk copies, one tile
// ahead, and go from shared memory straight into mma.sync fragments: the
// order of channels within a dot product is free, so a lane's 16 bytes of a
// key are its fragments of four steps, and the order of keys within a tile is
// chosen so that the scores' accumulator is the probabilities' operand and a
// lane's V bytes of four keys pair up by byte permutes. No transposition
// passes through shared memory.
// Measured: 64 users of 0 to 16K tokens, 32 / 2 heads of 64, 137 MB of codes in
// 43 us (3.2 TB/s); 32 users of 8K, 32 / 8 heads of 128, 537 MB in 135 us
// with the join (4.0 TB/s). No unit is full (40 % of the issue slots, ALU 36 %,
// tensor core 22 %): converting codes, and an exponential and about three more
// instructions for each of a key's 16 scores, follow one another in a warp, and
// three warps a scheduler do not cover that. At D = 128 registers are short too
// (254 bytes spilled a thread).
constexpr int kDecodeWarps = 12;

template <int D>
struct Decode {
  static constexpr int kWarps = kDecodeWarps, kThreads = 32 * kWarps;
  static constexpr int kTile = D == 64 ? 64 : 32;     // keys
  static constexpr int kPart = kTile * D;             // bytes of K or V
  static constexpr int kStages = 2;                   // one in work, one coming
  static constexpr int kStage = 2 * kPart;
  static constexpr int kGroups = kTile / 16;          // runs of 16 keys: within one page
  static constexpr int kRows = 16;
  // Shared memory: stages, their barriers, what the warps hold, prefix.
  static constexpr int kBars = kWarps * kStages * kStage;
  static constexpr int kPieces = kBars + kWarps * kStages * 8;    // [warp][2]
  static constexpr int kPrefix = kPieces + kWarps * 2 * 32;
  static constexpr int kBytes = kPrefix + (kSlice + 1) * 8;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

// Column n of an 8-key score tile is key n / 2, or 4 + (n / 2 ^ 1) for odd n:
// the rows that neighbouring lanes read then lie in different banks (D = 64).
__device__ __forceinline__ int key_of_column(int n) { return n & 1 ? 4 + ((n >> 1) ^ 1) : n >> 1; }

// A warp's part of an item that began in an earlier share (piece 0) or goes on
// into the next one (piece 1).
struct Piece {
  int state;  // 0: none, 1: the item ends here, 2: it goes on
  int first, rows, row0, kv_head;
  long long end;  // of the item's tiles
};
static_assert(sizeof(Piece) == 32, "piece");

struct Cursor {  // a tile of the CTA's share: its item and place
  long long tile;          // position among all tiles
  long long item_begin, item_end;
  int user, kv_head, row0;
  Span span;               // of the user
};

// Four channels of a row's result, and its log-sum.
template <typename T>
__device__ __forceinline__ void write_row(const cxs_cache_attend_call& a, const Shape& z, int first,
                                          int kv_head, int row, int dim, int d, float4 sum, float m,
                                          float l) {
  const bool some = !(l == 0.f);
  const float inv = some ? 1.f / l : 0.f;
  const long long head =
      (long long)(first + row / z.group) * a.heads + kv_head * z.group + row % z.group;
  alignas(8) T y[4] = {from_float<T>(some ? sum.x * inv : 0.f), from_float<T>(some ? sum.y * inv : 0.f),
                       from_float<T>(some ? sum.z * inv : 0.f), from_float<T>(some ? sum.w * inv : 0.f)};
  *reinterpret_cast<uint2*>((T*)a.out + head * dim + d) = *reinterpret_cast<const uint2*>(y);
  if (a.lse && d == 0) a.lse[head] = some ? (m + log2f(l)) * kLn2 : -kInf;
}

// The join of partial results for four channels of a row.
struct Join {
  float m = -kInf, l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  // Parts k0, k0 + step, ... (four, below `parts`), all loads in flight at once.
  template <int D, int ROWS, typename F>
  __device__ __forceinline__ void add4(F part, int k0, int step, int parts, int r, int d) {
    float2 stat[4];
    float4 v[4];
    float top = m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* from = part(min(k0 + j * step, parts - 1));
      stat[j] = *reinterpret_cast<const float2*>(from + ROWS * D + 2 * r);
      v[j] = *reinterpret_cast<const float4*>(from + r * D + d);
      if (k0 + j * step >= parts) stat[j] = make_float2(-kInf, 0.f);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, stat[j].x);
    const float base = top == -kInf ? 0.f : top, old = ex2(m - base);
    m = top;
    l *= old;
    sum.x *= old, sum.y *= old, sum.z *= old, sum.w *= old;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (k0 + j * step >= parts) break;
      add(stat[j], v[j], base);
    }
  }
  __device__ __forceinline__ void add(float2 stat, float4 v, float base) {
    const float f = ex2(stat.x - base);
    l = fmaf(stat.y, f, l);
    sum.x = fmaf(v.x, f, sum.x);
    sum.y = fmaf(v.y, f, sum.y);
    sum.z = fmaf(v.z, f, sum.z);
    sum.w = fmaf(v.w, f, sum.w);
  }
};

template <int D>
__device__ __forceinline__ int item_tiles(const Span& s) {
  constexpr int T = Decode<D>::kTile;
  if (s.count == 0) return 0;
  const int n = (s.length + T - 1) / T - s.begin / T;
  // An item without keys still writes its rows. One more: finding an item,
  // loading its queries and writing its rows take about as long as a tile.
  return (n > 0 ? n : 1) + 1;
}

// HIDES: rows of a user may see different keys, and V may have NaN codes. Its
// registers are short at D = 128: 5 tokens of 8 users of 8K, 93.6 us against 91.1
// without it, 3 tokens at D = 64 28.8 against 28.0.
template <int FORMAT, typename T, int D, bool HIDES>
__global__ void __launch_bounds__(Decode<D>::kThreads, 1)
    decode_kernel(const cxs_cache_attend_call a, const Shape z) {
  using K = Decode<D>;
  const cxs_cache_call& c = a.cache;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int g = lane / 4, t = lane % 4;
  long long* prefix = reinterpret_cast<long long*>(smem + K::kPrefix);

  // Tiles before each user (items of a user have equal tile counts).
  __shared__ long long warp_sum[K::kWarps];
  {
    long long base = 0;
    for (int b0 = 0; b0 < z.users; b0 += K::kThreads) {
      const int b = b0 + threadIdx.x;
      long long n = 0;
      if (b < z.users) {
        int bad = 0;
        const Span s = user_span(a, z, b, &bad);
        n = (long long)item_tiles<D>(s) * c.kv_heads *
            (((long long)s.count * z.group + K::kRows - 1) / K::kRows);
        if (bad && blockIdx.x == 0) report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
      }
      long long sum = n;
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (lane == 31) warp_sum[warp] = sum;
      __syncthreads();
      long long before = base, all = base;
      for (int w = 0; w < K::kWarps; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
      }
      if (b < z.users) prefix[b] = before + sum - n;
      base = all;
      __syncthreads();
    }
    if (threadIdx.x == 0) prefix[z.users] = base;
  }
  __syncthreads();
  const long long total = prefix[z.users];
  // Neighbouring shares lie in one CTA, at least 3, for the join at its end.
  // (Few tiles: shares of one, 3 a CTA, take 9.2 us for 100 keys and 12.9 for 4K,
  // shares of two, 6 a CTA, 12.8 and 14.5; with more tiles than that, shares of
  // two: 8 users of 8K, 17.5 us against 20.4.)
  const Shares shares(total, z);
  const int per = min(max((shares.count + z.grid - 1) / z.grid, 3), K::kWarps);
  const int worker = (int)blockIdx.x * per + warp;
  const bool busy = warp < per && worker < shares.count;
  Partial* const partials = reinterpret_cast<Partial*>(a.workspace);
  Partial& mine = partials[blockIdx.x];
  constexpr int kSize = K::kRows * (D + 2);
  // Partial results of the CTAs, then of the warps, two each.
  float* const cta_parts =
      reinterpret_cast<float*>(partials + z.grid) + (long long)blockIdx.x * 2 * kSize;
  float* const warp_parts = reinterpret_cast<float*>(partials + z.grid) +
                            ((long long)z.grid + (long long)blockIdx.x * K::kWarps) * 2 * kSize;
  Piece* const pieces = reinterpret_cast<Piece*>(smem + K::kPieces);  // [warp][2]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) mine.parts = 0;
  __shared__ int nan_seen[K::kWarps];  // V had NaN codes where keys are hidden
  if (lane == 0) nan_seen[warp] = 0;
  if (lane < 2) pieces[2 * warp + lane].state = 0;
  __syncwarp();
  const long long lo = busy ? shares.begin(worker) : 0, hi = busy ? shares.begin(worker + 1) : 0;
  float* const scratch = warp_parts + (long long)warp * 2 * kSize;

  // The item of a tile, found from the last one.
  auto seek = [&](Cursor& p) {
    if (p.tile < p.item_end) return;
    if (p.tile >= hi) return;
    int u = p.user;
    if (p.tile >= prefix[u + 1]) {  // the next user with tiles
      int l = u + 1, h = z.users - 1;
      while (l < h) {
        const int m = (l + h) / 2;
        if (prefix[m + 1] > p.tile) h = m; else l = m + 1;
      }
      u = l;
    }
    int bad = 0;
    const Span s = user_span(a, z, u, &bad);
    const int n = item_tiles<D>(s);
    const long long item = divide(p.tile - prefix[u], n);
    p.user = u;
    p.span = s;
    p.item_begin = prefix[u] + item * n;
    p.item_end = p.item_begin + n;
    const int rows16 = (int)divide(item, c.kv_heads);
    p.kv_head = (int)(item - (long long)rows16 * c.kv_heads);
    p.row0 = rows16 * K::kRows;
  };

  uint8_t* const stages = smem + warp * K::kStages * K::kStage;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + K::kBars) + warp * K::kStages;
  if (lane < K::kStages) cxs::mbar_init(bars + lane, 1);
  cxs::fence_mbar_init();
  __syncwarp();
  // A tile's copies: piece_keys keys of one page each, lane 2 i its K, lane
  // 2 i + 1 its V.
  const int piece_bits = min(__ffs(c.page_size), __ffs(K::kTile)) - 1;
  const int page_bits = __ffs(c.page_size) - 1;
  const int copies = 2 * (K::kTile >> piece_bits), piece_bytes = D << piece_bits;
  // A copy's page, looked up one tile before the copy is issued; -2 where it
  // holds no token that a row sees.
  auto look_up = [&](Cursor& p) -> int {
    if (p.tile >= hi) return -2;
    seek(p);
    if (p.tile == p.item_begin && ++p.tile >= hi) return -2;  // (an item's first is no tile)
    const int at = (p.span.begin / K::kTile + (int)(p.tile - p.item_begin) - 1) * K::kTile +
                   (lane / 2 << piece_bits);
    if (lane >= copies || at >= p.span.length || at + (1 << piece_bits) <= p.span.begin) return -2;
    return __ldg(c.table + p.user * c.table_stride + (at >> page_bits));
  };
  // Copies of the tile at `p` into a stage. Returns this lane's scale (of its
  // copy's page and part) and which copies there are.
  auto fetch = [&](const Cursor& p, int stage, int id, unsigned* there) -> float {
    if (p.tile >= hi) return 1.f;
    const int key0 = (p.span.begin / K::kTile + (int)(p.tile - p.item_begin) - 1) * K::kTile;
    const bool mine = id >= 0 && id < c.pages;
    if (!mine && id != -2) report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
    *there = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) cxs::mbar_expect_tx(bars + stage, __popc(*there) * piece_bytes);
    __syncwarp();
    if (!mine) return 1.f;
    const long long cell = ((long long)id * c.kv_heads + p.kv_head) * 2 + (lane & 1);
    cxs::bulk_g2s(stages + stage * K::kStage + (lane & 1) * K::kPart + lane / 2 * piece_bytes,
                  (const uint8_t*)c.codes + (cell * c.page_size + (key0 & (c.page_size - 1))) * D,
                  piece_bytes, bars + stage);
    return __ldg(c.scales + cell);
  };

  if (busy) {
    Cursor item{lo, -1, -1, 0, 0, 0, {}};
    seek(item);
    Cursor ahead = item;
    long long here = lo;          // the next tile
    int taken = 0;                // tiles taken so far: stage taken % 2
    unsigned next_there = 0;      // of the tile that is coming
    int ahead_id = look_up(ahead);
    float next_scale = fetch(ahead, 0, ahead_id, &next_there);
    ++ahead.tile;
    ahead_id = look_up(ahead);
    // Where this lane reads: its 16 channels of a key, its D / 8 of V.
    const int k_at = key_of_column(g) * D + 16 * t;
    const int v_at0 = t * D + D / 8 * g, v_at1 = (4 + (t ^ 1)) * D + D / 8 * g;
    bool lost = false;  // a copy did not come

    float o[D / 8][4], m0, m1, l0, l1;  // rows g and g + 8
    while (true) {
      const long long item_hi = item.item_end < hi ? item.item_end : hi;
      const Span& s = item.span;
      const int rows = s.count * z.group;
      const int first_tile = s.begin / K::kTile;
      // This lane's rows g and g + 8: what they see, and their queries as
      // operands (its 16 channels of each 64 are four steps' operand elements),
      // scaled by a power of two (and the scale's sign).
      uint32_t q[D / 16][4];
      float back0, back1;
      int2 see0 = make_int2(0, 0), see1 = make_int2(0, 0);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = item.row0 + g + 8 * half;
        const bool live = row < rows;
        const T* from = (const T*)a.query;
        if (live) {
          const int token = row / z.group;
          from += (long long)(s.first + token) * a.q_token_stride +
                  (long long)(item.kv_head * z.group + row - token * z.group) * a.q_head_stride;
          const int2 see = row_range(a, s, token);
          if (half) see1 = see; else see0 = see;
        }
        alignas(16) T in[D / 4];
        const bool wide = ((uintptr_t)from & 15) == 0;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {  // 8 of the lane's channels
          const T* const part = from + 64 * (j / 2) + 16 * t + 8 * (j % 2);
          if (wide) {
            *reinterpret_cast<uint4*>(in + 8 * j) = *reinterpret_cast<const uint4*>(part);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) in[8 * j + e] = part[e];
          }
        }
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < D / 4; ++e) {
          const float x = fabsf(to_float(in[e]));
          if (x < kInf) top = fmaxf(top, x);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
        if (e < -100) e = -100;
        if (top == 0.f) e = 14;
        float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        if (a.scale < 0.f) up = -up;
        if (a.scale == 0.f) up = 0.f;  // every score is 0
        const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
        if (half) back1 = down; else back0 = down;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float lo_half = live ? to_float(in[2 * i]) * up : 0.f;
          const float hi_half = live ? to_float(in[2 * i + 1]) * up : 0.f;
          q[i / 2][half + 2 * (i % 2)] = pack_half2(lo_half, hi_half);
        }
      }
      const float unit = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      m0 = m1 = -kInf;
      l0 = l1 = 0.f;
      // All rows of the tile see the keys [all.x, all.y).
      int2 all = make_int2(max(see0.x, see1.x), min(see0.y, see1.y));
      if (item.row0 + g >= rows) all = make_int2(0, s.length);
      else if (item.row0 + g + 8 >= rows) all = see0;
      all.x = __reduce_max_sync(0xffffffffu, all.x);
      all.y = __reduce_min_sync(0xffffffffu, all.y);

      if (here == item.item_begin) ++here;
#pragma unroll 1
      for (; here < item_hi; ++here) {
        // The stage taken in the previous round is free: the next tile's copies.
        __syncwarp();
        const float scale = next_scale;
        const unsigned there = next_there;
        next_scale = fetch(ahead, (taken + 1) % 2, ahead_id, &next_there);
        ++ahead.tile;
        ahead_id = look_up(ahead);
        if (!cxs::mbar_try_wait(bars + taken % 2, taken / 2 & 1)) {
          const long long since = clock64();
          while (!cxs::mbar_try_wait(bars + taken % 2, taken / 2 & 1) && !lost)
            lost = clock64() - since > kSpinLimit;
          if (lost) report(c.error, CXS_DEVICE_ERR_COPY_TIMEOUT);
        }
        uint8_t* const ks = stages + taken % 2 * K::kStage;
        ++taken;
        uint8_t* const vs = ks + K::kPart;
        const int key0 = (first_tile + (int)(here - item.item_begin) - 1) * K::kTile;
        const bool partial = there != (1u << copies) - 1 || key0 + K::kTile > s.length;
        const bool edge = key0 < all.x || key0 + K::kTile > all.y;  // hidden from some row
        if (partial || (HIDES && edge)) {
          // V of keys without a token becomes 0: a probability of 0 times
          // whatever the bytes hold could be NaN. So do NaN codes where some row
          // does not see their keys.
          uint32_t found = 0;
#pragma unroll 1
          for (int r = lane; r < K::kTile; r += 32) {
            const bool gone = key0 + r >= s.length || !(there >> (r >> piece_bits) * 2 & 1);
            if (!HIDES && !gone) continue;
#pragma unroll 1
            for (int i = 0; i < D; i += 16) {
              uint4* const at = reinterpret_cast<uint4*>(vs + r * D + i);
              *at = gone ? make_uint4(0, 0, 0, 0) : without_nan(*at, &found);
            }
          }
          if (HIDES && found) *(volatile int*)&nan_seen[warp] = 1;
          cxs::fence_proxy_async_shared();
          __syncwarp();
        }

        float x[K::kTile / 8][4];
#pragma unroll
        for (int n = 0; n < K::kTile / 8; ++n) {
          x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
          for (int j = 0; j < D / 64; ++j) {
            const uint4 w = *reinterpret_cast<const uint4*>(ks + 8 * n * D + k_at + 64 * j);
            mma16816(x[n], q[4 * j + 0], half2_of<FORMAT>(w.x, 0), half2_of<FORMAT>(w.x, 1));
            mma16816(x[n], q[4 * j + 1], half2_of<FORMAT>(w.y, 0), half2_of<FORMAT>(w.y, 1));
            mma16816(x[n], q[4 * j + 2], half2_of<FORMAT>(w.z, 0), half2_of<FORMAT>(w.z, 1));
            mma16816(x[n], q[4 * j + 3], half2_of<FORMAT>(w.w, 0), half2_of<FORMAT>(w.w, 1));
          }
        }
        // -infinity where a row does not see the key.
        if (partial || edge) {
#pragma unroll
          for (int n = 0; n < K::kTile / 8; ++n) {
            const int ka = key0 + 8 * n + t, kb = key0 + 8 * n + 4 + (t ^ 1);
            const bool gone = !(there >> (8 * n >> piece_bits) * 2 & 1);
            if (gone || ka < see0.x || ka >= see0.y) x[n][0] = -kInf;
            if (gone || kb < see0.x || kb >= see0.y) x[n][1] = -kInf;
            if (gone || ka < see1.x || ka >= see1.y) x[n][2] = -kInf;
            if (gone || kb < see1.x || kb >= see1.y) x[n][3] = -kInf;
          }
        }
        // A score is x f + lift: f = scale log2(e) s_k (and the row's power of
        // two), lift = log2 s_v, per = 1 / s_v.
        float f0[K::kGroups], f1[K::kGroups], lift[K::kGroups], per[K::kGroups];
        float t0 = -kInf, t1 = -kInf;
        // (Each copy's lane works out its part of them.)
        const float my_scale = usable_scale(scale), my_f = my_scale * unit;
        const float my_lift = __log2f(my_scale), my_per = ex2(-my_lift);
#pragma unroll
        for (int u = 0; u < K::kGroups; ++u) {
          const int from = (16 * u >> piece_bits) * 2;
          const float sk = __shfl_sync(0xffffffffu, my_f, from);
          lift[u] = __shfl_sync(0xffffffffu, my_lift, from + 1);
          per[u] = __shfl_sync(0xffffffffu, my_per, from + 1);
          // Never 0, which times a hidden score would be NaN; NaN stays NaN.
          f0[u] = sk * back0 < 1.2e-38f ? 1.2e-38f : sk * back0;
          f1[u] = sk * back1 < 1.2e-38f ? 1.2e-38f : sk * back1;
          const float(&ya)[4] = x[2 * u];
          const float(&yb)[4] = x[2 * u + 1];
          t0 = fmaxf(t0, fmaf(fmaxf(fmaxf(ya[0], ya[1]), fmaxf(yb[0], yb[1])), f0[u], lift[u]));
          t1 = fmaxf(t1, fmaf(fmaxf(fmaxf(ya[2], ya[3]), fmaxf(yb[2], yb[3])), f1[u], lift[u]));
        }
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
        const bool g0 = t0 > m0 + kLag, g1 = t1 > m1 + kLag;
        if (__any_sync(0xffffffffu, g0 || g1)) {
          const float c0 = !g0 ? 1.f : m0 == -kInf ? 0.f : ex2(m0 - t0);
          const float c1 = !g1 ? 1.f : m1 == -kInf ? 0.f : ex2(m1 - t1);
          if (g0) m0 = t0;
          if (g1) m1 = t1;
          l0 *= c0;
          l1 *= c1;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][0] *= c0;
            o[i][1] *= c0;
            o[i][2] *= c1;
            o[i][3] *= c1;
          }
        }
        const float b0 = m0 == -kInf ? 0.f : m0 - kHead, b1 = m1 == -kInf ? 0.f : m1 - kHead;
#pragma unroll
        for (int u = 0; u < K::kGroups; ++u) {
          float(&ya)[4] = x[2 * u];
          float(&yb)[4] = x[2 * u + 1];
          const float s0 = lift[u] - b0, s1 = lift[u] - b1;
          const float2 pa0 = exp2_pair(ya[0], ya[1], f0[u], s0), pb0 = exp2_pair(yb[0], yb[1], f0[u], s0);
          const float2 pa1 = exp2_pair(ya[2], ya[3], f1[u], s1), pb1 = exp2_pair(yb[2], yb[3], f1[u], s1);
          const float2 sum0 = __fadd2_rn(pa0, pb0), sum1 = __fadd2_rn(pa1, pb1);
          l0 = fmaf(sum0.x + sum0.y, per[u], l0);
          l1 = fmaf(sum1.x + sum1.y, per[u], l1);
          const uint32_t p[4] = {pack_half2(pa0.x, pa0.y), pack_half2(pa1.x, pa1.y),
                                 pack_half2(pb0.x, pb0.y), pack_half2(pb1.x, pb1.y)};
          // Keys of this lane's four operand rows; D / 8 of their channels each.
          constexpr int kWords = D / 32;
          uint32_t w[4][kWords];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* from = vs + (16 * u + 8 * (i / 2)) * D + (i % 2 ? v_at1 : v_at0);
            if (D == 64) {
              const uint2 v = *reinterpret_cast<const uint2*>(from);
              w[i][0] = v.x;
              w[i][1] = v.y;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(from);
              w[i][0] = v.x;
              w[i][1] = v.y;
              w[i][kWords - 2] = v.z;
              w[i][kWords - 1] = v.w;
            }
          }
#pragma unroll
          for (int n = 0; n < kWords; ++n) {
            const uint32_t a01 = __byte_perm(w[0][n], w[1][n], 0x5140);
            const uint32_t a23 = __byte_perm(w[0][n], w[1][n], 0x7362);
            const uint32_t b01 = __byte_perm(w[2][n], w[3][n], 0x5140);
            const uint32_t b23 = __byte_perm(w[2][n], w[3][n], 0x7362);
            mma16816(o[4 * n + 0], p, half2_of<FORMAT>(a01, 0), half2_of<FORMAT>(b01, 0));
            mma16816(o[4 * n + 1], p, half2_of<FORMAT>(a01, 1), half2_of<FORMAT>(b01, 1));
            mma16816(o[4 * n + 2], p, half2_of<FORMAT>(a23, 0), half2_of<FORMAT>(b23, 0));
            mma16816(o[4 * n + 3], p, half2_of<FORMAT>(a23, 1), half2_of<FORMAT>(b23, 1));
          }
        }
      }

      // The item's result, or this share's part of it: slot 0 for an item that
      // began in an earlier share, slot 1 for one that goes on into the next.
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      m0 -= kHead;  // what O and l are relative to
      m1 -= kHead;
      const bool begins = item.tile == item.item_begin, whole = begins && item_hi == item.item_end;
      float* const part = scratch + (begins ? K::kRows * (D + 2) : 0);
      // Accumulator i, columns 2t, 2t + 1: channels (D / 8) column + i.
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = g + 4 * (e & 2), row = item.row0 + r;
        if (row >= rows) continue;
        const float m = e < 2 ? m0 : m1, l = e < 2 ? l0 : l1;
        const int d = D / 8 * (2 * t + (e & 1));
#pragma unroll
        for (int i = 0; i < D / 8; i += 4) {
          const float4 sum = make_float4(o[i][e], o[i + 1][e], o[i + 2][e], o[i + 3][e]);
          if (whole)
            write_row<T>(a, z, s.first, item.kv_head, row, D, d + i, sum, m, l);
          else
            *reinterpret_cast<float4*>(part + r * D + d + i) = sum;
        }
        if (!whole && d == 0)
          *reinterpret_cast<float2*>(part + K::kRows * D + 2 * r) = make_float2(m, l);
      }
      if (!whole && lane == 0)
        pieces[2 * warp + begins] =
            Piece{item_hi == item.item_end ? 1 : 2, s.first, rows, item.row0, item.kv_head, item.item_end};
      item.tile = item_hi;
      if (item_hi >= hi) break;
      seek(item);
    }
    if (lost) {  // copies still on their way end before the CTA does
      const long long since = clock64();
      for (int use = max(taken - 2, 0); use < taken; ++use)
        while (!cxs::mbar_try_wait(bars + use % 2, use / 2 & 1) && clock64() - since < kSpinLimit) {
        }
    }
    __syncwarp();
    if (HIDES && *(volatile int*)&nan_seen[warp]) {
      // The warp's items once more, for rows that see NaN values (here, where
      // nothing else is held: at each item's end it cost 5 %).
      item = Cursor{lo, -1, -1, 0, 0, 0, {}};
#pragma unroll 1
      while (item.tile < hi) {
        seek(item);
        const Span& s = item.span;
        const long long item_hi = item.item_end < hi ? item.item_end : hi;
        const bool begins = item.tile == item.item_begin, whole = begins && item_hi == item.item_end;
        const int rows = s.count * z.group, first_tile = s.begin / K::kTile;
        const int tile0 = first_tile + (int)(item.tile - item.item_begin) - !begins;
        const int tile1 = first_tile + (int)(item_hi - item.item_begin) - 1;
        const int2 all = seen_by_all(a, z, s, item.row0, min(rows, item.row0 + K::kRows) - 1);
        // (Tiles that every row sees whole went as they are.)
        const int2 skip = make_int2((all.x + K::kTile - 1) / K::kTile * K::kTile,
                                    all.y / K::kTile * K::kTile);
        const long long half_page = (long long)c.page_size * D;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {  // what this lane wrote of a row
          const int r = g + 4 * (e & 2), row = item.row0 + r;
          if (row >= rows) continue;
          const int2 see = row_range(a, s, row / z.group);
          const long long head = (long long)(s.first + row / z.group) * a.heads +
                                 item.kv_head * z.group + row % z.group;
          mark_nans<T, D>((const uint8_t*)c.codes + (2 * item.kv_head + 1) * half_page,
                          2 * c.kv_heads * half_page, c.pages, c.table + item.user * c.table_stride,
                          c.page_size, max(see.x, tile0 * K::kTile), min(see.y, tile1 * K::kTile),
                          skip, (T*)a.out + head * D,
                          whole ? nullptr
                                : scratch + (begins ? K::kRows * (D + 2) : 0) + r * D,
                          D / 8 * (2 * t + (e & 1)), D / 8);
        }
        item.tile = item_hi;
      }
    }
  }
  __syncthreads();

  // Each item that the CTA holds in parts, in the order of the shares: one that
  // comes in with the first warp, then those that begin in a warp and go on.
  for (int start = -1; start < per; ++start) {
    const bool before = start < 0;  // it began in an earlier CTA
    const int first = before ? 0 : start;
    const Piece piece = pieces[2 * first + !before];
    if (!piece.state) continue;
    bool on = piece.state == 2;
    int last = first;
    while (on && last + 1 < per) on = pieces[2 * ++last].state == 2;
    const int parts = last - first + 1;
    float* const to = cta_parts + (before ? 0 : kSize);
    for (int i = threadIdx.x; i < K::kRows * D / 4; i += K::kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4, row = piece.row0 + r;
      if (row >= piece.rows) continue;
      Join join;
      for (int k0 = 0; k0 < parts; k0 += 4)
        join.add4<D, K::kRows>([&](int k) {
          return warp_parts + (2 * (first + k) + (k == 0 && !before)) * kSize;
        }, k0, 1, parts, r, d);
      if (!before && !on) {
        write_row<T>(a, z, piece.first, piece.kv_head, row, D, d, join.sum, join.m, join.l);
      } else {
        *reinterpret_cast<float4*>(to + r * D + d) = join.sum;
        if (d == 0)
          *reinterpret_cast<float2*>(to + K::kRows * D + 2 * r) = make_float2(join.m, join.l);
      }
    }
    if (!before && on && threadIdx.x == 0) {
      mine.first = piece.first;
      mine.rows = piece.rows;
      mine.row0 = piece.row0;
      mine.kv_head = piece.kv_head;
      mine.parts = shares.of(piece.end - 1) / per - (int)blockIdx.x + 1;
    }
  }
  clear_rows<T, D>(a, z, blockIdx.x, z.grid, threadIdx.x, K::kThreads);
}

// Joins the partial results of the item (of ROWS rows) that starts in CTA
// blockIdx.x and goes on into later ones: 16 rows, a thread for four channels
// of a row and every GROUPS-th CTA's part. Latency-bound: in each of the groups
// four parts' loads are in flight at a time.
template <typename T, int D, int ROWS, int GROUPS>
__global__ void __launch_bounds__(GROUPS * 4 * D)
    combine_kernel(const cxs_cache_attend_call a, const Shape z) {
  constexpr int kSize = ROWS * (D + 2), kLanes = 4 * D;  // threads of a group
  __shared__ float4 sums[GROUPS > 1 ? GROUPS * kLanes : 1];
  __shared__ float2 stats[GROUPS > 1 ? GROUPS * 16 : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Partial* partials = reinterpret_cast<const Partial*>(a.workspace);
  const float* const own =
      reinterpret_cast<const float*>(partials + z.grid) + (long long)blockIdx.x * 2 * kSize;
  const Partial item = partials[blockIdx.x];
  if (item.parts == 0 || item.row0 + 16 * (int)blockIdx.y >= item.rows) return;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int in_block = lane / (D / 4), r = 16 * blockIdx.y + in_block, d = lane % (D / 4) * 4;
  const int row = item.row0 + r;
  Join join;
  if (row < item.rows)  // (the parts hold nothing of other rows)
    for (int k0 = group; k0 < item.parts; k0 += 4 * GROUPS)
      join.add4<D, ROWS>([&](int k) { return own + (k == 0 ? kSize : 2 * k * kSize); }, k0, GROUPS,
                         item.parts, r, d);
  if (GROUPS > 1) {
    sums[threadIdx.x] = join.sum;
    if (d == 0) stats[group * 16 + in_block] = make_float2(join.m, join.l);
    __syncthreads();
    if (group > 0) return;
    float m = -kInf;
    for (int i = 0; i < GROUPS; ++i) m = fmaxf(m, stats[i * 16 + in_block].x);
    join = Join();
    join.m = m;
    for (int i = 0; i < GROUPS; ++i)
      join.add(stats[i * 16 + in_block], sums[i * kLanes + lane], m == -kInf ? 0.f : m);
  }
  if (row < item.rows)
    write_row<T>(a, z, item.first, item.kv_head, row, D, d, join.sum, join.m, join.l);
}

// ------------------------------------------------------------------ host ---

template <int FORMAT, typename T, int D, bool HIDES>
int launch_decode_as(const cxs_cache_attend_call& a, const Shape& z, cudaStream_t stream) {
  using K = Decode<D>;
  static cxs_host::OncePerDevice ready;
  const int status = ready.run([] {
    CXS_CUDA(cudaFuncSetAttribute(decode_kernel<FORMAT, T, D, HIDES>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, K::kBytes));
    return (int)CXS_OK;
  });
  if (status != CXS_OK) return status;
  decode_kernel<FORMAT, T, D, HIDES><<<z.grid, K::kThreads, K::kBytes, stream>>>(a, z);
  CXS_LAUNCH_CHECK("cache attend");
  return CXS_OK;
}

// Only e4m3 has NaN codes, and one token without a window hides no key.
template <int FORMAT, typename T, int D>
int launch_decode(const cxs_cache_attend_call& a, const Shape& z, cudaStream_t stream) {
  if (FORMAT == CXS_FORMAT_E4M3 && (a.window > 0 || (a.causal && a.cache.max_tokens > 1)))
    return launch_decode_as<FORMAT, T, D, FORMAT == CXS_FORMAT_E4M3>(a, z, stream);
  return launch_decode_as<FORMAT, T, D, false>(a, z, stream);
}

template <typename T, int D>
int launch_combine(const cxs_cache_attend_call& a, const Shape& z, bool few, bool spread,
                   cudaStream_t stream) {
  // Its CTAs may start while the last CTAs before finish; they wait for them
  // on the device.
  cudaLaunchConfig_t config = {};
  constexpr int kGroups = 256 / D;  // for few rows, or many parts: 1024 threads
  config.gridDim = dim3(z.grid, few ? 1 : kTileRows / 16);
  config.blockDim = dim3(few || spread ? kGroups * 4 * D : 4 * D);
  config.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  if (few)
    CXS_CUDA(cudaLaunchKernelEx(&config, combine_kernel<T, D, 16, kGroups>, a, z));
  else if (spread)
    CXS_CUDA(cudaLaunchKernelEx(&config, combine_kernel<T, D, kTileRows, kGroups>, a, z));
  else
    CXS_CUDA(cudaLaunchKernelEx(&config, combine_kernel<T, D, kTileRows, 1>, a, z));
  CXS_LAUNCH_CHECK("cache attend join");
  return CXS_OK;
}

}  // namespace

int cxs::cache8::check_attend(const cxs_cache_attend_call* a, const char* what) {
  if (!a) return set_error(CXS_ERR_INVALID, "%s: null call", what);
  const int status = cxs_host::check_cache(&a->cache, what);
  if (status != CXS_OK) return status;
  if (a->cache.type == CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "%s: queries must be bf16 or fp16", what);
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return set_error(CXS_ERR_INVALID, "%s: heads must be a multiple of kv_heads", what);
  if (a->window < 0) return set_error(CXS_ERR_INVALID, "%s: negative window", what);
  if ((long long)a->cache.max_tokens * a->heads > 0x40000000ll)
    return set_error(CXS_ERR_CAPACITY, "%s: more than 2^30 rows of one user", what);
  return CXS_OK;
}

int cxs::cache8::check_attend_pointers(const cxs_cache_attend_call* a, long long workspace,
                                       const char* what) {
  const int status = cxs_host::check_cache_pointers(&a->cache, what);
  if (status != CXS_OK) return status;
  if (!a->query || !a->out) return set_error(CXS_ERR_INVALID, "%s: null query or out", what);
  if ((uintptr_t)a->out % 16) return set_error(CXS_ERR_INVALID, "%s: out must be 16-byte aligned", what);
  if (!a->workspace || (uintptr_t)a->workspace % 16 || a->workspace_bytes < workspace)
    return set_error(CXS_ERR_INVALID, "%s: workspace missing, unaligned or too small", what);
  return CXS_OK;
}

// SMs of the current device (looked up once).
int cxs::cache8::sm_count(int* sms) {
  static int known;
  static cxs_host::OncePerDevice looked;
  const int status = looked.run([] {
    int device = 0, n = 0;
    CXS_CUDA(cudaGetDevice(&device));
    CXS_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
    __atomic_store_n(&known, n, __ATOMIC_RELAXED);
    return (int)CXS_OK;
  });
  *sms = __atomic_load_n(&known, __ATOMIC_RELAXED);
  return status;
}

// Most rows of a user and KV head for which the mma.sync kernel runs: it takes
// 16 rows at a time and reads the keys again for the next 16, the tcgen05
// kernel takes up to 256 at about the same cost. Measured (us, mma.sync /
// tcgen05, e4m3; 1 user of 16K tokens, 8 of 8K, 64 of 4K):
//   D = 64, 2 KV heads    64 rows   23 / 41    32 / 33    65 / 80
//                        128 rows   28 / 42    43 / 35   110 / 82
//   D = 128, 8 KV heads   32 rows   47 / 43    89 / 97   260 / 334
//                         64 rows   60 / 45   142 / 100  480 / 340
bool cxs::cache8::few_rows(const cxs_cache_attend_call& a) {
  return (long long)a.cache.max_tokens * (a.heads / a.cache.kv_heads) <= (a.cache.dim == 64 ? 64 : 32);
}

long long cxs::cache8::partial_bytes(const cxs_cache_attend_call& a, bool few) {
  // Two partial results for each CTA and, of few rows, each warp.
  const long long slots = 2 * kMostCtas * (few ? 1 + kDecodeWarps : 1);
  const long long rows = few ? 16 : kTileRows;
  return kMostCtas * sizeof(Partial) +
         slots * rows * (a.cache.dim + 2) * (long long)sizeof(float);
}

int cxs::cache8::launch_join(const cxs_cache_attend_call& a, const Shape& z, bool few, bool spread,
                             cudaStream_t s) {
  if (a.cache.type == CXS_TYPE_BF16)
    return a.cache.dim == 64 ? launch_combine<__nv_bfloat16, 64>(a, z, few, spread, s)
                             : launch_combine<__nv_bfloat16, 128>(a, z, few, spread, s);
  return a.cache.dim == 64 ? launch_combine<__half, 64>(a, z, few, spread, s)
                           : launch_combine<__half, 128>(a, z, few, spread, s);
}

extern "C" int cxs_cache_attend_workspace(const cxs_cache_attend_call* call, int64_t* bytes) {
  const int status = check_attend(call, "cache attend");
  if (status != CXS_OK) return status;
  if (!bytes) return set_error(CXS_ERR_INVALID, "cache attend: null result");
  *bytes = partial_bytes(*call, few_rows(*call));
  return CXS_OK;
}

extern "C" int cxs_cache_attend(const cxs_cache_attend_call* call, void* stream) {
  int status = check_attend(call, "cache attend");
  if (status != CXS_OK) return status;
  const cxs_cache_call& c = call->cache;
  if (c.tokens == 0) return CXS_OK;
  if (c.users == 0) return set_error(CXS_ERR_INVALID, "cache attend: rows without users");
  const bool few = few_rows(*call);
  status = check_attend_pointers(call, partial_bytes(*call, few), "cache attend");
  if (status != CXS_OK) return status;
  int sms = 0;
  status = sm_count(&sms);
  if (status != CXS_OK) return status;
  const int grid = sms < kMostCtas ? sms : kMostCtas;
  cudaStream_t s = (cudaStream_t)stream;
  for (int user0 = 0; user0 < c.users; user0 += kSlice) {
    cxs_cache_attend_call a = *call;
    const int left = c.users - user0;
    const Shape z{call->heads / c.kv_heads, user0, left < kSlice ? left : kSlice, left <= kSlice,
                  grid, few ? grid * kDecodeWarps : grid, 2, few ? 3 * grid : 0};
    a.cache.table += user0 * c.table_stride;
    a.cache.lengths += user0;
    if (a.cache.offsets) a.cache.offsets += user0;
    if (few) {
      CXS_CACHE_FORMAT(c.format, F, {
        if (c.type == CXS_TYPE_BF16)
          status = c.dim == 64 ? launch_decode<F, __nv_bfloat16, 64>(a, z, s)
                               : launch_decode<F, __nv_bfloat16, 128>(a, z, s);
        else
          status = c.dim == 64 ? launch_decode<F, __half, 64>(a, z, s)
                               : launch_decode<F, __half, 128>(a, z, s);
      });
    } else {
      status = launch_tile(a, z, s);
    }
    if (status != CXS_OK) return status;
    status = launch_join(a, z, few, false, s);
    if (status != CXS_OK) return status;
  }
  return CXS_OK;
}
