// Attention over the dense 8-bit cache: few query rows a KV head, the joining
// of partial results, and the entry points.
#include <cuda_pipeline_primitives.h>

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

// ------------------------------------------------- few rows: one warp, 16 ---

// One CTA of 8 warps per SM. A warp takes a tile of keys at a time with all
// 16 rows: K and V codes go global -> shared with 16-byte asynchronous copies
// (zeros for tokens no row sees), two tiles ahead, then straight into
// mma.sync fragments: the order of channels within a dot product is free, so
// a lane's 16 bytes of a key are its fragments of four steps, and the order
// of keys within a tile is chosen so that the scores' accumulator is the
// probabilities' operand and a lane's V bytes of four keys pair up by
// byte permutes. No transposition passes through shared memory.
template <int D>
struct Decode {
  static constexpr int kWarps = 8, kThreads = 32 * kWarps;
  static constexpr int kTile = D == 64 ? 64 : 32;     // keys
  static constexpr int kPart = kTile * D;             // bytes of K or V
  static constexpr int kStages = 3;
  static constexpr int kStage = 2 * kPart;            // 8 KB; also holds a warp's O (16 x D fp32)
  static constexpr int kGroups = kTile / 16;          // runs of 16 keys: within one page
  static constexpr int kRows = 16;
  static_assert(kStage >= kRows * D * 4, "a stage holds a warp's O");
  // Shared memory: stages, then scales, page flags, row statistics, prefix.
  static constexpr int kScales = kWarps * kStages * kStage;
  static constexpr int kBad = kScales + kWarps * kStages * 2 * kGroups * 4;
  static constexpr int kStats = kBad + kWarps * kStages * 4;
  static constexpr int kPrefix = (kStats + kWarps * kRows * 2 * 4 + 15) / 16 * 16;
  static constexpr int kBytes = kPrefix + (kSlice + 1) * 8;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

// 16-byte chunk c of key row r in a tile. The permutation spreads the rows
// that one load instruction touches over all banks (rows 0..3 or 4..7 of a
// run of 8 with two neighbouring chunks for V, rows t and 4 + (t ^ 1) with
// four chunks for K).
template <int D>
__device__ __forceinline__ int chunk_at(int r, int c) {
  if (D == 64) return r * D + ((c ^ (r & 2)) << 4);
  return r * D + ((c ^ (2 * ((r ^ ((r >> 1) & 2)) & 3))) << 4);
}

// Column n of an 8-key score tile is key n / 2, or 4 + (n / 2 ^ 1) for odd n.
__device__ __forceinline__ int key_of_column(int n) { return n & 1 ? 4 + ((n >> 1) ^ 1) : n >> 1; }

struct Cursor {  // a tile of the CTA's share: its item and place
  long long tile;          // position among all tiles
  long long item_begin, item_end;
  int user, kv_head, row0;
  Span span;               // of the user
};

template <int D>
__device__ __forceinline__ int item_tiles(const Span& s) {
  constexpr int T = Decode<D>::kTile;
  if (s.count == 0) return 0;
  const int n = (s.length + T - 1) / T - s.begin / T;
  return n > 0 ? n : 1;  // an item without keys still writes its rows
}

template <int FORMAT, typename T, int D>
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
  const long long wanted = (total + z.min_tiles - 1) / z.min_tiles;
  const int ctas = wanted < z.grid ? (int)wanted : z.grid;
  Partial* partials = reinterpret_cast<Partial*>(a.workspace);
  Partial& mine = partials[blockIdx.x];
  clear_rows<T, D>(a, z, blockIdx.x, gridDim.x);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) mine.parts = 0;
  if ((int)blockIdx.x >= ctas) return;
  const long long lo = share(total, blockIdx.x, ctas), hi = share(total, blockIdx.x + 1, ctas);
  float* scratch = reinterpret_cast<float*>(partials + z.grid) +
                   (long long)blockIdx.x * 2 * K::kRows * (D + 2);

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
    const long long item = (p.tile - prefix[u]) / n;
    p.user = u;
    p.span = s;
    p.item_begin = prefix[u] + item * n;
    p.item_end = p.item_begin + n;
    p.kv_head = (int)(item % c.kv_heads);
    p.row0 = (int)(item / c.kv_heads) * K::kRows;
  };

  // Copies of the tile at `p` into a stage (commits a group in any case).
  uint8_t* const stages = smem + warp * K::kStages * K::kStage;
  float* const scales = reinterpret_cast<float*>(smem + K::kScales) + warp * K::kStages * 2 * K::kGroups;
  int* const bads = reinterpret_cast<int*>(smem + K::kBad) + warp * K::kStages;
  auto fetch = [&](const Cursor& p, int stage) {
    if (p.tile < hi) {
      const Span& s = p.span;
      const int tile = s.begin / K::kTile + (int)(p.tile - p.item_begin);
      const int key0 = tile * K::kTile;
      // Lane u < groups: the page of run u of 16 keys.
      int page = -1;
      if (lane < K::kGroups) {
        const int at = key0 + 16 * lane;
        if (at < s.length && at + 16 > s.begin) {
          page = c.table[p.user * c.table_stride + at / c.page_size];
          if (page < 0 || page >= c.pages) {
            page = -1;
            report(c.error, CXS_DEVICE_ERR_BAD_BLOCK);
          }
        }
      }
      const unsigned missing = __ballot_sync(0xffffffffu, lane < K::kGroups && page < 0);
      if (lane == 0) bads[stage] = missing;
      uint8_t* const dst = stages + stage * K::kStage;
      constexpr int kChunks = D / 16, kStep = 32 / kChunks;  // rows of one instruction
      const int row = lane / kChunks, chunk = lane % kChunks;
#pragma unroll
      for (int u = 0; u < K::kGroups; ++u) {
        const int pg = __shfl_sync(0xffffffffu, page, u);
        const long long cell = ((long long)(pg < 0 ? 0 : pg) * c.kv_heads + p.kv_head) * 2;
        const uint8_t* src = (const uint8_t*)c.codes + cell * c.page_size * D;
        const int slot0 = (key0 + 16 * u) & (c.page_size - 1);
#pragma unroll
        for (int j = 0; j < 16 / kStep; ++j) {
          const int r = j * kStep + row;                       // key of the run
          const int key = key0 + 16 * u + r;
          const bool live = pg >= 0 && key < s.length;
          const uint8_t* from = src + (live ? (slot0 + r) * D + chunk * 16 : 0);
          const int to = chunk_at<D>(16 * u + r, chunk);
          __pipeline_memcpy_async(dst + to, from, 16, live ? 0 : 16);
          __pipeline_memcpy_async(dst + K::kPart + to,
                                  from + (live ? c.page_size * D : 0), 16, live ? 0 : 16);
        }
        if (lane < 2)
          __pipeline_memcpy_async(scales + (stage * K::kGroups + u) * 2 + lane,
                                  c.scales + cell + lane, 4, pg < 0 ? 4 : 0);
      }
    }
    __pipeline_commit();
  };

  Cursor ahead{lo + warp, -1, -1, 0, 0, 0, {}}, item{lo, -1, -1, 0, 0, 0, {}};
  long long here = lo + warp;  // the next tile this warp takes
  int fill = 0;
#pragma unroll 1
  for (; fill < K::kStages - 1; ++fill) {
    seek(ahead);
    fetch(ahead, fill);
    ahead.tile += K::kWarps;
  }
  int use = 0;

  float o[D / 8][4], m0, m1, l0, l1;  // rows g and g + 8
  while (item.tile < hi) {
    seek(item);
    const long long item_hi = item.item_end < hi ? item.item_end : hi;
    const Span& s = item.span;
    const int rows = s.count * z.group;
    const int first_tile = s.begin / K::kTile;
    // The rows' queries as operands, scaled by a power of two per row.
    uint32_t q[D / 16][4];
    float back0, back1;
    int2 see0 = make_int2(0, 0), see1 = make_int2(0, 0);
    {
      float v[2][D / 4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = item.row0 + g + 8 * half;
        const bool live = r < rows;
        const T* from = (const T*)a.query;
        if (live) {
          from += (long long)(s.first + r / z.group) * a.q_token_stride +
                  (long long)(item.kv_head * z.group + r % z.group) * a.q_head_stride;
          const int2 see = row_range(a, s, r / z.group);
          if (half) see1 = see; else see0 = see;
        }
        float top = 0.f;
        const bool wide = ((uintptr_t)from & 15) == 0;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          alignas(16) T in[16];
          if (wide) {
            reinterpret_cast<uint4*>(in)[0] = reinterpret_cast<const uint4*>(from + 64 * j + 16 * t)[0];
            reinterpret_cast<uint4*>(in)[1] = reinterpret_cast<const uint4*>(from + 64 * j + 16 * t)[1];
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) in[e] = from[64 * j + 16 * t + e];
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = live ? to_float(in[e]) : 0.f;
            v[half][16 * j + e] = x;
            if (fabsf(x) < kInf) top = fmaxf(top, fabsf(x));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
        if (e < -100) e = -100;
        if (top == 0.f) e = 14;
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
        if (half) back1 = down; else back0 = down;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) v[half][i] *= up;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        q[i][0] = pack_half2(v[0][4 * i], v[0][4 * i + 1]);
        q[i][1] = pack_half2(v[1][4 * i], v[1][4 * i + 1]);
        q[i][2] = pack_half2(v[0][4 * i + 2], v[0][4 * i + 3]);
        q[i][3] = pack_half2(v[1][4 * i + 2], v[1][4 * i + 3]);
      }
    }
    const float unit = a.scale * kLog2e;
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

    int latest = -1;  // the stage this warp consumed last (free until the next fetch)
#pragma unroll 1
    for (; here < item_hi; here += K::kWarps) {
      // The stage consumed in the previous round is free: fetch ahead into it.
      __syncwarp();
      seek(ahead);
      fetch(ahead, fill);
      ahead.tile += K::kWarps;
      fill = fill + 1 == K::kStages ? 0 : fill + 1;
      __pipeline_wait_prior(K::kStages - 1);
      __syncwarp();
      const uint8_t* ks = stages + use * K::kStage;
      const uint8_t* vs = ks + K::kPart;
      const float* sc = scales + use * 2 * K::kGroups;
      const int missing = bads[use];
      latest = use;
      use = use + 1 == K::kStages ? 0 : use + 1;
      const int key0 = (first_tile + (int)(here - item.item_begin)) * K::kTile;

      float x[K::kTile / 8][4];
#pragma unroll
      for (int n = 0; n < K::kTile / 8; ++n) {
        x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
        const int r = 8 * n + key_of_column(g);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(ks + chunk_at<D>(r, t + 4 * j));
          mma16816(x[n], q[4 * j + 0], half2_of<FORMAT>(w.x, 0), half2_of<FORMAT>(w.x, 1));
          mma16816(x[n], q[4 * j + 1], half2_of<FORMAT>(w.y, 0), half2_of<FORMAT>(w.y, 1));
          mma16816(x[n], q[4 * j + 2], half2_of<FORMAT>(w.z, 0), half2_of<FORMAT>(w.z, 1));
          mma16816(x[n], q[4 * j + 3], half2_of<FORMAT>(w.w, 0), half2_of<FORMAT>(w.w, 1));
        }
      }
      // x = scale log2(e) s_k q.c + log2 s_v; -inf where a row does not see the key.
      float per[K::kGroups];  // 1 / s_v
#pragma unroll
      for (int u = 0; u < K::kGroups; ++u) {
        const float sk = usable_scale(sc[2 * u]) * unit, sv = usable_scale(sc[2 * u + 1]);
        const float lift = __log2f(sv);
        per[u] = __frcp_rn(sv);
        const float f0 = sk * back0, f1 = sk * back1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float(&y)[4] = x[2 * u + h];
          y[0] = fmaf(y[0], f0, lift);
          y[1] = fmaf(y[1], f0, lift);
          y[2] = fmaf(y[2], f1, lift);
          y[3] = fmaf(y[3], f1, lift);
        }
      }
      if (missing || key0 < all.x || key0 + K::kTile > all.y) {
#pragma unroll
        for (int n = 0; n < K::kTile / 8; ++n) {
          const int ka = key0 + 8 * n + t, kb = key0 + 8 * n + 4 + (t ^ 1);
          const bool gone = missing >> (n / 2) & 1;
          if (gone || ka < see0.x || ka >= see0.y) x[n][0] = -kInf;
          if (gone || kb < see0.x || kb >= see0.y) x[n][1] = -kInf;
          if (gone || ka < see1.x || ka >= see1.y) x[n][2] = -kInf;
          if (gone || kb < see1.x || kb >= see1.y) x[n][3] = -kInf;
        }
      }
      float t0 = -kInf, t1 = -kInf;
#pragma unroll
      for (int n = 0; n < K::kTile / 8; ++n) {
        t0 = fmaxf(t0, fmaxf(x[n][0], x[n][1]));
        t1 = fmaxf(t1, fmaxf(x[n][2], x[n][3]));
      }
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
      if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1)) {
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float c0 = m0 == -kInf ? 0.f : ex2(m0 - n0), c1 = m1 == -kInf ? 0.f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
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
      const float b0 = m0 == -kInf ? 0.f : m0, b1 = m1 == -kInf ? 0.f : m1;
#pragma unroll
      for (int u = 0; u < K::kGroups; ++u) {
        float(&ya)[4] = x[2 * u];
        float(&yb)[4] = x[2 * u + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ya[e] = ex2(ya[e] - (e < 2 ? b0 : b1));
          yb[e] = ex2(yb[e] - (e < 2 ? b0 : b1));
        }
        l0 = fmaf((ya[0] + ya[1]) + (yb[0] + yb[1]), per[u], l0);
        l1 = fmaf((ya[2] + ya[3]) + (yb[2] + yb[3]), per[u], l1);
        const uint32_t p[4] = {pack_half2(ya[0], ya[1]), pack_half2(ya[2], ya[3]),
                               pack_half2(yb[0], yb[1]), pack_half2(yb[2], yb[3])};
        // Keys of this lane's four operand rows; D / 8 of their channels each.
        constexpr int kWords = D / 32;
        uint32_t w[4][kWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * u + 8 * (i / 2) + (i & 1 ? 4 + (t ^ 1) : t);
          if (D == 64) {
            const uint2 v = *reinterpret_cast<const uint2*>(vs + chunk_at<D>(r, g / 2) + (g & 1) * 8);
            w[i][0] = v.x;
            w[i][1] = v.y;
          } else {
            const uint4 v = *reinterpret_cast<const uint4*>(vs + chunk_at<D>(r, g));
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

    // Join the warps. Each writes O into the stage it consumed last (nothing
    // is in flight there), rows of D fp32, and its rows' M and l.
    float* const stats = reinterpret_cast<float*>(smem + K::kStats);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    int* const where = reinterpret_cast<int*>(warp_sum);  // stage of each warp, -1: none
    __syncwarp();
    if (lane == 0) where[warp] = latest < 0 ? -1 : (warp * K::kStages + latest) * K::kStage;
    if (latest >= 0) {
      if (t == 0) {
        stats[(warp * K::kRows + g) * 2] = m0;
        stats[(warp * K::kRows + g) * 2 + 1] = l0;
        stats[(warp * K::kRows + g + 8) * 2] = m1;
        stats[(warp * K::kRows + g + 8) * 2 + 1] = l1;
      }
      float* dst = reinterpret_cast<float*>(stages + latest * K::kStage);
      // Accumulator i, columns 2t, 2t + 1: channels (D / 8) column + i.
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < D / 8; i += 4)
          *reinterpret_cast<float4*>(dst + (g + 4 * (e & 2)) * D + (D / 8) * (2 * t + (e & 1)) + i) =
              make_float4(o[i][e], o[i + 1][e], o[i + 2][e], o[i + 3][e]);
    }
    __syncthreads();
    const bool whole = item.tile == item.item_begin && item_hi == item.item_end;
    // An item that began in an earlier share leaves its partial in slot 0,
    // one that begins here and goes on in slot 1.
    float* const part = scratch + (item.tile == item.item_begin ? K::kRows * (D + 2) : 0);
    for (int i = threadIdx.x; i < K::kRows * D / 4; i += K::kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      const int row = item.row0 + r;
      if (row >= rows) continue;
      float m = -kInf;
      for (int w = 0; w < K::kWarps; ++w)
        if (where[w] >= 0) m = fmaxf(m, stats[(w * K::kRows + r) * 2]);
      const float base = m == -kInf ? 0.f : m;
      float l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < K::kWarps; ++w) {
        if (where[w] < 0) continue;
        const float f = ex2(stats[(w * K::kRows + r) * 2] - base);
        l = fmaf(stats[(w * K::kRows + r) * 2 + 1], f, l);
        const float4 v = *reinterpret_cast<const float4*>(smem + where[w] + (r * D + d) * 4);
        sum.x = fmaf(v.x, f, sum.x);
        sum.y = fmaf(v.y, f, sum.y);
        sum.z = fmaf(v.z, f, sum.z);
        sum.w = fmaf(v.w, f, sum.w);
      }
      if (whole) {
        const bool some = !(l == 0.f);
        const float inv = some ? 1.f / l : 0.f;
        const long long head = (long long)(s.first + row / z.group) * a.heads +
                               item.kv_head * z.group + row % z.group;
        T* out = (T*)a.out + head * D + d;
        out[0] = from_float<T>(some ? sum.x * inv : 0.f);
        out[1] = from_float<T>(some ? sum.y * inv : 0.f);
        out[2] = from_float<T>(some ? sum.z * inv : 0.f);
        out[3] = from_float<T>(some ? sum.w * inv : 0.f);
        if (a.lse && d == 0) a.lse[head] = some ? (m + log2f(l)) * kLn2 : -kInf;
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = sum;
        if (d == 0) {
          part[K::kRows * D + 2 * r] = m;
          part[K::kRows * D + 2 * r + 1] = l;
        }
      }
    }
    if (!whole && item.tile == item.item_begin && threadIdx.x == 0) {
      // The last share that holds a tile of the item.
      const int last = share_of(total, item.item_end - 1, ctas);
      mine.first = s.first;
      mine.rows = rows;
      mine.row0 = item.row0;
      mine.kv_head = item.kv_head;
      mine.parts = last - (int)blockIdx.x + 1;
    }
    __syncthreads();  // the stages are free again
    item.tile = item_hi;
  }
  __pipeline_wait_prior(0);
}

// Joins the partial results of the item (of ROWS rows) that starts in share
// blockIdx.x and goes on into later ones: 16 rows a CTA, one thread per four
// channels of a row, in the order of the shares.
template <typename T, int D, int ROWS>
__global__ void combine_kernel(const cxs_cache_attend_call a, const Shape z) {
  constexpr int kRows = ROWS, kSize = kRows * (D + 2);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Partial* partials = reinterpret_cast<const Partial*>(a.workspace);
  const Partial item = partials[blockIdx.x];
  if (item.parts == 0) return;
  const float* scratch =
      reinterpret_cast<const float*>(partials + z.grid) + (long long)blockIdx.x * 2 * kSize;
  const int r = 16 * blockIdx.y + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  const int row = item.row0 + r;
  if (row >= item.rows) return;
  auto part = [&](int i) { return scratch + (i == 0 ? kSize : 2 * i * kSize); };
  float m = -kInf;
#pragma unroll 8
  for (int i = 0; i < item.parts; ++i) m = fmaxf(m, part(i)[kRows * D + 2 * r]);
  const float base = m == -kInf ? 0.f : m;
  float l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = 0; i < item.parts; ++i) {
    const float f = ex2(part(i)[kRows * D + 2 * r] - base);
    l = fmaf(part(i)[kRows * D + 2 * r + 1], f, l);
    const float4 v = *reinterpret_cast<const float4*>(part(i) + r * D + d);
    sum.x = fmaf(v.x, f, sum.x);
    sum.y = fmaf(v.y, f, sum.y);
    sum.z = fmaf(v.z, f, sum.z);
    sum.w = fmaf(v.w, f, sum.w);
  }
  const bool some = !(l == 0.f);
  const float inv = some ? 1.f / l : 0.f;
  const long long head =
      (long long)(item.first + row / z.group) * a.heads + item.kv_head * z.group + row % z.group;
  T* out = (T*)a.out + head * D + d;
  out[0] = from_float<T>(some ? sum.x * inv : 0.f);
  out[1] = from_float<T>(some ? sum.y * inv : 0.f);
  out[2] = from_float<T>(some ? sum.z * inv : 0.f);
  out[3] = from_float<T>(some ? sum.w * inv : 0.f);
  if (a.lse && d == 0) a.lse[head] = some ? (m + log2f(l)) * kLn2 : -kInf;
}

// ------------------------------------------------------------------ host ---

int check_attend(const cxs_cache_attend_call* a) {
  if (!a) return set_error(CXS_ERR_INVALID, "cache attend: null call");
  const int status = cxs_host::check_cache(&a->cache, "cache attend");
  if (status != CXS_OK) return status;
  if (a->cache.type == CXS_TYPE_F32)
    return set_error(CXS_ERR_INVALID, "cache attend: queries must be bf16 or fp16");
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return set_error(CXS_ERR_INVALID, "cache attend: heads must be a multiple of kv_heads");
  if (a->window < 0) return set_error(CXS_ERR_INVALID, "cache attend: negative window");
  if ((long long)a->cache.max_tokens * a->heads > 0x40000000ll)
    return set_error(CXS_ERR_CAPACITY, "cache attend: more than 2^30 rows of one user");
  return CXS_OK;
}

// SMs of the current device (looked up once).
int sm_count(int* sms) {
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

// Largest grid a call uses: one CTA per SM of a B200. A constant, so that the
// workspace's size does not depend on the device.
constexpr int kMostCtas = 148;

// Most rows of a user and KV head for which the mma.sync kernel runs.
constexpr int kFewRows = 64;

bool few_rows(const cxs_cache_attend_call& a) {
  return (long long)a.cache.max_tokens * (a.heads / a.cache.kv_heads) <= kFewRows;
}

long long workspace_bytes(const cxs_cache_attend_call& a) {
  const long long rows = few_rows(a) ? 16 : kTileRows;
  return kMostCtas * (sizeof(Partial) + 2 * rows * (a.cache.dim + 2) * (long long)sizeof(float));
}

template <int FORMAT, typename T, int D>
int launch_decode(const cxs_cache_attend_call& a, const Shape& z, cudaStream_t stream) {
  using K = Decode<D>;
  static cxs_host::OncePerDevice ready;
  const int status = ready.run([] {
    CXS_CUDA(cudaFuncSetAttribute(decode_kernel<FORMAT, T, D>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, K::kBytes));
    return (int)CXS_OK;
  });
  if (status != CXS_OK) return status;
  decode_kernel<FORMAT, T, D><<<z.grid, K::kThreads, K::kBytes, stream>>>(a, z);
  CXS_LAUNCH_CHECK("cache attend");
  return CXS_OK;
}

template <typename T, int D>
int launch_combine(const cxs_cache_attend_call& a, const Shape& z, bool few, cudaStream_t stream) {
  // Its CTAs may start while the last CTAs before finish; they wait for them
  // on the device.
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(z.grid, few ? 1 : kTileRows / 16);
  config.blockDim = dim3(16 * D / 4);
  config.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  if (few)
    CXS_CUDA(cudaLaunchKernelEx(&config, combine_kernel<T, D, 16>, a, z));
  else
    CXS_CUDA(cudaLaunchKernelEx(&config, combine_kernel<T, D, kTileRows>, a, z));
  CXS_LAUNCH_CHECK("cache attend join");
  return CXS_OK;
}

}  // namespace

extern "C" int cxs_cache_attend_workspace(const cxs_cache_attend_call* call, int64_t* bytes) {
  const int status = check_attend(call);
  if (status != CXS_OK) return status;
  if (!bytes) return set_error(CXS_ERR_INVALID, "cache attend: null result");
  *bytes = workspace_bytes(*call);
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
  if (!call->workspace || (uintptr_t)call->workspace % 16 ||
      call->workspace_bytes < workspace_bytes(*call))
    return set_error(CXS_ERR_INVALID, "cache attend: workspace missing, unaligned or too small");
  int sms = 0;
  status = sm_count(&sms);
  if (status != CXS_OK) return status;
  const int grid = sms < kMostCtas ? sms : kMostCtas;
  const bool few = few_rows(*call);
  cudaStream_t s = (cudaStream_t)stream;
  for (int user0 = 0; user0 < c.users; user0 += kSlice) {
    cxs_cache_attend_call a = *call;
    const int left = c.users - user0;
    const Shape z{call->heads / c.kv_heads, user0, left < kSlice ? left : kSlice, left <= kSlice,
                  grid, few ? Decode<64>::kWarps : 2};
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
    if (c.type == CXS_TYPE_BF16)
      status = c.dim == 64 ? launch_combine<__nv_bfloat16, 64>(a, z, few, s)
                           : launch_combine<__nv_bfloat16, 128>(a, z, few, s);
    else
      status = c.dim == 64 ? launch_combine<__half, 64>(a, z, few, s)
                           : launch_combine<__half, 128>(a, z, few, s);
    if (status != CXS_OK) return status;
  }
  return CXS_OK;
}
