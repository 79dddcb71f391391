// Attention of users that have their first tokens in common, over the dense
// 8-bit cache: the common tokens are read once for all of a group's rows.
//
// Mathematics. A row's softmax runs over the common keys and its user's own:
//   out = (sum_common p v + sum_own p v) / (sum_common p + sum_own p),
// one running maximum and sum for both, so nothing is joined that one pass of the
// tile kernel (cache8_tile.cuh) does not already join. Its items are 256 query
// rows of a group, whichever users they belong to.
//
// plan_kernel works out, from lengths and offsets on the device, what the items
// are and where each CTA's equal share of their tiles begins.
#include "cache8_tile.cuh"

using cxs_host::set_error;

namespace {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;

// Sum of v over the threads before this one; *total: over all.
__device__ __forceinline__ long long block_scan(long long v, long long* total) {
  __shared__ long long sums[kPlanWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();  // (the sums of the scan before have been read)
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  long long all = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const long long before = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);
  return sum - v + (warp > 0 ? before : 0);
}

// Most users and groups whose offsets, runs and plans are kept in shared memory:
// the searches among them are chains of loads (3.4 us of the plan's 8 from global).
constexpr int kFewUsers = 2048, kFewGroups = 512;

__global__ void __launch_bounds__(kPlanThreads)
    plan_kernel(const cxs_cache_shared_call call, const Shape z, const SharedPlan plan,
                int* first_item) {
  const cxs_cache_attend_call& a = call.attend;
  const cxs_cache_call& c = a.cache;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, groups = call.group_count;
  __shared__ int gaps, many, offsets_here[kFewUsers + 1], first_here[kFewGroups];
  __shared__ long long runs_here[kFewUsers + kFewGroups];
  __shared__ GroupPlan groups_here[kFewGroups];
  const bool here = c.users <= kFewUsers && groups <= kFewGroups;
  const int* const offsets = here ? offsets_here : c.offsets;
  long long* const runs_at = here ? runs_here : plan.runs;
  GroupPlan* const groups_at = here ? groups_here : plan.groups;
  if (here) first_item = first_here;
  const auto first_row = [&](int user) { return offsets ? offsets[user] : user; };
  cxs::after_earlier();
  cxs::next_may_come();
  // Offsets and groups must ascend within the packed rows and the users.
  bool broken = false;
  for (int u = threadIdx.x; u <= c.users; u += kPlanThreads) {
    const int lo = c.offsets ? c.offsets[u] : u;
    if (here) offsets_here[u] = lo;
    if (u == c.users) break;
    const int hi = c.offsets ? c.offsets[u + 1] : u + 1;
    broken |= lo < 0 || hi < lo || hi > c.tokens;
  }
  for (int g = threadIdx.x; g < groups; g += kPlanThreads) {
    const int lo = call.groups[g], hi = call.groups[g + 1];
    broken |= lo < 0 || hi < lo || hi > c.users;
  }
  if (threadIdx.x == 0) gaps = many = 0;
  if (__syncthreads_or(broken)) {
    if (threadIdx.x == 0) {
      report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
      *plan.head = PlanHead{1};
      plan.gaps[0] = Gap{0, c.tokens};
    }
    for (int i = threadIdx.x; i < z.grid; i += kPlanThreads) plan.shares[i].total = 0;
    return;
  }
  // A warp for each group: the tokens that all its rows see, its users' own runs.
  const int most = c.width * c.page_size;
  for (int g = warp; g < groups; g += kPlanWarps) {
    const int u0 = call.groups[g], u1 = call.groups[g + 1];
    const int lo = first_row(u0), hi = first_row(u1);
    int seen = most, bad = 0, none = 0, longest = 0, holder = u1;
    for (int u = u0 + lane; u < u1; u += 32) {
      const int n = first_row(u + 1) - first_row(u), length = c.lengths[u];
      none |= n > c.max_tokens;
      bad |= length < 0 || length > most;
      if (n == 0) continue;  // (it may hold other tokens, or none)
      holder = min(holder, u);
      seen = min(seen, max(a.causal ? min(length, length - n + 1) : length, 0));
      longest = max(longest, min(length, most));
    }
    seen = __reduce_min_sync(0xffffffffu, seen);
    longest = __reduce_max_sync(0xffffffffu, longest);
    holder = __reduce_min_sync(0xffffffffu, holder);
    none = __any_sync(0xffffffffu, none);
    int shared = call.shared[g];
    bad |= shared < 0;
    shared = min(max(shared, 0), seen);
    // An item's own keys are counted in 32 bits.
    none |= (long long)(longest - shared) * min(u1 - u0, kTileRows) > (1 << 30);
    long long runs = 0;
    for (int base = u0; base < u1; base += 32) {
      const int u = base + lane;
      int mine = 0;
      if (u < u1 && first_row(u + 1) > first_row(u)) {
        const int length = min(c.lengths[u], most);
        if (length > shared) mine = (length + 15) / 16 - shared / 16;
      }
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (u < u1) plan.runs[u + g] = runs_at[u + g] = runs + sum - mine;
      runs += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (bad || none) report(c.error, CXS_DEVICE_ERR_BAD_LENGTH);
    if (lane == 0) {
      plan.runs[u1 + g] = runs_at[u1 + g] = runs;
      groups_at[g] = GroupPlan{lo, none ? 0 : hi - lo, shared, holder};
      if (none) plan.gaps[atomicAdd(&gaps, 1)] = Gap{lo, hi};
      else if ((hi - lo) * z.group > kTileRows / 2) many = 1;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    plan.gaps[gaps] = Gap{0, first_row(call.groups[0])};
    plan.gaps[gaps + 1] = Gap{first_row(call.groups[groups]), c.tokens};
  }
  // Items of the groups before each.
  long long items = 0;
  for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int g = g0 + threadIdx.x;
    const long long rows = g < groups ? (long long)groups_at[g].count * z.group : 0;
    long long all;
    const long long before = block_scan((rows + kTileRows - 1) / kTileRows, &all);
    if (g < groups) first_item[g] = (int)(items + before);
    items += all;
  }
  __syncthreads();
  long long total = 0;
  for (int i0 = 0; i0 < items; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    ItemPlan item = {};
    if (i < items) {
      int l = 0, h = groups - 1;  // the last group that begins at or before i
      while (l < h) {
        const int m = (l + h + 1) / 2;
        if (first_item[m] <= i) l = m; else h = m - 1;
      }
      const GroupPlan group = groups_at[l];
      const int end = call.groups[l + 1] - 1;
      item.group = l;
      item.of = group;
      item.tile_row = i - first_item[l];
      const int row0 = item.tile_row * kTileRows;
      const int row1 = min(group.count * z.group, row0 + kTileRows) - 1;
      item.user_a = user_of(offsets, group.first + row0 / z.group, group.user0, end);
      item.user_b = user_of(offsets, group.first + row1 / z.group, item.user_a, end);
      const long long* const runs = runs_at + l;
      item.common_tiles = (group.shared + kKeys - 1) / kKeys;
      item.tiles = item.common_tiles +
                   (int)((runs[item.user_b + 1] - runs[item.user_a] + kRuns - 1) / kRuns);
      if (item.tiles == 0) item.tiles = 1;  // (its rows are written all the same)
    }
    long long all;
    const long long cost = i < items ? (long long)(item.tiles + kItemCost) * c.kv_heads : 0;
    item.before = total + block_scan(cost, &all);
    if (i < items) plan.items[i] = item;
    total += all;
  }
  __syncthreads();
  if (threadIdx.x == 0) *plan.head = PlanHead{gaps + 2};
  // Where each share begins: among all tiles, without the items' own costs.
  const Shares shares(total, z);
  for (int i = threadIdx.x; i < z.grid; i += kPlanThreads) {
    plan.shares[i].total = total;
    plan.shares[i].solo = !many;
  }
  for (int i = threadIdx.x; shares.count > 0 && i <= shares.count; i += kPlanThreads) {
    long long at = total - (long long)kItemCost * items * c.kv_heads;
    if (i < shares.count) {
      const long long place = shares.begin(i);
      int l = 0, h = (int)items - 1;  // the last item that begins at or before it
      while (l < h) {
        const int m = (l + h + 1) / 2;
        if (plan.items[m].before <= place) l = m; else h = m - 1;
      }
      const ItemPlan item = plan.items[l];
      const int cost = item.tiles + kItemCost, kv_head = (int)divide(place - item.before, cost);
      const long long begin = item.before + (long long)kv_head * cost;
      at = begin - kItemCost * ((long long)l * c.kv_heads + kv_head) +
           max(place - begin - kItemCost, 0ll);
      plan.shares[i].low = at;
      plan.shares[i].id = l;
      plan.shares[i].kv_head = kv_head;
      plan.shares[i].item = item;
    }
    if (i > 0) plan.shares[i - 1].high = at;
  }
}

// Where the plan's parts lie behind the partial results; the bytes of all.
long long lay_out(const cxs_cache_shared_call& call, char* workspace, SharedPlan* plan,
                  int** first_item) {
  const cxs_cache_call& c = call.attend.cache;
  const long long group = call.attend.heads / c.kv_heads;
  const long long groups = call.group_count;
  long long at = partial_bytes(call.attend, false);
  auto take = [&](long long bytes) {
    at = (at + 15) / 16 * 16;
    char* const from = workspace + at;
    at += bytes;
    return from;
  };
  plan->head = (PlanHead*)take(sizeof(PlanHead));
  plan->groups = (GroupPlan*)take(groups * sizeof(GroupPlan));
  plan->items = (ItemPlan*)take((c.tokens * group / kTileRows + groups) * sizeof(ItemPlan));
  plan->shares = (SharePlan*)take(kMostCtas * sizeof(SharePlan));
  plan->runs = (long long*)take((c.users + groups) * sizeof(long long));
  plan->gaps = (Gap*)take((groups + 2) * sizeof(Gap));
  *first_item = (int*)take(groups * sizeof(int));
  return at;
}

// Groups of few rows: every user reads all its keys by itself.
bool few_shared(const cxs_cache_shared_call& call) {
  const cxs_cache_call& c = call.attend.cache;
  return few_rows(call.attend) &&
         (long long)c.tokens * (call.attend.heads / c.kv_heads) <=
             (long long)call.group_count * (c.dim == 64 ? 64 : 32);
}

int check_shared(const cxs_cache_shared_call* call) {
  const char* const what = "cache attend shared";
  if (!call) return set_error(CXS_ERR_INVALID, "%s: null call", what);
  const int status = check_attend(&call->attend, what);
  if (status != CXS_OK) return status;
  if (call->attend.window) return set_error(CXS_ERR_INVALID, "%s: no window", what);
  if (call->group_count < 0 || call->group_count > call->attend.cache.users)
    return set_error(CXS_ERR_INVALID, "%s: groups must be 0 .. users", what);
  if ((long long)call->attend.cache.tokens * call->attend.heads > 0x40000000ll)
    return set_error(CXS_ERR_CAPACITY, "%s: more than 2^30 rows", what);
  return CXS_OK;
}

long long workspace_of(const cxs_cache_shared_call& call) {
  SharedPlan plan;
  int* first_item;
  return few_shared(call) ? partial_bytes(call.attend, true)
                          : lay_out(call, nullptr, &plan, &first_item);
}

}  // namespace

extern "C" int cxs_cache_attend_shared_workspace(const cxs_cache_shared_call* call,
                                                 int64_t* bytes) {
  const int status = check_shared(call);
  if (status != CXS_OK) return status;
  if (!bytes) return set_error(CXS_ERR_INVALID, "cache attend shared: null result");
  *bytes = workspace_of(*call);
  return CXS_OK;
}

extern "C" int cxs_cache_attend_shared(const cxs_cache_shared_call* call, void* stream) {
  const char* const what = "cache attend shared";
  int status = check_shared(call);
  if (status != CXS_OK) return status;
  const cxs_cache_call& c = call->attend.cache;
  if (c.tokens == 0) return CXS_OK;
  if (c.users == 0 || call->group_count == 0)
    return set_error(CXS_ERR_INVALID, "%s: rows without users or groups", what);
  status = check_attend_pointers(&call->attend, workspace_of(*call), what);
  if (status != CXS_OK) return status;
  if (!call->groups || !call->shared) return set_error(CXS_ERR_INVALID, "%s: null groups or shared", what);
  if (few_shared(*call)) return cxs_cache_attend(&call->attend, stream);
  int sms = 0;
  status = sm_count(&sms);
  if (status != CXS_OK) return status;
  const int grid = sms < kMostCtas ? sms : kMostCtas;
  cudaStream_t s = (cudaStream_t)stream;
  const Shape z{call->attend.heads / c.kv_heads, 0, c.users, 1, grid, grid, 2, 0};
  SharedPlan plan;
  int* first_item;
  lay_out(*call, (char*)call->attend.workspace, &plan, &first_item);
  status = cxs_host::launch_early("cache attend shared plan", plan_kernel, 1, kPlanThreads, 0, 0, s,
                                  *call, z, plan, first_item);
  status = launch_of<true>(call->attend, z, plan, s);
  if (status != CXS_OK) return status;
  return launch_join(call->attend, z, false, false, s);
}
