// Attention of the newest tokens over the paged cache in 8 bits, for rows that share leading pages: what a group of rows shares is read once for all of them.
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^((q . k_j) scale log2(e) - m),  k_j and v_j codes times their block's scale.
// A plan says which rows share what.  Rows with the same first page are compared with the lowest of them; of these the rows that share S pages or more are a
// group, with the S that saves most, S times the rows but one.  The queries of a group's rows lie one behind the other in tiles of 32 (queries x heads of one head of the cache) over
// the shared pages, and every row's in tiles of their own over the rest. A tile's keys are cut into jobs of about one size, a workgroup each for every head of the cache, which leaves
// a state (maximum, sum, weighted values); a second launch makes one of the states of a row's queries.
//
// What bounds it: the bytes of the pages, and two launches with a chain of look-ups in each (job, queries, page, keys), some 12 us for a call that reads next to nothing of 128
// features.  64 rows of 64 to 4000 tokens that share nothing, 32 heads on 8 of 128, int8: 59 us, 4.0 TB/s (cache_attention 52).  64 rows behind 7936 shared tokens, 16 heads on 4, e4m3:
// 37 (cache_attention 73); 16 rows behind 99968, int8: 43 (182).  In these the first-level caches hand on 127 and 210 MB, every tile its own, at 4 to 5.5 TB/s; loads alone, as many
// in flight and nothing cached, take 23 us for 100 MB and 39 for 200.  Tiles of 32 rows, as two share the codes' way to fp16: a wave with more would leave one wave a SIMD, while four waves on the
// same keys, 32 rows each, were not tried; fewer instructions do not help (codes of int8 as subnormal numbers with the offset of 128 taken off by the products, 600 -> 480 vector instructions for 64 keys and 32 rows: 1 to 3 % of the time).
#include "prefix_kernels.h"

#include "cache_codes.h"

#include <limits.h>

namespace sspmm {

namespace {

typedef unsigned long long u64;

constexpr int kRows = 32;   // of a tile
constexpr int kWaves = 4;   // of a workgroup, which share a job's units
constexpr int kPlaces = 512;     // for workgroups, two a CU
constexpr int kJobKeys = 1280;   // that a workgroup goes over in the time that it takes to begin and to end (some 14 us)
constexpr int kLeastKeys = 256;  // of a job, as far as there are: 64 for each of its waves
constexpr int kMostRounds = 4;   // jobs for each place, and one a tile more, are the most that a plan makes
constexpr int kMostStates = kMostRounds * kPlaces + 2;  // of a query: jobs of two tiles

// ---- the plan: 32-bit words, in this order
//   header  jobs, 0, 0, 0
//   jobs    those of the shared pages first, of all tiles of a group the same keys side by side; then the rows' own, the longest rows first
//   rows    by their number
//   order   the rows, group after group, and their lengths
//   leaders, shared pages (of the first launch)
constexpr int kHeaderWords = 4;
struct Job {
  int row;           // of the table
  int unit0, unit1;  // of the row
  int end;           // positions of the row from here on are not the job's
  int all_seen;      // every query sees the keys below
  int member;        // place in the order of the row whose queries come first in the tile's group
  int first, count;  // its first query among theirs, and queries
  int states;        // the first row of its state
  int unused[3];     // (whole blocks of 16 bytes)
};
struct RowPlan {
  // A tile's jobs leave as many rows as it has queries, one job's behind the other's, and one tile's behind the other's.
  int shared_states, shared_jobs;  // of the first tile of the group: its jobs' first row; jobs of a tile, 0: there is no group
  int shared_queries, place;       // of the group; the row's place in it
  int own_states, own_jobs;
  int unused[2];  // (the same)
};
struct Ordered {
  int row, length;  // tokens, also those that the table has no slot for
};
struct PrefixPlan {
  int32_t *header;
  Job *jobs;
  RowPlan *rows;
  Ordered *order;
  int32_t *leaders, *shared;
  __host__ __device__ PrefixPlan(int32_t *at, const PrefixShape &s, int n) {
    header = at;
    jobs = reinterpret_cast<Job *>(at + kHeaderWords);
    rows = reinterpret_cast<RowPlan *>(jobs + s.jobs);
    order = reinterpret_cast<Ordered *>(rows + n);
    leaders = reinterpret_cast<int32_t *>(order + n);
    shared = leaders + n;
  }
  __host__ __device__ long long words(int n) const { return shared + n - header; }
};

// Keys of a unit, all of them in one page.
__host__ __device__ constexpr int unit_of(int page_size) { return page_size == 32 ? 32 : 64; }

// Pages that lie whole in front of the row's first query.
__device__ __forceinline__ int full_pages(int length, int queries, int page_size, int slots) {
  return (int)min((long long)slots, max(0ll, (long long)length - queries + 1) / page_size);
}

// The lowest row that begins with the same page as `row`, and the pages that the two share: by WAVES waves, of which this is number `wave`; with more than one, a workgroup.
template <int WAVES>
__device__ __forceinline__ int2 compare(int row, int wave, const int32_t *table, int rows, int slots, const int32_t *lengths, int page_size, int queries, int (&ends)[WAVES]) {
  const int lane = threadIdx.x & 63;
  const int32_t *const own = table + (long long)row * slots;
  const int first = own[0], full = full_pages(lengths[row], queries, page_size, slots);
  int leader = -1, shared = 0;
  if (first >= 0 && full > 0) {
    int most = 0;
    for (int at = 0; at < rows && leader < 0; at += 64) {
      const int r = at + lane;
      const int begins = r < rows ? table[(long long)r * slots] : -1, pages = r < rows ? full_pages(lengths[r], queries, page_size, slots) : 0;
      const u64 those = __ballot(begins == first && pages > 0);
      if (those) {
        const int lowest = __builtin_ctzll(those);
        leader = at + lowest;
        most = min(full, __builtin_amdgcn_readlane(pages, lowest));
      }
    }
    const int32_t *const other = table + (long long)leader * slots;
    // (a wave looks at 512 slots at a time)
    constexpr int kAtOnce = 8;
    for (shared = 0; shared < most;) {
      const int from = shared + 64 * kAtOnce * wave;
      bool same[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int s = from + 64 * i + lane, at = min(s, most - 1);
        const int mine = own[at];
        same[i] = s < most && mine >= 0 && mine == other[at];
      }
      int end = INT_MAX;  // the first that differs
#pragma unroll
      for (int i = kAtOnce - 1; i >= 0; --i) {
        const u64 differ = __ballot(!same[i]);
        end = differ ? from + 64 * i + __builtin_ctzll(differ) : end;
      }
      if constexpr (WAVES > 1) {
        __syncthreads();
        if (lane == 0) ends[wave] = end;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) end = min(end, ends[i]);
      }
      shared += 64 * kAtOnce * WAVES;
      if (end != INT_MAX) {
        shared = min(end, most);
        break;
      }
    }
  }
  return {leader, shared};
}

// A workgroup a row.
constexpr int kCompareWaves = 4;
__global__ __launch_bounds__(64 * kCompareWaves) void plan_prefixes_compare_kernel(PrefixPlan plan, const int32_t *table, int rows, int slots, const int32_t *lengths, int page_size,
                                                                                   int queries) {
  __shared__ int ends[kCompareWaves];
  const int row = blockIdx.x;
  const int2 found = compare<kCompareWaves>(row, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), table, rows, slots, lengths, page_size, queries, ends);
  if (threadIdx.x == 0) {
    plan.leaders[row] = found.x;
    plan.shared[row] = found.y;
  }
}

// Sum of v over the threads in front of the own one, and over all.
__device__ __forceinline__ u64 sum_before(u64 v, u64 (&waves)[kMostPlanRows / 64], u64 &all) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const u64 upto = wave_inclusive_sum(v);
  __syncthreads();
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  const u64 sums = wave_inclusive_sum(lane < (int)(blockDim.x >> 6) ? waves[lane] : 0);
  const auto of = [&](int i) { return (u64)(uint32_t)__builtin_amdgcn_readlane((int)sums, i) | (u64)(uint32_t)__builtin_amdgcn_readlane((int)(sums >> 32), i) << 32; };
  all = of(63);
  return upto - v + (wave ? of(wave - 1) : 0);
}

// One workgroup, a thread a row (and more threads than that).  table: no launch has compared the rows, but here a wave does it for each
// (up to 8: 3 rows 7.6 us and, with the launch, 9.2, 8 rows 8.7 and 9.5, 16 rows 15.3 and 11.8).
constexpr int kFewRows = 8;
__global__ __launch_bounds__(kMostPlanRows) void plan_prefixes_kernel(PrefixPlan plan, const int32_t *table, int rows, int slots, const int32_t *lengths, int page_size, int queries,
                                                                      PrefixShape shape) {
  __shared__ int2 found[kMostPlanRows];  // leader, shared pages
  __shared__ int base[kMostPlanRows];
  __shared__ int in_orders[kMostPlanRows], lengths_of[kMostPlanRows], group_queries[kMostPlanRows];
  __shared__ int by_rank[kMostPlanRows], shared_job[kMostPlanRows], own_job[kMostPlanRows], shared_states[kMostPlanRows], own_states[kMostPlanRows];
  __shared__ u64 best[kMostPlanRows], waves[kMostPlanRows / 64];
  const int r = threadIdx.x;
  const bool there = r < rows;
  found[r] = {-1, 0};
  best[r] = 0;
  if (table) {
    const int wave = __builtin_amdgcn_readfirstlane(r >> 6);
    int none[1];
    __syncthreads();
    if (wave < rows) {
      const int2 of_row = compare<1>(wave, 0, table, rows, slots, lengths, page_size, queries, none);
      if ((r & 63) == 0) found[wave] = of_row;
    }
  } else if (there) {
    found[r] = {plan.leaders[r], plan.shared[r]};
  }
  __syncthreads();
  const int leader = found[r].x, mine = found[r].y;
  // ---- the pages that a group shares: of its rows' numbers the one that saves most
  if (leader >= 0) {
    int as_many = 0;
#pragma unroll 8
    for (int i = 0; i < rows; ++i) as_many += (found[i].x == leader) & (found[i].y >= mine);
    const u64 saved = (u64)mine * (u64)(as_many - 1);
    if (saved) atomicMax(&best[leader], saved << 26 | (u64)mine);  // (fewer than 2^26 slots)
  }
  __syncthreads();
  const u64 chosen = leader >= 0 ? best[leader] : 0;
  const int pages = (int)(chosen & ((1u << 26) - 1)), own_pages = chosen && mine >= pages ? pages : 0;
  const bool member = own_pages > 0, leads = member && leader == r;
  // ---- order: a group's rows stand where its leader would
  __syncthreads();
  found[r].y = own_pages;
  __syncthreads();
  int place = 0, members = 0;
  if (member)
#pragma unroll 8
    for (int i = 0; i < rows; ++i) {
      const int one = (found[i].x == leader) & (found[i].y > 0);
      members += one;
      place += one & (i < r);
    }
  u64 all;
  const u64 at = sum_before(there ? (leads ? members : member ? 0 : 1) : 0, waves, all);
  base[r] = (int)at;
  __syncthreads();
  const int in_order = member ? base[leader] + place : (int)at;
  const int length = there ? max(0, lengths[r]) : 0, end = (int)min((long long)length, (long long)slots * page_size);
  if (there) plan.order[in_order] = {r, length};
  // ---- jobs: the groups' tiles in the order of their leaders, then every row's own
  const int from = own_pages * page_size, unit = unit_of(page_size);
  const int stacked = leads ? members * shape.row_queries : 0;  // queries of the group
  const int group_tiles = (stacked + kRows - 1) / kRows, own_tiles = there ? (shape.row_queries + kRows - 1) / kRows : 0;
  const int group_units = from / unit, own_units = (end - from + unit - 1) / unit;
  u64 units, all_tiles, shared_jobs, jobs, states;
  sum_before((u64)group_tiles * group_units + (u64)own_tiles * own_units, waves, units);
  sum_before((u64)(group_units ? group_tiles : 0) + (u64)(own_units ? own_tiles : 0), waves, all_tiles);
  // Units of a job, at most: as few as leave no more jobs than there are places, so that all run at once, found by halving; or, with too many tiles for that, so many that
  // the last jobs' time and what beginning and ending take of all together are least.
  const int least = kLeastKeys / unit;
  const u64 most_jobs = (u64)kMostRounds * shape.target;  // (and one a tile more; the buffers have room for so many)
  int size = max(max(least, (int)sqrtf((float)units * (float)(kJobKeys / unit) / (float)shape.target)), (int)min((units + most_jobs - 1) / most_jobs, (u64)1 << 27));
  if (4 * all_tiles <= 3 * (u64)shape.target) {
    // (jobs of n units in all tiles are fewer than n / size + tiles)
    u64 low = max((u64)least, (units + shape.target - 1) / shape.target), high = max(low, (units + shape.target - all_tiles - 1) / (shape.target - all_tiles));
    while (low < high) {
      const u64 step = (high - low + 3) / 4;
      u64 mine = 0, counts;
      for (int i = 0; i < 3; ++i) {  // three sizes at a time; a thread's jobs matter up to the places
        const uint32_t at = (uint32_t)(low + i * step);  // (below 2^29; 32 bits divide much faster than 64)
        const u64 jobs = (u64)group_tiles * (((uint32_t)group_units + at - 1) / at) + (u64)own_tiles * (((uint32_t)own_units + at - 1) / at);
        mine |= min(jobs, (u64)2 * kPlaces) << 21 * i;
      }
      sum_before(mine, waves, counts);
      int few = 0;  // sizes that are too small
      for (int i = 0; i < 3; ++i) few += (counts >> 21 * i & ((1u << 21) - 1)) > (u64)shape.target;
      if (few < 3) high = min(high, low + few * step);
      if (few > 0) low = min(high, low + (few - 1) * step + 1);
    }
    size = (int)high;
  }
  const int group_cuts = (group_units + size - 1) / size, own_cuts = (own_units + size - 1) / size;  // jobs of a tile
  shared_job[r] = (int)sum_before((u64)group_tiles * group_cuts, waves, shared_jobs);
  lengths_of[r] = there ? own_units : -1;
  __syncthreads();
  int rank = there ? 0 : r;
  if (there)
#pragma unroll 8
    for (int i = 0; i < rows; ++i) rank += (lengths_of[i] > own_units) | ((lengths_of[i] == own_units) & (i < r));
  by_rank[rank] = r;
  __syncthreads();
  // (own_job and by_rank are of the r'th longest row)
  const int ranked_units = there ? lengths_of[by_rank[r]] : 0, ranked_cuts = (ranked_units + size - 1) / size;
  own_job[r] = (int)(shared_jobs + sum_before((u64)own_tiles * ranked_cuts, waves, jobs));
  // (rows of states are below 2^25)
  const u64 states_before = sum_before((u64)stacked * group_cuts | (there ? (u64)shape.row_queries * own_cuts : 0) << 32, waves, states);
  shared_states[r] = (int)(uint32_t)states_before;
  own_states[r] = (int)(uint32_t)states + (int)(states_before >> 32);
  group_queries[r] = stacked;
  in_orders[r] = in_order;
  lengths_of[r] = length;
  __syncthreads();
  if (there) plan.rows[r] = {member ? shared_states[leader] : 0, member ? group_cuts : 0, member ? group_queries[leader] : 0, place, own_states[r], own_cuts, {0, 0}};
  const int all_jobs = (int)(shared_jobs + jobs);
  for (int j = r; j < all_jobs; j += blockDim.x) {
    const bool of_group = j < (int)shared_jobs;
    const int *const first_job = of_group ? shared_job : own_job;
    int at = 0;  // the last whose first job is not behind j
    for (int step = kMostPlanRows / 2; step > 0; step /= 2)
      if (at + step < rows && first_job[at + step] <= j) at += step;
    const int row = of_group ? at : by_rank[at], which = j - first_job[at];
    const int start = found[row].y * page_size, stop = (int)min((long long)lengths_of[row], (long long)slots * page_size);
    const int row_units = of_group ? start / unit : (stop - start + unit - 1) / unit, cuts = (row_units + size - 1) / size;
    const int tiles = ((of_group ? group_queries[row] : shape.row_queries) + kRows - 1) / kRows;
    const int tile = which % tiles, cut = which / tiles, first = tile * kRows;
    const int count = min(kRows, (of_group ? group_queries[row] : shape.row_queries) - first);
    const int each = row_units / cuts, more = row_units % cuts;  // units of a job, and the first jobs that have one more
    const int unit0 = (of_group ? 0 : start / unit) + cut * each + min(cut, more);
    plan.jobs[j] = {row, unit0, unit0 + each + (cut < more), of_group ? start : stop,
                    of_group ? INT_MAX : lengths_of[row] - queries + 1, in_orders[row], first, count,
                    (of_group ? shared_states[row] : own_states[row]) + first * cuts + cut * count, {0, 0, 0}};
  }
  if (r == 0) plan.header[0] = all_jobs;
}

template <typename T, int FORMAT, int D, int TILES, int UNIT>
struct CacheRows {
  static constexpr int kKeyTiles = UNIT / 16, kParts = D / 16, kSteps = D / 32, kShares = UNIT / 32;
  static constexpr int kKeyWords = D >= 64 ? 4 : 2;  // of a load of K: 16 bytes, or 8 where a group's share of a row is no more
  static constexpr int kKeyLoads = D / (16 * kKeyWords);  // of a row by a lane
  static constexpr int kValueWords = UNIT / 16;
  typedef uint32_t KeyWords __attribute__((ext_vector_type(kKeyWords)));
  typedef uint32_t ValueWords __attribute__((ext_vector_type(kValueWords)));

  uintx4 q[TILES][kSteps];
  float c[TILES];
  int seen[TILES];  // keys that the row sees: those below
  floatx4 o[TILES][kParts];  // features 16 part + 4 g + i of row m
  float run_max[TILES], run_sum[TILES];

  // Row m of tile t: its features at `at`.
  __device__ __forceinline__ void load_query(int t, const uint16_t *at, int sees) {
    const int g = (threadIdx.x & 63) >> 4;
    seen[t] = sees;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = D >= 64 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 8 * g;
      q[t][s] = *reinterpret_cast<const uintx4 *>(at + d);
    }
  }
  // bf16 goes to fp16 by way of a power of two for the row, which leaves its largest magnitude in 2^14 .. 2^15
  __device__ __forceinline__ void convert_query(int t, float scale_log2e) {
    c[t] = scale_log2e;
    if constexpr (!__is_same(T, Fp16)) {
      float most = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, fmaxf(fabsf(T::lower(q[t][s][j])), fabsf(T::upper(q[t][s][j]))));
      most = max_over_rows(most);
      const int e = max((int)(__float_as_uint(most) >> 23) - 127 - 14, -126);
      const bool usual = most < INFINITY;  // (else as they are)
      const float up = usual ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.f;
      c[t] *= usual ? __uint_as_float((uint32_t)(127 + e) << 23) : 1.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) q[t][s][j] = Fp16::pack(T::lower(q[t][s][j]) * up, T::upper(q[t][s][j]) * up);
    }
  }

  // Units unit0 .. unit1 - 1 of the sequence whose pages `table` lists, `length` positions of which are something.  all_seen: every row sees the keys below.
  // query(): asks for the queries, once the first unit's page has been asked for.
  template <typename Query>
  __device__ __forceinline__ void attend(const CachePool &pool, const int32_t *table, int head, int unit0, int unit1, int all_seen, int length, float scale_log2e,
                                         const Query &query) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      run_max[t] = kLowest;
      run_sum[t] = 0.f;
#pragma unroll
      for (int part = 0; part < kParts; ++part) o[t][part] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    const long long block = (long long)pool.page_size * D;
    KeyWords kk[kKeyTiles][kKeyLoads];
    ValueWords vv[kParts];
    const int page_units = pool.page_size / UNIT, page_bits = 31 - __builtin_clz(page_units);  // (1 or 2)
    const auto place_of = [&](int u) { return (u & (page_units - 1)) * UNIT; };  // in its page
    const auto usable = [&](int pg) { return pg >= 0 && pg < pool.pages; };
    // Pages and scales of 64 units at a time, one a lane, so that no unit waits for them.
    int pages_of = 0;
    float k_scales = 0.f, v_scales = 0.f;
    const auto ask_pages = [&](int u) { pages_of = table[min(u + lane, unit1 - 1) >> page_bits]; };
    const auto ask_scales = [&]() {
      const float *const scale = pool.scales + (long long)(usable(pages_of) ? pages_of : 0) * 2 * pool.kv_heads + head;
      k_scales = scale[0];
      v_scales = scale[pool.kv_heads] * kValueUnit;
    };
    // A page's keys and values at unit u; a tile of 16 keys, or 16 features, of them.
    const auto keys_at = [&](int u, int pg) { return pool.keys + ((long long)(usable(pg) ? pg : 0) * pool.kv_heads + head) * block + place_of(u) * D; };
    const auto values_at = [&](int u, int pg) { return pool.values + ((long long)(usable(pg) ? pg : 0) * pool.kv_heads + head) * block + place_of(u) + UNIT / 4 * g; };
    const auto load_k = [&](const unsigned char *at, int kt) {
      const unsigned char *const row = at + (UNIT / 4 * (m >> 2) + 4 * kt + (m & 3)) * D + 4 * kKeyWords * g;
#pragma unroll
      for (int i = 0; i < kKeyLoads; ++i) kk[kt][i] = *reinterpret_cast<const KeyWords *>(row + 64 * i);
    };
    const auto load_v = [&](const unsigned char *at, int part) { vv[part] = *reinterpret_cast<const ValueWords *>(at + (16 * part + m) * pool.page_size); };

    int page = 0;
    if (unit0 < unit1) ask_pages(unit0);
    query();
    if (unit0 < unit1) {
      page = __builtin_amdgcn_readlane(pages_of, 0);
#pragma unroll
      for (int kt = 0; kt < kKeyTiles; ++kt) load_k(keys_at(unit0, page), kt);
      ask_scales();
#pragma unroll
      for (int part = 0; part < kParts; ++part) load_v(values_at(unit0, page), part);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) convert_query(t, scale_log2e);
    for (int u = unit0; u < unit1; ++u) {
      const bool more = u + 1 < unit1, there = usable(page);
      const int at = (u - unit0) & 63;
      const float k_scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k_scales), at));
      const float v_scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_scales), at));
      if (at == 63 && more) {
        ask_pages(u + 1);
        ask_scales();
      }
      const int page_next = __builtin_amdgcn_readlane(pages_of, (at + 1) & 63);
      // (the next unit's loads follow upon the last use of a register; behind the last unit, its own once more)
      const unsigned char *const keys_next = keys_at(more ? u + 1 : u, more ? page_next : page), *const values_next = values_at(more ? u + 1 : u, more ? page_next : page);
      floatx4 s[TILES][kKeyTiles];
#pragma unroll
      for (int kt = 0; kt < kKeyTiles; ++kt) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) s[t][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          const int i = D >= 64 ? step / 2 : 0, w = D >= 64 ? 2 * (step % 2) : 0;
          const uintx4 k = as_halfs<FORMAT>(kk[kt][i][w], kk[kt][i][w + 1]);
#pragma unroll
          for (int t = 0; t < TILES; ++t) s[t][kt] = mfma(k, q[t][step], s[t][kt]);
        }
        load_k(keys_next, kt);
      }
      const int key0 = u * UNIT, key = key0 + UNIT / 4 * g;
      const bool cut = !there || key0 + UNIT > all_seen;  // uniform: some row does not see some key
      float v_scale_of[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const float f = k_scale * c[t];
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; ++kt) s[t][kt] *= f;
        v_scale_of[t] = v_scale;
      }
      if (__builtin_expect(cut, 0)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const int left = there ? seen[t] - key : INT_MIN;
#pragma unroll
          for (int kt = 0; kt < kKeyTiles; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][kt][i] = 4 * kt + i >= left ? -INFINITY : s[t][kt][i];
          // (a row that sees nothing of the page does not see that its scale is NaN either)
          if (!there || key0 >= seen[t]) v_scale_of[t] = 0.f;
        }
      }
      uintx4 pt[TILES][kShares];
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float most = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, s[t][kt][i]);
        most = max_over_rows(most);
        // The reference point moves only when a row's maximum has grown by more than 2^8, and lies 2^7 below it then: fp16 holds 2^15, but loses what is
        // below 2^-25, and many keys of small probabilities are not nothing.  (fp16 for the matrix instructions, as the codes; root mean square errors are 1.0 to 1.3 times those of
        // probabilities in 32 bits.)
        const float new_max = fmaxf(run_max[t], most - 7.0f);
        if (__ballot(new_max - run_max[t] > 8.0f) != 0) {
          const float down = half_way_down(new_max - run_max[t]);
          run_max[t] = new_max;
          run_sum[t] = run_sum[t] * down * down;
#pragma unroll
          for (int part = 0; part < kParts; ++part) o[t][part] = o[t][part] * down * down;
        }
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; ++kt)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float a = __builtin_amdgcn_exp2f(s[t][kt][i] - run_max[t]), b = __builtin_amdgcn_exp2f(s[t][kt][i + 1] - run_max[t]);
            run_sum[t] += a + b;
            pt[t][kt / 2][2 * (kt % 2) + i / 2] = Fp16::pack(a, b);
          }
      }
      // (Nothing: but the compiler of ROCm 7.2 loses half of such a pair of words between here and there, and reuses its register, unless both are
      // wanted at one place.  -verify-machineinstrs finds it; the build asks for that.)
#pragma unroll
      for (int part = 0; part < kParts; ++part) asm volatile("" : "+v"(vv[part]));
      if (FORMAT == 1 && (!there || key0 + UNIT > length)) {  // (what lies behind the sequence, or in no page of it, may be NaN)
#pragma unroll
        for (int w = 0; w < kValueWords; ++w) {
          const int left = there ? max(0, min(4, length - key - 4 * w)) : 0;
          const uint32_t mask = left == 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
#pragma unroll
          for (int part = 0; part < kParts; ++part) vv[part][w] &= mask;
        }
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        floatx4 sum[TILES];
#pragma unroll
        for (int w = 0; w < kShares; ++w) {
          const uintx4 v = as_halfs<FORMAT>(vv[part][2 * w], vv[part][2 * w + 1]);
#pragma unroll
          for (int t = 0; t < TILES; ++t) sum[t] = mfma(v, pt[t][w], w == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : sum[t]);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][part][i] = fmaf(sum[t][i], v_scale_of[t], o[t][part][i]);
        load_v(values_next, part);
      }
      page = page_next;
    }
  }

  // The waves' sums of this workgroup to one reference point for each row, and that and the sums of the exponentials beside them.  Ends with a barrier.
  template <int WAVES>
  __device__ __forceinline__ void join(int wave, float (&state)[WAVES][2][16 * TILES], float (&sums)[WAVES][16 * TILES][D]) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      run_sum[t] = sum_over_rows(run_sum[t]);
      if (g == 0) {
        state[wave][0][16 * t + m] = run_max[t];
        state[wave][1][16 * t + m] = run_sum[t];
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      float most = state[0][0][16 * t + m];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) most = fmaxf(most, state[w][0][16 * t + m]);
      const float down = half_way_down(most - run_max[t]);
#pragma unroll
      for (int part = 0; part < kParts; ++part) *reinterpret_cast<floatx4 *>(&sums[wave][16 * t + m][16 * part + 4 * g]) = o[t][part] * down * down;
    }
    __syncthreads();
  }
  // Features d .. d + 3 of row r over all waves, after that: their sum, its reference point and the sum of its exponentials.
  template <int WAVES>
  __device__ __forceinline__ floatx4 joined(const float (&state)[WAVES][2][16 * TILES], const float (&sums)[WAVES][16 * TILES][D], int r, int d, float &most,
                                            float &total) const {
    most = state[0][0][r];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) most = fmaxf(most, state[w][0][r]);
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      x += *reinterpret_cast<const floatx4 *>(&sums[w][r][d]);
      const float down = half_way_down(most - state[w][0][r]);
      total += state[w][1][r] * down * down;
    }
    return x;
  }
};

// A job by the workgroup.
template <typename T, int FORMAT, int D, int TILES, int UNIT>
__device__ __forceinline__ void work_on(const PrefixAttentionArgs &p, const PrefixPlan &plan, const Job &job, int head, float *lds) {
  typedef float States[kWaves][2][16 * TILES];
  typedef float Sums[kWaves][16 * TILES][D];
  States &state = *reinterpret_cast<States *>(lds + sizeof(Sums) / 4);
  Sums &sums = *reinterpret_cast<Sums *>(lds);
  const int m = threadIdx.x & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads / p.pool.kv_heads, row_queries = p.queries * group;
  CacheRows<T, FORMAT, D, TILES, UNIT> w;
  const auto query = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      // (places behind the last query take that one's: its maxima move no reference point that it does not move itself)
      const int at = job.first + min(16 * t + m, job.count - 1), r = at % row_queries, i = r / group;
      const Ordered row = plan.order[job.member + at / row_queries];
      w.load_query(t, p.q + (long long)row.row * p.q_seq + (long long)i * p.q_row + (long long)(head * group + r % group) * p.q_head, row.length - p.queries + 1 + i);
    }
  };
  const int units = job.unit1 - job.unit0;
  w.attend(p.pool, p.pool.table + (long long)job.row * p.pool.slots, head, job.unit0 + units * wave / kWaves, job.unit0 + units * (wave + 1) / kWaves, job.all_seen, job.end,
           p.scale_log2e, query);
  w.template join<kWaves>(wave, state, sums);
  const long long row = head * p.shape.state_rows + job.states;
  float *const values = p.partial + row * D, *const sums_to = p.partial + p.pool.kv_heads * p.shape.state_rows * D + 2 * row;
  for (int at = threadIdx.x; at < 16 * TILES * D / 4; at += 64 * kWaves) {
    const int r = at / (D / 4), d = (at % (D / 4)) * 4;
    if (r >= job.count) break;
    float most, total;
    const floatx4 x = w.joined(state, sums, r, d, most, total);
    *reinterpret_cast<floatx4 *>(values + r * D + d) = x;
    if (d == 0) {
      sums_to[2 * r] = most;
      sums_to[2 * r + 1] = total;
    }
  }
}

template <typename T, int FORMAT, int D, int UNIT>
__global__ __launch_bounds__(64 * kWaves, 2) void prefix_attention_kernel(const PrefixAttentionArgs p) {
  __shared__ __align__(16) float lds[kWaves * kRows * (D + 2)];
  const PrefixPlan plan(const_cast<int32_t *>(p.plan), p.shape, p.rows);
  const int kv = p.pool.kv_heads, jobs = plan.header[0];
  int number = blockIdx.x / kv, head = blockIdx.x % kv;
  if (kv < 8 && 8 % kv == 0) {
    // Workgroup ids go round-robin to the 8 XCDs: a head's jobs go to 8 / kv of them, one after the other, so that tiles that read the same keys do so through one L2.
    const int parts = 8 / kv, each = (jobs + parts - 1) / parts, xcd = blockIdx.x & 7;
    head = xcd % kv;
    number = (int)(blockIdx.x >> 3) < each ? xcd / kv * each + (int)(blockIdx.x >> 3) : jobs;
  }
  if (number >= jobs) return;
  const Job job = plan.jobs[number];
  if (job.count > 16) work_on<T, FORMAT, D, 2, UNIT>(p, plan, job, head, lds);
  else work_on<T, FORMAT, D, 1, UNIT>(p, plan, job, head, lds);
}

// A workgroup a query and head: its states of the shared pages and of the rest as one.  Their weights (a factor to be taken twice) first, then D / 4 threads for the
// features and 1024 / D sets of them that take every so manyth state.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_attention_join_kernel(const PrefixAttentionArgs p) {
  constexpr int kSets = 1024 / D;
  __shared__ float weights[kMostStates];
  __shared__ __align__(16) float part[kSets][D];
  __shared__ float largest[4], totals[4];
  const PrefixPlan plan(const_cast<int32_t *>(p.plan), p.shape, p.rows);
  const int kv = p.pool.kv_heads, group = p.heads / kv, row_queries = p.queries * group;
  const int h = blockIdx.x % p.heads, i = blockIdx.x / p.heads % p.queries, b = blockIdx.x / p.heads / p.queries;
  const int head = h / group, r = i * group + h % group, tid = threadIdx.x;
  const RowPlan row = plan.rows[b];
  const float *const values = p.partial + head * p.shape.state_rows * D, *const sums = p.partial + (kv * D + 2 * head) * p.shape.state_rows;
  // ---- where they lie
  const int shared_query = row.place * row_queries + r, shared_first = shared_query / kRows * kRows, own_first = r / kRows * kRows;
  const int shared_step = min(kRows, row.shared_queries - shared_first), own_step = min(kRows, row_queries - own_first);
  const long long shared_at = (long long)row.shared_states + shared_first * row.shared_jobs + shared_query % kRows;
  const long long own_at = (long long)row.own_states + own_first * row.own_jobs + r % kRows;
  const int states = row.shared_jobs + row.own_jobs;
  const auto place = [&](int s) { return s < row.shared_jobs ? shared_at + (long long)s * shared_step : own_at + (long long)(s - row.shared_jobs) * own_step; };
  float most = kLowest;
  for (int s = tid; s < states; s += 256) most = fmaxf(most, sums[2 * place(s)]);
  most = wave_max_all(most);
  if ((tid & 63) == 0) largest[tid >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
  float total = 0.f;
  for (int s = tid; s < states; s += 256) {
    const float down = half_way_down(most - sums[2 * place(s)]);
    weights[s] = down;
    total += sums[2 * place(s) + 1] * down * down;
  }
  total = wave_sum_all(total);
  if ((tid & 63) == 0) totals[tid >> 6] = total;
  __syncthreads();
  total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
  const int set = tid / (D / 4), d = (tid % (D / 4)) * 4;
  floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = set; s < states; s += kSets) x += *reinterpret_cast<const floatx4 *>(values + place(s) * D + d) * weights[s] * weights[s];
  *reinterpret_cast<floatx4 *>(&part[set][d]) = x;
  __syncthreads();
  if (set != 0) return;
  for (int j = 1; j < min(kSets, states); ++j) x += *reinterpret_cast<const floatx4 *>(&part[j][d]);
  const float inv = total > 0.f || total != total ? 1.0f / kValueUnit / total : 0.f;
  uint16_t *const to = p.out + (long long)b * p.out_seq + (long long)i * p.out_row + (long long)h * p.out_head + d;
  *reinterpret_cast<uintx2 *>(to) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
}

template <typename T, int FORMAT, int D>
hipError_t launch(const PrefixAttentionArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.shape.jobs * a.pool.kv_heads + 7) / 8 * 8 + 8));  // (each XCD may have one more)
  if (unit_of(a.pool.page_size) == 32) hipLaunchKernelGGL((prefix_attention_kernel<T, FORMAT, D, 32>), grid, dim3(64 * kWaves), 0, stream, a);
  else hipLaunchKernelGGL((prefix_attention_kernel<T, FORMAT, D, 64>), grid, dim3(64 * kWaves), 0, stream, a);
  hipLaunchKernelGGL((prefix_attention_join_kernel<T, D>), dim3((unsigned)(a.rows * a.queries * a.heads)), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <typename T, int FORMAT>
hipError_t launch(const PrefixAttentionArgs &a, hipStream_t stream) {
  return a.pool.d == 128 ? launch<T, FORMAT, 128>(a, stream) : a.pool.d == 64 ? launch<T, FORMAT, 64>(a, stream) : launch<T, FORMAT, 32>(a, stream);
}

}  // namespace

PrefixShape prefix_shape(int rows, int queries, int heads, int kv_heads) {
  PrefixShape s;
  s.row_queries = queries * (heads / kv_heads);
  // own tiles; shared ones, full but for one in a group of two rows or more
  s.tiles = (long long)rows * ((s.row_queries + kRows - 1) / kRows) + (long long)rows * s.row_queries / kRows + rows / 2;
  s.target = max(1, kPlaces / kv_heads);
  s.jobs = s.tiles + kMostRounds * s.target;  // (a tile of n units has fewer than n / size + 1, and all tiles' n / size are that many rounds of places at most)
  // a job's queries, 32 at most, are a tile's, and all tiles' no more than twice the rows'
  s.state_rows = 2ll * rows * s.row_queries + (long long)kMostRounds * s.target * kRows;
  return s;
}
size_t prefix_plan_ints(const PrefixShape &shape, int rows) { return (size_t)PrefixPlan(nullptr, shape, rows).words(rows); }
size_t prefix_attention_floats(const PrefixShape &shape, int kv_heads, int d) {
  return (size_t)kv_heads * (size_t)shape.state_rows * (d + 2);
}

hipError_t launch_plan_prefixes(const PrefixShape &shape, const int32_t *table, int rows, int slots, const int32_t *lengths, int page_size, int queries, int32_t *plan,
                                hipStream_t stream) {
  const PrefixPlan at(plan, shape, rows);
  const bool few = rows <= kFewRows;
  if (!few) hipLaunchKernelGGL(plan_prefixes_compare_kernel, dim3(rows), dim3(64 * kCompareWaves), 0, stream, at, table, rows, slots, lengths, page_size, queries);
  hipLaunchKernelGGL(plan_prefixes_kernel, dim3(1), dim3(few ? max(256, 64 * rows) : max(256, (rows + 63) / 64 * 64)), 0, stream, at, few ? table : nullptr, rows, slots, lengths,
                     page_size, queries, shape);
  return hipGetLastError();
}

hipError_t launch_prefix_attention(int type, int format, const PrefixAttentionArgs &a, hipStream_t stream) {
  if (type == 0) return format == 0 ? launch<Fp16, 0>(a, stream) : launch<Fp16, 1>(a, stream);
  return format == 0 ? launch<Bf16, 0>(a, stream) : launch<Bf16, 1>(a, stream);
}

}  // namespace sspmm
