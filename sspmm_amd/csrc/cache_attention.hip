// Attention of the newest tokens of every sequence over its paged cache in 8 bits:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^((q . k_j) scale log2(e) - m),  k_j and v_j codes times their block's scale.
// Bound by the cache's bytes, each read once: a wave's loads go from memory to the registers that the products read.  64 rows of 4000 tokens, 32 heads on
// 8 of 128 features, int8 101 us, 5.2 TB/s (caches that are in no cache of the chip's); of 64 to 4063 tokens 52 us, 4.5 TB/s: with two workgroups a CU a unit of 64
// keys is some 1.4 us of a wave's instructions (half of them make fp16 of the codes) behind 10 us of launch, look-ups and joining, which short rows
// pay for (256 rows of 450 tokens 69 us, 3.4 TB/s).  Tried without gain: two units' loads ahead (52 -> 58 us, a wave has no time to spare for
// them), units of 32 keys, three workgroups a CU (eleven spilled registers, 65 us), non-temporal loads.
#include "cache_kernels.h"

#include "cache_codes.h"

namespace sspmm {

namespace {

constexpr int kMostSplits = 256;

// The sequence that a workgroup takes: of 64 consecutive ones the longest go first, where there are more workgroups than CUs; but of those that become
// the CUs' second ones the shortest, so that a CU that has begun on the longest gets the least beside it (64 rows of 64 to 4063 tokens, 8 heads of the
// cache: 57.0 -> 52.3 us).
__device__ __forceinline__ int longest_first(const int32_t *lengths, int sequences) {
  const int z = blockIdx.z, each = gridDim.x * gridDim.y;
  if (each * gridDim.z <= 256 || sequences == 1) return z;
  const int lane = threadIdx.x & 63, first = z & ~63, count = min(64, sequences - first);
  const int round = 256 / each, end = min(2 * round, count);  // sequences in a round of the CUs, in both of the first
  const int place = z >= round && z < end ? round + end - 1 - z : z - first;
  const int mine = lane < count ? lengths[first + lane] : -1;
  int rank = lane < count ? 0 : 64;
  for (int j = 0; j < count; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    rank += other > mine || (other == mine && j < lane);
  }
  return first + __builtin_ctzll(__ballot(rank == place));
}

__device__ __forceinline__ long long partial_floats(int rows, int d) { return (long long)rows * (d + 2); }

// A workgroup owns 16 * TILES rows (queries x heads of one head of the cache; row i * group + j is query i, head j of the group) of one
// sequence and one of its `splits` shares of the keys, a wave its part of those, UNIT keys at a time, all of them in one page.  Scores are
// made transposed, K Q^T: the lane of row m and group g holds keys UNIT / 4 * g .. of the unit, which is the operand of the second product
// V^T P^T as it is, and the order in which values lie in a page.
template <typename T, int FORMAT, int D, int TILES, int UNIT, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 2) void cache_attention_kernel(const CacheAttentionArgs p) {
  constexpr int kKeyTiles = UNIT / 16, kParts = D / 16, kSteps = D / 32, kShares = UNIT / 32, kRows = 16 * TILES;
  constexpr int kKeyWords = D >= 64 ? 4 : 2;  // of a load of K: 16 bytes, or 8 where a group's share of a row is no more
  constexpr int kKeyLoads = D / (16 * kKeyWords);  // of a row by a lane
  constexpr int kValueWords = UNIT / 16;
  typedef uint32_t KeyWords __attribute__((ext_vector_type(kKeyWords)));
  typedef uint32_t ValueWords __attribute__((ext_vector_type(kValueWords)));
  __shared__ float state[kWaves][2][kRows];
  __shared__ __align__(16) float sums[kWaves][kRows][D];
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const CachePool pool = p.pool;
  const int group = p.heads / pool.kv_heads, rows = p.queries * group, tiles = (rows + kRows - 1) / kRows;
  const int split = blockIdx.y, head = blockIdx.x % pool.kv_heads, tile = blockIdx.x / pool.kv_heads;
  const int seq = longest_first(p.lengths, p.sequences);
  // (tokens that the table has no slot for are nowhere, but the queries' positions count them)
  const int all_length = max(0, p.lengths[seq]), length = (int)min((long long)all_length, (long long)pool.slots * pool.page_size);
  const int units = (length + UNIT - 1) / UNIT, pieces = p.splits * kWaves, piece = split * kWaves + wave;
  const int unit0 = (int)((long long)units * piece / pieces), unit1 = (int)((long long)units * (piece + 1) / pieces);

  // ---- queries.  bf16 goes to fp16 by way of a power of two for the row, which leaves its largest magnitude in 2^14 .. 2^15
  uintx4 q[TILES][kSteps];
  float c[TILES];
  int seen[TILES];  // keys that the row sees: those below
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    // (Places behind the last row take that one's query: it lies in the workgroup's own tile, since out may be q and others write theirs while this reads, and
    // its maxima move no reference point that it does not move itself.)
    const int r = min(tile * kRows + 16 * t + m, rows - 1), i = r / group;
    seen[t] = all_length - p.queries + 1 + i;
    const uint16_t *const at = p.q + (long long)seq * p.q_seq + (long long)i * p.q_row + (long long)(head * group + r % group) * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = D >= 64 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 8 * g;
      q[t][s] = *reinterpret_cast<const uintx4 *>(at + d);
    }
    c[t] = p.scale_log2e;
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

  floatx4 o[TILES][kParts];  // features 16 part + 4 g + i of row m
  float run_max[TILES], run_sum[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    run_max[t] = kLowest;
    run_sum[t] = 0.f;
#pragma unroll
    for (int part = 0; part < kParts; ++part) o[t][part] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t *const table = p.pool.table + (long long)seq * pool.slots;
  const long long block = (long long)pool.page_size * D;
  KeyWords kk[kKeyTiles][kKeyLoads];
  ValueWords vv[kParts];
  const int page_units = pool.page_size / UNIT, page_bits = 31 - __builtin_clz(page_units);  // (1 or 2)
  const auto place_of = [&](int u) { return (u & (page_units - 1)) * UNIT; };  // in its page
  const auto usable = [&](int pg) { return pg >= 0 && pg < pool.pages; };
  // Pages and scales of 64 units at a time, one a lane, so that no unit waits for them.
  int pages_of = 0;
  float k_scales = 0.f, v_scales = 0.f;
  const auto look_up = [&](int u) {
    const int mine = min(u + lane, unit1 - 1);
    pages_of = table[mine >> page_bits];
    const float *const scale = pool.scales + (long long)(usable(pages_of) ? pages_of : 0) * 2 * pool.kv_heads + head;
    k_scales = scale[0];
    v_scales = scale[pool.kv_heads] * kValueUnit;
  };
  const auto load_k = [&](int u, int pg) {
    const unsigned char *const at = pool.keys + ((long long)(usable(pg) ? pg : 0) * pool.kv_heads + head) * block + place_of(u) * D;
#pragma unroll
    for (int kt = 0; kt < kKeyTiles; ++kt) {
      const unsigned char *const row = at + (UNIT / 4 * (m >> 2) + 4 * kt + (m & 3)) * D + 4 * kKeyWords * g;
#pragma unroll
      for (int i = 0; i < kKeyLoads; ++i) {
        kk[kt][i] = *reinterpret_cast<const KeyWords *>(row + 64 * i);
      }
    }
  };
  const auto load_v = [&](int u, int pg) {
    const unsigned char *const at = pool.values + ((long long)(usable(pg) ? pg : 0) * pool.kv_heads + head) * block + place_of(u) + UNIT / 4 * g;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const unsigned char *const row = at + (16 * part + m) * pool.page_size;
      vv[part] = *reinterpret_cast<const ValueWords *>(row);
    }
  };

  int page = 0;
  if (unit0 < unit1) {
    look_up(unit0);
    page = __builtin_amdgcn_readlane(pages_of, 0);
    load_k(unit0, page);
    load_v(unit0, page);
  }
  for (int u = unit0; u < unit1; ++u) {
    const bool more = u + 1 < unit1, there = usable(page);
    const int at = (u - unit0) & 63;
    const float k_scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k_scales), at));
    const float v_scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_scales), at));
    if (at == 63 && more) look_up(u + 1);
    const int page_next = __builtin_amdgcn_readlane(pages_of, (at + 1) & 63);
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
    }
    if (more) load_k(u + 1, page_next);
    const int key0 = u * UNIT, key = key0 + UNIT / 4 * g;
    const bool cut = !there || key0 + UNIT > all_length - p.queries + 1;  // uniform: some row does not see some key
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
      // below 2^-25, and many keys of small probabilities are not nothing.
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
    }
    if (more) load_v(u + 1, page_next);
    page = page_next;
  }

  // ---- the waves' states as one
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
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, state[w][0][16 * t + m]);
    const float down = half_way_down(most - run_max[t]);
#pragma unroll
    for (int part = 0; part < kParts; ++part) *reinterpret_cast<floatx4 *>(&sums[wave][16 * t + m][16 * part + 4 * g]) = o[t][part] * down * down;
  }
  __syncthreads();
  const int r0 = tile * kRows;
  float *const partial =
      p.splits > 1 ? p.partial + ((((long long)seq * pool.kv_heads + head) * tiles + tile) * p.splits + split) * partial_floats(kRows, D) : nullptr;
  for (int at = threadIdx.x; at < kRows * D / 4; at += 64 * kWaves) {
    const int r = at / (D / 4), d = (at % (D / 4)) * 4, row = r0 + r;
    if (row >= rows) continue;
    float most = state[0][0][r], total = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, state[w][0][r]);
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      x += *reinterpret_cast<const floatx4 *>(&sums[w][r][d]);
      const float down = half_way_down(most - state[w][0][r]);
      total += state[w][1][r] * down * down;
    }
    if (partial) {
      *reinterpret_cast<floatx4 *>(partial + (long long)r * D + d) = x;
      if (d == 0) {
        partial[(long long)kRows * D + r] = most;
        partial[(long long)kRows * D + kRows + r] = total;
      }
    } else {
      const float inv = total > 0.f || total != total ? 1.0f / kValueUnit / total : 0.f;
      const int i = row / group, h = head * group + row % group;
      uint16_t *const to = p.out + (long long)seq * p.out_seq + (long long)i * p.out_row + (long long)h * p.out_head + d;
      *reinterpret_cast<uintx2 *>(to) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
    }
  }
}

// The splits' states of one row as one: their weights (a factor to be taken twice) first, then D / 4 threads for the features and 1024 / D sets of them that take every so
// manyth split.  A launch of its own, 4.5 us for 64 splits of 16 rows: three dependent loads and two barriers.
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attention_join_kernel(const CacheAttentionArgs p, int row_tiles) {
  constexpr int kSets = 1024 / D;
  __shared__ float weights[kMostSplits];
  __shared__ __align__(16) float part[kSets][D];
  __shared__ float largest[4], totals_of[4];
  const int kRows = 16 * row_tiles, group = p.heads / p.pool.kv_heads, rows = p.queries * group, tiles = (rows + kRows - 1) / kRows;
  const int row = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, tile = row / kRows, r = row % kRows, tid = threadIdx.x;
  const long long pitch = partial_floats(kRows, D);
  const float *const base = p.partial + (((long long)seq * p.pool.kv_heads + head) * tiles + tile) * p.splits * pitch;
  const float *const own = base + (long long)kRows * D + r;
  // (a split a thread: there are no more than 256)
  const bool mine = tid < p.splits;
  const float max_here = mine ? own[tid * pitch] : kLowest, sum_here = mine ? own[tid * pitch + kRows] : 0.f;
  float most = wave_max_all(max_here);
  if ((tid & 63) == 0) largest[tid >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
  const float down = half_way_down(most - max_here);
  if (mine) weights[tid] = down;
  const float sum = wave_sum_all(mine ? sum_here * down * down : 0.f);
  if ((tid & 63) == 0) totals_of[tid >> 6] = sum;
  __syncthreads();
  const float total = (totals_of[0] + totals_of[1]) + (totals_of[2] + totals_of[3]);
  const int set = tid / (D / 4), d = (tid % (D / 4)) * 4;
  floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = set; s < p.splits; s += kSets) x += *reinterpret_cast<const floatx4 *>(base + s * pitch + (long long)r * D + d) * weights[s] * weights[s];
  *reinterpret_cast<floatx4 *>(&part[set][d]) = x;
  __syncthreads();
  if (set != 0) return;
  for (int i = 1; i < kSets; ++i) x += *reinterpret_cast<const floatx4 *>(&part[i][d]);
  const float inv = total > 0.f || total != total ? 1.0f / kValueUnit / total : 0.f;
  const int i = row / group, h = head * group + row % group;
  uint16_t *const to = p.out + (long long)seq * p.out_seq + (long long)i * p.out_row + (long long)h * p.out_head + d;
  *reinterpret_cast<uintx2 *>(to) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
}

// Rows of the largest tiles, workgroups for the rows and heads, waves of one, and shares of the keys.
//
// Long rows that are few are split, as far as every CU has a workgroup, in shares of 512 keys or more; the join has to be earned: 128 workgroups (16 rows, 8 heads of
// 128 features) split in two 2500 tokens 27.8 -> 24.3 us, 4000 38 -> 32, 8000 68 -> 56, 16 rows of 64 to 4000 33 -> 26; 192 workgroups of 4000 tokens 41 -> 50: up to
// 128, and where rows have room for more than 2048 (one row of 131009 tokens, 4 heads: 64 splits best).
// Eight waves a workgroup where there are few and nothing is split: eight rows of 3 to 1500 tokens, 12 heads of 64 features 13.0 -> 11.1 us; 64 rows of 2000, 8 heads
// of 128 48 -> 56 us (one workgroup a CU has room), eight of 100 4.9 -> 6.1.
// The host does not know the lengths, only the table's room for them: a row of 100 tokens takes 5.8 us with a table of two pages and 9.1 with one of 4096 positions
// or more, where most shares are empty and are joined all the same; and a long row among many is not split: 131009 tokens, 4 heads of the cache, 28 us alone, 378 with
// 31 rows of 200 beside it (two shares), 740 with 32.
struct Shape {
  int row_tiles, tiles, waves, splits;
};
Shape shape_of(int sequences, int queries, int heads, int kv_heads, long long longest) {
  Shape s;
  const int rows = queries * (heads / kv_heads);
  s.row_tiles = rows > 16 ? 2 : 1;
  s.tiles = (rows + 16 * s.row_tiles - 1) / (16 * s.row_tiles);
  const long long wide = (long long)sequences * kv_heads * s.tiles;
  const bool whole = wide > 128 || longest <= 2048;
  s.waves = whole && wide <= 128 && longest > 512 ? 8 : 4;
  s.splits = whole ? 1 : (int)max(1ll, min(min((256 + wide - 1) / wide, (longest + 511) / 512), (long long)kMostSplits));
  return s;
}

template <typename T, int FORMAT, int D, int TILES, int UNIT>
void launch(const CacheAttentionArgs &a, const Shape &s, const dim3 &grid, hipStream_t stream) {
  if (s.waves == 8) hipLaunchKernelGGL((cache_attention_kernel<T, FORMAT, D, TILES, UNIT, 8>), grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL((cache_attention_kernel<T, FORMAT, D, TILES, UNIT, 4>), grid, dim3(256), 0, stream, a);
}

template <typename T, int FORMAT, int D>
hipError_t launch(const CacheAttentionArgs &a, const Shape &s, hipStream_t stream) {
  const dim3 grid(a.pool.kv_heads * s.tiles, a.splits, a.sequences);
  if (a.pool.page_size == 32) {
    if (s.row_tiles == 1) launch<T, FORMAT, D, 1, 32>(a, s, grid, stream);
    else launch<T, FORMAT, D, 2, 32>(a, s, grid, stream);
  } else {
    if (s.row_tiles == 1) launch<T, FORMAT, D, 1, 64>(a, s, grid, stream);
    else launch<T, FORMAT, D, 2, 64>(a, s, grid, stream);
  }
  if (a.splits > 1)
    hipLaunchKernelGGL((cache_attention_join_kernel<T, D>), dim3(a.queries * (a.heads / a.pool.kv_heads), a.pool.kv_heads, a.sequences), dim3(256), 0, stream, a,
                       s.row_tiles);
  return hipGetLastError();
}

template <typename T, int FORMAT>
hipError_t launch(const CacheAttentionArgs &a, const Shape &s, hipStream_t stream) {
  return a.pool.d == 128 ? launch<T, FORMAT, 128>(a, s, stream) : a.pool.d == 64 ? launch<T, FORMAT, 64>(a, s, stream) : launch<T, FORMAT, 32>(a, s, stream);
}

}  // namespace

size_t cache_attention_workspace(int sequences, int queries, int heads, int kv_heads, int d, long long longest) {
  const Shape s = shape_of(sequences, queries, heads, kv_heads, longest);
  return s.splits <= 1 ? 0 : (size_t)sequences * kv_heads * s.tiles * s.splits * (size_t)(16 * s.row_tiles) * (d + 2);
}

hipError_t launch_cache_attention(int type, int format, CacheAttentionArgs a, hipStream_t stream) {
  const Shape s = shape_of(a.sequences, a.queries, a.heads, a.pool.kv_heads, (long long)a.pool.slots * a.pool.page_size);
  a.splits = s.splits;
  if (type == 0) return format == 0 ? launch<Fp16, 0>(a, s, stream) : launch<Fp16, 1>(a, s, stream);
  return format == 0 ? launch<Bf16, 0>(a, s, stream) : launch<Bf16, 1>(a, s, stream);
}

}  // namespace sspmm
