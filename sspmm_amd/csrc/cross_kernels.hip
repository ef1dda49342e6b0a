// Attention of a sequence's few queries, a token's as a rule, over its packed states in 16 bits:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^((q . k_j - m) scale log2(e)).
// Bound by the bytes of k and v, each read once for all queries and heads of a group: a token of each of 64 sequences on 50 to 2000 states, 32 heads on 8 of 128, bf16 (276 MB), 57 us, 4.8 TB/s, again and
// again (the last-level cache has a part of it), 70 us, 4.0 TB/s, where nothing is cached.  Four tokens on 40 states or fewer, 4 heads of 64, 4.6 us: the launch and its chain of look-ups.
#include "prompt_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

#include <type_traits>

namespace sspmm {

namespace {

constexpr int kUnit = 32;  // keys of a unit
constexpr int kWaves = 4;
constexpr int kMostSplits = 64;

// Pieces of 16 bytes of V's row r lie at place piece ^ swizzle(r): the transpose reads take 32 bytes of each of eight consecutive rows at a time, which then fall on all banks.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return (r / (128 / D) & (D / 16 - 1)) * 2;
}

// Where a workgroup works: tile number `tile` of the packed queries.  Numbers offsets[b] * group / kRows + b .. are sequence b's, enough for its tiles however it lies.
struct Tile {
  int first, rows, row0;     // the sequence's first query; queries x heads of the group; the tile's first of these
  int key_first, keys;
};
template <int kRows>
__device__ __forceinline__ bool tile_of(const PromptArgs &p, int group, int tile, Tile &t) {
  const auto base = [&](int b) { return (int)((long long)max(0, min(p.offsets[b], p.tokens)) * group / kRows) + b; };
  const int b = __builtin_amdgcn_readfirstlane(last_not_above(p.sequences, tile, base));
  t.first = max(0, min(p.offsets[b], p.tokens));
  t.rows = (max(t.first, min(p.offsets[b + 1], p.tokens)) - t.first) * group;
  t.row0 = (tile - base(b)) * kRows;
  t.key_first = max(0, min(p.key_offsets[b], p.key_tokens));
  t.keys = max(t.key_first, min(p.key_offsets[b + 1], p.key_tokens)) - t.key_first;
  return t.row0 >= 0 && t.row0 < t.rows;
}

__device__ __forceinline__ long long state_floats(int rows, int d) { return (long long)rows * (d + 2); }

// A workgroup owns 16 * TILES rows (row i * group + j is query i, head j of a group) of a sequence and a head of k and v, and one of `splits` shares of its keys; a wave
// a part of these, 32 keys at a time.  Scores are made transposed, K Q^T (16 x 16 x 32 instructions), K from memory to the registers as the instruction takes it; lane
// (m, g) then holds keys 4 g .. 4 g + 3 and 16 + 4 g .. of row m, which is the operand P^T of V^T P^T.  V^T comes from transpose reads of the unit's V, which the wave has put into its own
// piece of LDS: no wave waits for another before its keys are done.  The next unit's K and V are on their way meanwhile.
template <typename T, int D, int TILES>
__global__ __launch_bounds__(64 * kWaves, 2) void cross_step_kernel(const PromptArgs p, int splits, float *partial) {
  constexpr int kRows = 16 * TILES, kSteps = D / 32, kParts = D / 16, kPieces = D / 8, kLoads = kUnit * kPieces / 64;
  // fp16 loses what is below 2^-25, and many keys of small probabilities are not nothing: their largest is 2^7 or more there.  bf16 does not, but its v may be as large as
  // 32 bits hold: probabilities are 2^-16 at most, and 2^16 keys' sum does not overflow (v below 2^-102 loses what is then below 2^-149).  In 16 bits the second product is a matrix
  // instruction's, as in the package's other attentions; root mean square errors are 1.0 to 1.3 (fp16) and 1.2 to 1.41 (bf16) times those of probabilities in 32 bits.
  constexpr float kHeadroom = __is_same(T, Fp16) ? 7.f : -24.f;
  constexpr int kTileBytes = kUnit * D * 2;
  typedef float Sums[kWaves][kRows][D];
  __shared__ __align__(16) unsigned char lds[sizeof(Sums) > kWaves * kTileBytes ? sizeof(Sums) : kWaves * kTileBytes];
  __shared__ float state[kWaves][2][kRows];
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads / p.kv_heads, head = blockIdx.x % p.kv_heads, split = blockIdx.x / p.kv_heads % splits, number = blockIdx.x / p.kv_heads / splits;
  Tile tile;
  if (!tile_of<kRows>(p, group, number, tile)) return;
  const int units = (tile.keys + kUnit - 1) / kUnit, pieces = splits * kWaves, piece = split * kWaves + wave;
  const int unit0 = (int)((long long)units * piece / pieces), unit1 = (int)((long long)units * (piece + 1) / pieces);

  uintx4 q[TILES][kSteps];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    // (places behind the last row take that one's query, which lies in the workgroup's own tile: out may be q)
    const int r = min(tile.row0 + 16 * t + m, tile.rows - 1), i = r / group;
    const uint16_t *const at = p.q + (long long)(tile.first + i) * p.q_row + (long long)(head * group + r % group) * p.q_head + 8 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[t][s] = *reinterpret_cast<const uintx4 *>(at + 32 * s);
  }

  const uint16_t *const k0 = p.k + (long long)tile.key_first * p.k_row + (long long)head * p.k_head;
  const uint16_t *const v0 = p.v + (long long)tile.key_first * p.v_row + (long long)head * p.v_head;
  unsigned char *const own = lds + wave * kTileBytes;
  uintx4 kk[2][kSteps], vv[kLoads];
  const auto load = [&](int u) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint16_t *const row = k0 + (long long)min(u * kUnit + 16 * kt + m, tile.keys - 1) * p.k_row + 8 * g;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kk[kt][s] = *reinterpret_cast<const uintx4 *>(row + 32 * s);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * 64 + lane, r = at / kPieces, c = at % kPieces;
      vv[i] = *reinterpret_cast<const uintx4 *>(v0 + (long long)min(u * kUnit + r, tile.keys - 1) * p.v_row + 8 * c);
    }
  };

  floatx4 o[TILES][kParts];  // features 16 part + 4 g + i of row m
  float run_max[TILES], run_sum[TILES];  // of the scores themselves; this lane's share of the sum
  const float c = p.scale_log2e;
  const auto pass = [&](auto again_) __attribute__((always_inline)) {
    constexpr bool again = decltype(again_)::value;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      run_max[t] = kLowest;
      run_sum[t] = 0.f;
#pragma unroll
      for (int part = 0; part < kParts; ++part) o[t][part] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (unit0 < unit1) load(unit0);
    for (int u = unit0; u < unit1; ++u) {
      const int left = tile.keys - u * kUnit;  // keys of the unit that there are
      floatx4 s[TILES][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          s[t][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int step = 0; step < kSteps; ++step) s[t][kt] = T::mfma_16x16x32(kk[kt][step], q[t][step], s[t][kt]);
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = i * 64 + lane, r = at / kPieces, piece = at % kPieces;
        *reinterpret_cast<uintx4 *>(own + r * (2 * D) + ((piece ^ swizzle<D>(r)) * 16)) = r < left ? vv[i] : uintx4{0, 0, 0, 0};
      }
      __builtin_amdgcn_wave_barrier();
      if (u + 1 < unit1) load(u + 1);
      if (left < kUnit) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][kt][i] = 16 * kt + 4 * g + i >= left ? -INFINITY : s[t][kt][i];
      }
      uintx4 pt[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float most = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, s[t][kt][i]);
        // The reference point moves only when some row's maximum has grown by more than 2^8.
        const float new_max = fmaxf(run_max[t], max_over_rows(most)), grown = (new_max - run_max[t]) * c;
        if (__ballot(grown > 8.0f) != 0) {
          const float down = half_way_down(grown);
          run_max[t] = new_max;
          run_sum[t] = run_sum[t] * down * down;
#pragma unroll
          for (int part = 0; part < kParts; ++part) o[t][part] = o[t][part] * down * down;
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            // (differences before they are scaled: scores of 2^27 leave no more than their own rounding)
            const float a = __builtin_amdgcn_exp2f(fmaf(s[t][kt][i] - run_max[t], c, kHeadroom));
            const float b = __builtin_amdgcn_exp2f(fmaf(s[t][kt][i + 1] - run_max[t], c, kHeadroom));
            run_sum[t] += a + b;
            pt[t][2 * kt + i / 2] = T::pack(a, b);
          }
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const int r = 4 * g + (m >> 2);  // (16 rows on: the same swizzle)
        const unsigned char *const at = own + r * (2 * D) + (((2 * part + ((m & 3) >> 1)) ^ swizzle<D>(r)) * 16) + (m & 1) * 8;
        const uintx2 lo = lds_read_tr(at), hi = lds_read_tr(at + 16 * (2 * D));
        uintx4 v = {lo[0], lo[1], hi[0], hi[1]};
        if constexpr (again) v = finite_part<T>(v);
#pragma unroll
        for (int t = 0; t < TILES; ++t) o[t][part] = T::mfma_16x16x32(v, pt[t], o[t][part]);
      }
      if constexpr (again) {
#pragma unroll 1
        for (int r = 0; r < kUnit; ++r)
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const uintx2 v = *reinterpret_cast<const uintx2 *>(own + r * (2 * D) + (((2 * part + (g >> 1)) ^ swizzle<D>(r)) * 16) + (g & 1) * 8);
            const float x[4] = {T::lower(v[0]), T::upper(v[0]), T::lower(v[1]), T::upper(v[1])};
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][part][i] += fabsf(x[i]) < INFINITY ? 0.f : x[i];
          }
      }
    }
  };
  pass(std::integral_constant<bool, false>{});
  // What is infinite in v, or NaN, reaches every row, also where its probability is nothing in 16 bits: a wave that finds a result which is not finite goes over its keys again, with
  // zeros in the place of these values, which are then added.
  float zero = 0.f;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
      for (int i = 0; i < 4; ++i) zero = fmaf(o[t][part][i], 0.f, zero);
  if (__builtin_expect(__ballot(zero != zero) != 0, 0)) pass(std::integral_constant<bool, true>{});

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
  Sums &sums = *reinterpret_cast<Sums *>(lds);
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    float most = state[0][0][16 * t + m];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, state[w][0][16 * t + m]);
    const float down = half_way_down((most - run_max[t]) * c);
#pragma unroll
    for (int part = 0; part < kParts; ++part) *reinterpret_cast<floatx4 *>(&sums[wave][16 * t + m][16 * part + 4 * g]) = o[t][part] * down * down;
  }
  __syncthreads();
  float *const to = splits > 1 ? partial + (((long long)number * p.kv_heads + head) * splits + split) * state_floats(kRows, D) : nullptr;
  for (int at = threadIdx.x; at < kRows * D / 4; at += 64 * kWaves) {
    const int r = at / (D / 4), d = (at % (D / 4)) * 4, row = tile.row0 + r;
    if (row >= tile.rows) continue;
    float most = state[0][0][r], total = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, state[w][0][r]);
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      x += *reinterpret_cast<const floatx4 *>(&sums[w][r][d]);
      const float down = half_way_down((most - state[w][0][r]) * c);
      total += state[w][1][r] * down * down;
    }
    if (to) {
      *reinterpret_cast<floatx4 *>(to + (long long)r * D + d) = x;
      if (d == 0) {
        to[(long long)kRows * D + r] = most;
        to[(long long)kRows * D + kRows + r] = total;
      }
    } else {
      const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
      const int i = row / group, h = head * group + row % group;
      uint16_t *const out = p.out + (long long)(tile.first + i) * p.out_row + (long long)h * p.out_head + d;
      *reinterpret_cast<uintx2 *>(out) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
    }
  }
}

// The shares' states of a tile's rows as one where they are few: D / 4 threads a row.
template <typename T, int D, int TILES>
__global__ __launch_bounds__(256) void cross_join_kernel(const PromptArgs p, int splits, const float *partial) {
  constexpr int kRows = 16 * TILES;
  const int group = p.heads / p.kv_heads, head = blockIdx.x % p.kv_heads, number = blockIdx.x / p.kv_heads;
  Tile tile;
  if (!tile_of<kRows>(p, group, number, tile)) return;
  const float *const from = partial + ((long long)number * p.kv_heads + head) * splits * state_floats(kRows, D);
  const float c = p.scale_log2e;
  for (int at = threadIdx.x; at < kRows * D / 4; at += 256) {
    const int r = at / (D / 4), d = (at % (D / 4)) * 4, row = tile.row0 + r;
    if (row >= tile.rows) return;
    float most = kLowest, total = 0.f;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float *const state = from + s * state_floats(kRows, D);
      const float theirs = state[(long long)kRows * D + r], sum = state[(long long)kRows * D + kRows + r];
      const floatx4 values = *reinterpret_cast<const floatx4 *>(state + (long long)r * D + d);
      const float new_most = fmaxf(most, theirs), down = half_way_down((new_most - most) * c), their_down = half_way_down((new_most - theirs) * c);
      total = total * down * down + sum * their_down * their_down;
      x = x * down * down + values * their_down * their_down;
      most = new_most;
    }
    const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
    const int i = row / group, h = head * group + row % group;
    uint16_t *const out = p.out + (long long)(tile.first + i) * p.out_row + (long long)h * p.out_head + d;
    *reinterpret_cast<uintx2 *>(out) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
  }
}

// Where they are many, a workgroup a row: their weights (a factor to be taken twice) first, a share a lane, then D / 4 threads for the features and 1024 / D sets of them that take
// every so manyth share.  (16 tokens on 16000 keys, 16 heads on 2, 64 shares: 59 us by the one above, 23 by this; 64 tokens on 1500 keys each, two shares: 86 and 95.)
template <typename T, int D, int TILES>
__global__ __launch_bounds__(256) void cross_join_many_kernel(const PromptArgs p, int splits, const float *partial) {
  constexpr int kRows = 16 * TILES, kSets = 1024 / D;
  __shared__ float weights[kMostSplits];
  __shared__ __align__(16) float part[kSets][D];
  const int group = p.heads / p.kv_heads, r = blockIdx.x % kRows, head = blockIdx.x / kRows % p.kv_heads, number = blockIdx.x / kRows / p.kv_heads;
  Tile tile;
  if (!tile_of<kRows>(p, group, number, tile) || tile.row0 + r >= tile.rows) return;
  const float *const from = partial + ((long long)number * p.kv_heads + head) * splits * state_floats(kRows, D);
  const int tid = threadIdx.x, lane = tid & 63, set = tid / (D / 4), d = (tid % (D / 4)) * 4;
  const float *const own = from + (long long)lane * state_floats(kRows, D) + (long long)kRows * D + r;
  const float max_here = lane < splits ? own[0] : kLowest, sum_here = lane < splits ? own[kRows] : 0.f;
  const float down = half_way_down((wave_max_all(max_here) - max_here) * p.scale_log2e);
  const float total = wave_sum_all(sum_here * down * down);
  if (tid < splits) weights[tid] = down;
  __syncthreads();
  floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = set; s < splits; s += kSets) x += *reinterpret_cast<const floatx4 *>(from + s * state_floats(kRows, D) + (long long)r * D + d) * weights[s] * weights[s];
  *reinterpret_cast<floatx4 *>(&part[set][d]) = x;
  __syncthreads();
  if (set != 0) return;
  for (int i = 1; i < kSets; ++i) x += *reinterpret_cast<const floatx4 *>(&part[i][d]);
  const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
  const int row = tile.row0 + r, i = row / group, h = head * group + row % group;
  uint16_t *const out = p.out + (long long)(tile.first + i) * p.out_row + (long long)h * p.out_head + d;
  *reinterpret_cast<uintx2 *>(out) = uintx2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
}

// Rows of the tiles (0: the prompts' kernel), how many there may be, and shares of the keys.
//
// The prompts' kernel takes 128 queries of a head a workgroup, and goes over a sequence's keys at 18 ns a key with 128 features (11 with 64, 8 with 32), as
// long as there is one workgroup a CU; this one reads k and v once for 32 rows or 16, at 4.8 TB/s, and some 4 us more where shares are joined.  The shorter estimate is taken,
// of the mean lengths, which are what the host knows.  us, this kernel and that: 64 sequences of a token on 1500 keys, 32 heads on 8 of 128 features, 78 and 235; 16 of
// 16 tokens 40 and 64, 8 of 32 33 and 31, 8 of 64 40 and 32; one of 64 on 16000 keys, 16 heads on 2, 36 and 207; two of 100 on 4000, 8 heads of 64, 17 and 40; 8 of 32
// on 512, 12 heads of 64, 14 and 10; 32 of one 16 and 14.
// A sequence that is many times longer than the mean has as few shares as the others: a token of each of 64 sequences, one on 65536 states and the others on 100, 798 us (alone 51); on 16000 145 (22).
// Shares are of 256 keys or more (of 128: four of one token on 8000 keys 46 us instead of 42), as many as fill the 512 places for workgroups, or a few times as many where the last round
// of them would leave more than a tenth of the places empty.
struct Shape {
  int row_tiles, splits;
  long long tiles;
};
Shape shape_of(int sequences, int tokens, int key_tokens, int heads, int kv_heads, int d) {
  const int group = heads / kv_heads;
  const long long rows = (long long)tokens * group, live = min((long long)sequences, (long long)tokens), mean = (rows + live - 1) / live, keys = key_tokens / sequences;
  Shape s;
  s.row_tiles = mean > 16 ? 2 : 1;
  s.tiles = rows / (16 * s.row_tiles) + sequences;
  const long long wide = live * ((mean + 16 * s.row_tiles - 1) / (16 * s.row_tiles)) * kv_heads;
  long long splits = (512 + wide - 1) / wide;
  const long long most = max(splits, 1536 / wide);
  while (splits < most && 10 * 512 * ((wide * splits + 511) / 512) > 11 * wide * splits) ++splits;
  s.splits = (int)max(1ll, min(min(splits, keys / 256), (long long)kMostSplits));
  const double theirs = (double)keys * (d == 128 ? 18e-3 : d == 64 ? 11e-3 : 8e-3) *
                        max(1.0, (double)live * ((tokens + live * 128 - 1) / (live * 128)) * heads / 256);
  const double ours = (double)wide * keys * d * 4 / 4.8e6 + (s.splits > 1 ? 4 : 0);
  // (32768 tokens on 20 states each, 16 heads on 8 of 64: 1237 us, by the prompts' kernel 3166)
  const long long blocks = s.tiles * kv_heads * (s.splits > 8 ? max(s.splits, 16 * s.row_tiles) : s.splits);  // of the larger launch
  if (theirs < ours || blocks >= 1 << 23) s.row_tiles = 0;  // (a launch has less than 2^32 threads)
  return s;
}

template <typename T, int D, int TILES>
hipError_t launch(const PromptArgs &a, const Shape &s, float *workspace, hipStream_t stream) {
  hipLaunchKernelGGL((cross_step_kernel<T, D, TILES>), dim3((unsigned)(s.tiles * a.kv_heads * s.splits)), dim3(64 * kWaves), 0, stream, a, s.splits, workspace);
  if (s.splits > 8)
    hipLaunchKernelGGL((cross_join_many_kernel<T, D, TILES>), dim3((unsigned)(s.tiles * a.kv_heads * 16 * TILES)), dim3(256), 0, stream, a, s.splits, workspace);
  else if (s.splits > 1)
    hipLaunchKernelGGL((cross_join_kernel<T, D, TILES>), dim3((unsigned)(s.tiles * a.kv_heads)), dim3(256), 0, stream, a, s.splits, workspace);
  return hipGetLastError();
}
template <typename T, int D>
hipError_t launch(const PromptArgs &a, const Shape &s, float *workspace, hipStream_t stream) {
  return s.row_tiles == 1 ? launch<T, D, 1>(a, s, workspace, stream) : launch<T, D, 2>(a, s, workspace, stream);
}
template <typename T>
hipError_t launch(int d, const PromptArgs &a, const Shape &s, float *workspace, hipStream_t stream) {
  return d == 128 ? launch<T, 128>(a, s, workspace, stream) : d == 64 ? launch<T, 64>(a, s, workspace, stream) : launch<T, 32>(a, s, workspace, stream);
}

}  // namespace

size_t cross_attention_workspace(int sequences, int tokens, int key_tokens, int heads, int kv_heads, int d) {
  const Shape s = shape_of(sequences, tokens, key_tokens, heads, kv_heads, d);
  return s.row_tiles == 0 || s.splits <= 1 ? 0 : (size_t)s.tiles * kv_heads * s.splits * (size_t)(16 * s.row_tiles) * (d + 2);
}

hipError_t launch_cross_attention(int type, int d, const PromptArgs &a, float *workspace, hipStream_t stream) {
  const Shape s = shape_of(a.sequences, a.tokens, a.key_tokens, a.heads, a.kv_heads, d);
  if (s.row_tiles == 0) return launch_prompt_attention(type, d, false, a, stream);
  return type == 0 ? launch<Fp16>(d, a, s, workspace, stream) : launch<Bf16>(d, a, s, workspace, stream);
}

}  // namespace sspmm
