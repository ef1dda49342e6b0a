// Attention over whole prompts that lie one behind the other: for every sequence and head
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^((q_i . k_j) scale log2(e) - m_i),  j <= i (causal) or all j of the sequence,
// with heads / kv_heads query heads on each head of k and v.  One pass over the keys with a running m_i and sum.
#include "prompt_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

#include <type_traits>

namespace sspmm {

namespace {

constexpr int kKeys = 64;  // keys of a tile
constexpr int kWaves = 4, kTileQueries = 32 * kWaves;  // of a group, and queries of a workgroup
constexpr uint32_t kSrdWord3 = 0x00020000u;

// A tile's row r is D elements in pieces of 16 bytes; piece c lies at place c ^ swizzle(r) of the row.  K's fragments are read by 32 lanes
// from 32 consecutive rows at the same piece, V's by 32 lanes from four consecutive rows at four consecutive pieces: with
// these either falls on all 64 banks.
template <int D>
__device__ __forceinline__ int swizzle_k(int r) {
  return D == 128 ? r & 15 : D == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int swizzle_v(int r) {
  return D == 128 ? (r & 3) * 4 : D == 64 ? ((r >> 1) & 1) * 4 : 0;
}

// 16 bytes a lane from memory straight into LDS, one lane's behind the other's from `to` on; what lies behind the descriptor's bytes comes as
// zeros.  As assembly because the compiler, which cannot tell one tile of LDS from another, makes every read of the tile that is worked on wait for
// the next one's loads (16001 tokens, 8 heads: 619 us with the builtin); the waits for these are the ones before the barriers below.
typedef int srd __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(srd from, uint32_t at, uint32_t to) {
  // m0 is the compiler's (it takes no such clobber): it is put back, which the load, once issued, does not mind.  (The wait is what a vector instruction that wrote
  // one of the scalars just before would need.)
  uint32_t kept;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(kept) : "s"(to), "v"(at), "s"(from) : "memory");
}
__device__ __forceinline__ srd descriptor(const uint16_t *base, uint32_t bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  return srd{(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)bytes, (int)kSrdWord3};
}

// The eight values with zeros in place of infinities and NaN.
template <typename T>
__device__ __forceinline__ uintx4 finite_part(uintx4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((v[i] & T::kExponent) == T::kExponent) v[i] &= 0xffff0000u;
    if (((v[i] >> 16) & T::kExponent) == T::kExponent) v[i] &= 0xffffu;
  }
  return v;
}

// A workgroup owns 128 consecutive queries of one sequence and head, 32 a wave, and passes over the keys they see in tiles of 64.
// Scores are made transposed, K Q^T, so that a lane holds 32 of a tile's 64 scores of ONE query: maxima and sums are taken
// inside the lane, but for one exchange with the lane 32 apart, and what the matrix instruction leaves is, rounded to 16 bits, the operand P^T
// of the second product V^T P^T, whose contraction slots are numbered accordingly: slots of lane half h in step t are keys
// 16 t + 4 h + {0 .. 3, 8 .. 11}.  V^T comes from transpose reads.  Two buffers of K and V, one barrier a tile, two workgroups a CU (64 KB and up to 228
// registers a lane with 128 features).
//
// Bound by the matrix instructions and the power they take: 16384 tokens, 8 heads of 128 features in bf16, 1.03 to 1.13 PFLOP/s causal and 1.05 to 1.17 not (three
// cards), where the library's product of 8192^3 reaches 1.1 to 1.25 in its first launches and 1.39 in a long run of them; the clock stands at 1.85 GHz, the matrix
// units are busy 53 % of the cycles, the vector ones 37 % (without the exponentials the launch takes 5 % less, with K and V from registers 33 %).  Tried without gain: all of K's operands asked for
// ahead, K two tiles and V one and a half ahead with two barriers a tile, 256 queries a workgroup, 64 queries a workgroup (1.4 times as long).
// Short prompts wait for their latencies: 512 tokens, 32 heads 15 us, eight tiles one after the other.
template <typename T, int D, int GROUPS, bool CAUSAL, bool AHEAD>
__global__ __launch_bounds__(64 * kWaves * GROUPS, 2) void prompt_attention_kernel(const PromptArgs p, int tiles) {
  constexpr int kPieces = D / 8, kTile = kKeys * D * 2;
  constexpr int kSteps = D / 16, kParts = D / 32;  // steps of the first product; parts of 32 features of the second
  constexpr int kLoads = kTile / (64 * kWaves * 16);  // pieces of 16 bytes of a tile that a thread fetches
  __shared__ __align__(16) unsigned char tiles_lds[GROUPS * 4 * kTile];  // of each group K, V, K, V
  __shared__ int once_more;
  __shared__ float states[GROUPS > 1 ? (GROUPS - 1) * kWaves * 2 * 64 : 1];
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * kWaves));
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % kWaves);
  unsigned char *const lds = tiles_lds + group * 4 * kTile;

  // ---- which queries
  int tile, head;
  {
    const int per_kv = p.heads / p.kv_heads;
    if (p.kv_heads % 8 == 0) {
      // Workgroup ids go round-robin to the 8 XCDs: a head of k and v stays with one of them and its L2.
      const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3, per = tiles * per_kv;
      const int kv = (i / per) * 8 + xcd, j = i % per;
      tile = j / per_kv;
      head = kv * per_kv + j % per_kv;
    } else {
      tile = blockIdx.x / p.heads;
      head = blockIdx.x % p.heads;
    }
  }
  // Numbers offsets[b] / 128 + b .. are sequence b's, enough for its tiles however it lies; a workgroup with one too many ends at once.  (Summing up
  // the tiles of the sequences before: 4096 sequences of 64 tokens, 8 heads 947 us instead of 360.)  Of 64 sequences at a time those with the most
  // keys go first: level x (a causal tile has about as many keys as places before it in its sequence, another as many as its sequence) is
  // the largest at which more tiles than those before this one are of x or more.
  int first = 0, length = -1, q0 = 0;  // the sequence's first row and rows, the workgroup's first query in it
  const auto base = [&](int chunk) { return max(0, min(p.offsets[64 * chunk], p.tokens)) / kTileQueries + 64 * chunk; };
  const int chunk = last_not_above((p.sequences + 63) / 64, tile, base);
  int left = tile - base(chunk);
  if (left >= 0) {
    const int b = 64 * chunk + lane;
    int lo = 0, hi = 0;
    if (b < p.sequences) {
      lo = max(0, min(p.offsets[b], p.tokens));
      hi = max(lo, min(p.offsets[b + 1], p.tokens));
    }
    const int count = (int)(((long long)(hi - lo) + kTileQueries - 1) / kTileQueries);
    const int all = (int)from_last_lane(wave_inclusive_sum((uint32_t)count));
    if (left >= all) return;
    int x = 1, above = 0, end = (int)from_last_lane(wave_inclusive_max((uint32_t)count)) + 1;  // above: tiles of `end` or more
    while (end - x > 1) {
      const int mid = (x + end) >> 1;
      const int n_mid = count < mid ? 0 : CAUSAL ? count - mid + 1 : count;
      const int upwards = (int)from_last_lane(wave_inclusive_sum((uint32_t)n_mid));
      if (upwards > left) {
        x = mid;
      } else {
        end = mid;
        above = upwards;
      }
    }
    left -= above;  // which of level x
    const unsigned long long those = __ballot(CAUSAL ? count >= x : count == x);
    const int which = CAUSAL ? left : left / x;
    const bool is = (those >> lane & 1) && __popcll(those & ((1ull << lane) - 1)) == which;
    const int at = __builtin_ctzll(__ballot(is));
    first = __builtin_amdgcn_readlane(lo, at);
    length = __builtin_amdgcn_readlane(hi, at) - first;
    q0 = (CAUSAL ? x - 1 : left % x) * kTileQueries;
  }
  if (length < 0) return;

  const int kv_head = head / (p.heads / p.kv_heads);
  const int my = q0 + 32 * wave + n;  // this lane's query
  const int seen = CAUSAL ? min(my + 1, length) : length;  // keys it sees: those below
  const int most = CAUSAL ? min(q0 + 32 * wave + 32, length) : length;  // (no query of the wave sees one from here on)
  const int last = CAUSAL ? min(q0 + kTileQueries, length) : length;
  const int key_tiles = (last + kKeys - 1) / kKeys;

  // ---- queries: lane (n, half) holds features 16 s + 8 half .. + 7 of its query
  uintx4 q[kSteps];
  {
    const uint16_t *at = p.q + (long long)(first + min(my, length - 1)) * p.q_row + (long long)head * p.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const uintx4 *>(at + 16 * s);
  }

  // ---- tiles come from memory straight into LDS; rows behind the sequence are zeros
  const uint16_t *const k0 = p.k + (long long)first * p.k_row + (long long)kv_head * p.k_head;
  const uint16_t *const v0 = p.v + (long long)first * p.v_row + (long long)kv_head * p.v_head;
  const uint32_t k_pitch = (uint32_t)p.k_row * 2, v_pitch = (uint32_t)p.v_row * 2;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds + wave * 1024;
  uint32_t k_at[kLoads], v_at[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int piece = (i * kWaves + wave) * 64 + lane, r = piece / kPieces, c = piece % kPieces;
    k_at[i] = r * k_pitch + (c ^ swizzle_k<D>(r)) * 16;
    v_at[i] = r * v_pitch + (c ^ swizzle_v<D>(r)) * 16;
  }
  const auto fetch = [&](int t) {
    const int rows = min(kKeys, length - t * kKeys);
    const srd sk = descriptor(k0 + (long long)t * kKeys * p.k_row, (rows - 1) * k_pitch + D * 2);
    const srd sv = descriptor(v0 + (long long)t * kKeys * p.v_row, (rows - 1) * v_pitch + D * 2);
    const uint32_t to = lds_at + (t / GROUPS & 1) * 2 * kTile;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds(sk, k_at[i], to + i * kWaves * 1024);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds(sv, v_at[i], to + kTile + i * kWaves * 1024);
  };

  // ---- where a lane's operands lie in a tile: of K in its first 32 rows by step, of V in the first 8 rows of a step by part
  uint32_t k_rd[kSteps], v_rd[kParts];
#pragma unroll
  for (int step = 0; step < kSteps; ++step) k_rd[step] = n * (D * 2) + (((2 * step + half) ^ swizzle_k<D>(n)) * 16);  // (32 rows on: the same swizzle)
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    const int r = 4 * half + ((lane & 15) >> 2), piece = 4 * part + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    v_rd[part] = kTile + r * (D * 2) + ((piece ^ swizzle_v<D>(r)) * 16) + (lane & 1) * 8;  // (8 rows on: the same swizzle)
  }

  floatx16 o[kParts];  // lane (n, half): features 32 part + 8 (i / 4) + 4 half + i % 4 of its query
  float run_max, run_sum;  // of the scaled scores; this lane's share of the sum
  const float c = p.scale_log2e;
  // fp16 loses what is below 2^-25, and many keys of small probabilities are not nothing: their largest is 2^7 or more there.  bf16 does not, but its v may be as
  // large as 32 bits hold: probabilities are 1 at most, so that sums overflow where the formula's do.
  constexpr float kHeadroom = __is_same(T, Fp16) ? 7.f : -8.f;

  const auto read_v = [&](const unsigned char *tile, int part, int step) __attribute__((always_inline)) {
    const unsigned char *const at = tile + v_rd[part] + 16 * step * (D * 2);
    const uintx2 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * (D * 2));
    return uintx4{lo[0], lo[1], hi[0], hi[1]};
  };
  const auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[part][i] = 0.f;
    run_max = -3.0e38f;
    run_sum = 0.f;
  };
  const auto move_by = [&](float grown) __attribute__((always_inline)) {  // the reference point, by so many powers of two
    const float down = half_way_down(grown);
    run_sum = run_sum * down * down;
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[part][i] = o[part][i] * down * down;
  };

  // Tile t, in `tile` of LDS.  cut: some query may not see all of its keys.
  const auto work_on = [&](auto cut_, const unsigned char *tile, int key0) {
    constexpr bool cut = decltype(cut_)::value;
    floatx16 s[2];
    uintx4 pt[4];
    const auto scores = [&](int kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
        s[kt] = T::mfma_32x32x16(*reinterpret_cast<const uintx4 *>(tile + k_rd[step] + 32 * kt * (D * 2)), q[step], s[kt]);
    };
    // The reference point of the exponentials moves only when some query's maximum has grown by more than 2^8: until then probabilities are up
    // to 2^8 times the first tile's largest, 2^15 in fp16 and 1 in bf16, and the accumulators stay as they are.
    const auto refer = [&]() {
      if constexpr (cut) {
        const int left = seen - key0 - 4 * half;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[kt][i] = 32 * kt + 8 * (i / 4) + i % 4 >= left ? -INFINITY : s[kt][i];
      }
      float most = s[0][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[kt][i]);
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
      const float new_max = fmaxf(run_max, fmaf(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])), c, -kHeadroom));
      if (__builtin_expect(__ballot(new_max - run_max > 8.0f) != 0, 0)) {
        move_by(new_max - run_max);
        run_max = new_max;
      }
    };
    const auto exponentials = [&](int kt) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = __builtin_amdgcn_exp2f(fmaf(s[kt][i], c, -run_max)), b = __builtin_amdgcn_exp2f(fmaf(s[kt][i + 1], c, -run_max));
        run_sum += a + b;  // (of the exponentials, not of what 16 bits make of them)
        pt[2 * kt + i / 8][(i % 8) / 2] = T::pack(a, b);
      }
    };
    const auto products = [&](int kt) {
#pragma unroll
      for (int step = 2 * kt; step < 2 * kt + 2; ++step)
#pragma unroll
        for (int part = 0; part < kParts; ++part) o[part] = T::mfma_32x32x16(read_v(tile, part, step), pt[step], o[part]);
    };

    // (the second half's exponentials run beside the first half's products)
    if constexpr (AHEAD) __builtin_amdgcn_s_setprio(1);
    scores(0);
    scores(1);
    refer();
    exponentials(0);
    products(0);
    if constexpr (AHEAD) __builtin_amdgcn_s_setprio(0);
    exponentials(1);
    products(1);
  };

  // The same for a workgroup that goes over its keys again, 32 of them at a time.  run_max is of the scores themselves here.
  const auto work_again = [&](const unsigned char *tile, int key0) __attribute__((always_inline)) {
#pragma unroll 1
    for (int kt = 0; kt < 2; ++kt) {
      floatx16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
        s = T::mfma_32x32x16(*reinterpret_cast<const uintx4 *>(tile + k_rd[step] + 32 * kt * (D * 2)), q[step], s);
      const int left = seen - key0 - 32 * kt - 4 * half;
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = 8 * (i / 4) + i % 4 >= left ? -INFINITY : s[i];
        most = fmaxf(most, s[i]);
      }
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
      const float new_max = fmaxf(run_max, fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
      const float grown = (new_max - run_max) * c;
      if (__ballot(grown > 8.0f) != 0) {
        move_by(grown);
        run_max = new_max;
      }
      uintx4 pt[2];
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = __builtin_amdgcn_exp2f(fmaf(s[i] - run_max, c, kHeadroom)), b = __builtin_amdgcn_exp2f(fmaf(s[i + 1] - run_max, c, kHeadroom));
        run_sum += a + b;
        pt[i / 8][(i % 8) / 2] = T::pack(a, b);
      }
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int part = 0; part < kParts; ++part)
          o[part] = T::mfma_32x32x16(finite_part<T>(read_v(tile, part, 2 * kt + step)), pt[step], o[part]);
    }
    uint32_t others = 0;
#pragma unroll 1
    for (int i = 0; i < kTile; i += 1024) {
      const uintx4 v = *reinterpret_cast<const uintx4 *>(tile + kTile + i + lane * 16), finite = finite_part<T>(v);
      others |= (v[0] ^ finite[0]) | (v[1] ^ finite[1]) | (v[2] ^ finite[2]) | (v[3] ^ finite[3]);
    }
    const int special = __ballot(others != 0) != 0 ? kKeys : 0;
#pragma unroll 1
    for (int r = 0; r < special; ++r) {
      const bool sees = key0 + r < seen;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int piece = 4 * part + i / 4;
          const uintx2 v = *reinterpret_cast<const uintx2 *>(tile + kTile + r * (D * 2) + ((piece ^ swizzle_v<D>(r)) * 16) + 8 * half);
          const float x[4] = {T::lower(v[0]), T::upper(v[0]), T::lower(v[1]), T::upper(v[1])};
#pragma unroll
          for (int j = 0; j < 4; ++j) o[part][i + j] += sees && !(fabsf(x[j]) < INFINITY) ? x[j] : 0.f;
        }
    }
  };

  // Group g works on tiles g, g + GROUPS, ...; all of them pass the same barriers.
  const std::integral_constant<bool, false> whole{};
  const std::integral_constant<bool, true> cut{};
  const auto next = [&](int t) {  // tile t is there, and nobody reads the group's tile before it any more
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    if (t + GROUPS < key_tiles) fetch(t + GROUPS);
  };
  const int whole_tiles = (CAUSAL ? min(q0 + 1, length) : length) / kKeys;  // that all queries of the workgroup see
  // A masked key's probability is zero, and so is what underflows, but zero times an infinity or a NaN in v is NaN.  A workgroup that finds a
  // result which is not finite goes over its keys again: the products are of the finite values then, and the others are added, key by key,
  // to the queries that see them.  (Looking at every tile at the mask's edge first: 512 tokens, 32 heads of 128 features 17.0 us instead of 15.1.)
  // So does one whose reference points lie beyond 2^24: an exponent is the score times c minus that, one rounding in all, but off by what the
  // reference point was rounded by, for all keys of the query alike.  Half a power of two at most up to there; at 2^28 eight of them, and the largest probability
  // may be infinite in fp16, or nothing.  The second time differences of scores are taken first.
  if (threadIdx.x == 0) once_more = 0;
  begin();
  if (group < key_tiles) fetch(group);
  int t0 = 0;  // group 0's tile
  for (; t0 + 2 * GROUPS <= whole_tiles; t0 += 2 * GROUPS) {
    const int t = t0 + group;
    next(t);
    work_on(whole, lds, t * kKeys);
    next(t + GROUPS);
    work_on(whole, lds + 2 * kTile, (t + GROUPS) * kKeys);
  }
  for (; t0 < key_tiles; t0 += GROUPS) {
    const int t = t0 + group;
    next(t);
    if (t * kKeys < most) work_on(cut, lds + (t / GROUPS & 1) * 2 * kTile, t * kKeys);
  }
  float zero = 0.f;
#pragma unroll
  for (int part = 0; part < kParts; ++part)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = fmaf(o[part][i], 0.f, zero);
  const bool far = seen > group * kKeys && !(fabsf(run_max) < 0x1p24f);  // (a query that sees none of the group's keys has no reference point)
  if (__ballot(zero != zero || far) != 0 && lane == 0) once_more = 1;
  __syncthreads();
  const bool again = __builtin_amdgcn_readfirstlane(once_more) != 0;
  if (__builtin_expect(again, 0)) {
    begin();
    if (group < key_tiles) fetch(group);
    for (t0 = 0; t0 < key_tiles; t0 += GROUPS) {
      const int t = t0 + group;
      next(t);
      if (t * kKeys < most) work_again(lds + (t / GROUPS & 1) * 2 * kTile, t * kKeys);
    }
  }

  if constexpr (GROUPS > 1) {
    // ---- the groups' states as one: the others leave theirs where their tiles were
    static_assert(kParts * 16 * 64 * 4 * kWaves <= 4 * kTile, "a group's accumulators fit its tiles");
    __syncthreads();
    if (group > 0) {
      floatx4 *const to = reinterpret_cast<floatx4 *>(lds) + wave * (kParts * 4 * 64) + lane;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(part * 4 + i) * 64] = floatx4{o[part][4 * i], o[part][4 * i + 1], o[part][4 * i + 2], o[part][4 * i + 3]};
      float *const st = states + ((group - 1) * kWaves + wave) * 128 + lane;
      st[0] = run_max;
      st[64] = run_sum;
    }
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g < GROUPS; ++g) {
      const float *const st = states + ((g - 1) * kWaves + wave) * 128 + lane;
      const float new_max = fmaxf(run_max, st[0]), unit = again ? c : 1.f;
      const float mine = half_way_down((new_max - run_max) * unit), theirs = half_way_down((new_max - st[0]) * unit);
      run_max = new_max;
      run_sum = run_sum * mine * mine + st[64] * theirs * theirs;
      const floatx4 *const from = reinterpret_cast<const floatx4 *>(tiles_lds + g * 4 * kTile) + wave * (kParts * 4 * 64) + lane;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const floatx4 x = from[(part * 4 + i) * 64];
#pragma unroll
          for (int j = 0; j < 4; ++j) o[part][4 * i + j] = o[part][4 * i + j] * mine * mine + x[j] * theirs * theirs;
        }
    }
  }

  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(run_sum), __float_as_uint(run_sum), false, false);
    run_sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (my >= length) return;
  const float inv = run_sum > 0.f || run_sum != run_sum ? 1.0f / run_sum : 0.f;  // (scores of -infinity only: zeros)
  uint16_t *const to = p.out + (long long)(first + my) * p.out_row + (long long)head * p.out_head + 4 * half;
#pragma unroll
  for (int part = 0; part < kParts; ++part)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uintx2 four = {T::pack(o[part][i] * inv, o[part][i + 1] * inv), T::pack(o[part][i + 2] * inv, o[part][i + 3] * inv)};
      *reinterpret_cast<uintx2 *>(to + 32 * part + 2 * i) = four;
    }
}

template <typename T, int D, int GROUPS, bool AHEAD>
hipError_t launch(bool causal, const PromptArgs &a, hipStream_t stream) {
  const long long tiles = (long long)a.tokens / kTileQueries + a.sequences;
  const unsigned threads = 64 * kWaves * GROUPS;
  if (tiles * a.heads >= 1 << 23) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  const unsigned blocks = (unsigned)(tiles * a.heads);
  if (causal)
    hipLaunchKernelGGL((prompt_attention_kernel<T, D, GROUPS, true, AHEAD>), dim3(blocks), dim3(threads), 0, stream, a, (int)tiles);
  else
    hipLaunchKernelGGL((prompt_attention_kernel<T, D, GROUPS, false, AHEAD>), dim3(blocks), dim3(threads), 0, stream, a, (int)tiles);
  return hipGetLastError();
}

// Two groups where one would leave half of the chip's 512 places for workgroups empty, or with a causal mask most of them while the last
// tiles of long sequences run (lengths known on average only: a sequence of a few hundred tokens has nothing to split).  One group and two, us: causal,
// 128 features, 4096 tokens 16 heads 108 and 82, 8 heads 74 and 60, 1000 tokens 16 heads 23.1 and 21.2; 2048 tokens 32 heads 58 and 59; not causal, 2048 tokens 8 heads
// 39.9 and 33.9; 8 x 512 tokens, 12 heads of 64 15.6 and 16.6.
long long workgroups(const PromptArgs &a) { return ((long long)a.tokens + kTileQueries - 1) / kTileQueries * a.heads; }
bool two_groups(bool causal, const PromptArgs &a) {
  const long long tiles = workgroups(a), length = a.tokens / a.sequences;
  return length >= 768 && (tiles <= 256 || (causal && tiles <= 512 && length >= 3000));
}

// Waves that are between a tile's scores and its first products go ahead of the others on their SIMD.  128 features, causal, 8 heads of 16001 tokens
// 551 -> 509 us, 16 of 8192 292 -> 276, 4 of 32768 1122 -> 1034, 12 of 20000 1195 -> 1180; 64 of 4096 273 -> 281, 32 of 2048 51.0 -> 52.2: for sequences of more than 6000
// tokens.  Not where little more than one round of workgroups has to be done, 512 places: 8 heads of 9000 tokens (568) 201 -> 211, 4 of 20000 (628) 460 -> 481,
// 12000 (752) 286 -> 306, 12500 (784) 329 -> 343, 13000 (816) 359 -> 365, 15000 (944) 465 -> 424.
// Without a mask the bad stretch ends sooner: 8 heads of 6500 tokens (408) 191 -> 180, 8192 (512) 267 -> 259, 9000 416 -> 436, 4 of 20000 917 -> 961, 12500 722 -> 671, 13000
// 757 -> 708, 16001 1011 -> 973, 32768 4143 -> 4037; 32 of 6500 (1632) 708 -> 729.  The mean length is what the host knows: 16001 tokens with two prompts of one token beside
// them go without (545 us, with it 503).
bool go_ahead(const PromptArgs &a) { return a.tokens / a.sequences > 6000 && (workgroups(a) <= 512 || workgroups(a) > 800); }

template <typename T, int D>
hipError_t launch(bool causal, const PromptArgs &a, hipStream_t stream) {
  if (two_groups(causal, a)) return launch<T, D, 2, false>(causal, a, stream);
  if constexpr (D == 128)
    if (go_ahead(a)) return launch<T, D, 1, true>(causal, a, stream);
  return launch<T, D, 1, false>(causal, a, stream);
}

template <typename T>
hipError_t launch(int d, bool causal, const PromptArgs &a, hipStream_t stream) {
  return d == 128 ? launch<T, 128>(causal, a, stream) : d == 64 ? launch<T, 64>(causal, a, stream) : launch<T, 32>(causal, a, stream);
}

}  // namespace

hipError_t launch_prompt_attention(int type, int d, bool causal, const PromptArgs &args, hipStream_t stream) {
  return type == 0 ? launch<Fp16>(d, causal, args, stream) : launch<Bf16>(d, causal, args, stream);
}

}  // namespace sspmm
