// Attention over whole prompts that lie one behind the other: for every sequence and head
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^((q_i . k_j) scale log2(e) - m_i),  j <= i (causal) or all j of the sequence,
// with heads / kv_heads query heads on each head of k and v.  One pass over the keys with a running m_i and sum.
#include "prompt_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

constexpr int kKeys = 64;  // keys of a tile
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

// 16 bytes a lane from memory straight into LDS, one lane's behind the other's; what lies behind `bytes` comes as zeros.
__device__ __forceinline__ void load_to_lds(const void *base, uint32_t bytes, uint32_t at, unsigned char *to) {
  typedef __attribute__((address_space(3))) void lds_void;
  const auto srd = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, kSrdWord3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(srd, (lds_void *)to, 16, (int)at, 0, 0, 0);
}

// Whether any of the eight values is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uintx4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= ((v[i] & T::kExponent) == T::kExponent) | (((v[i] >> 16) & T::kExponent) == T::kExponent);
  return bad;
}

// The eight values, with ones where the value is of a kind and zeros elsewhere: 0 = finite values as they are (zeros elsewhere),
// 1 = +infinity, 2 = -infinity, 3 = NaN.
template <typename T>
__device__ __forceinline__ uintx4 of_kind(uintx4 v, int kind) {
  uintx4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t u = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = (v[i] >> (16 * h)) & 0xffffu;
      const bool special = (x & T::kExponent) == T::kExponent;
      const int is = !special ? 0 : x == T::kInfinity ? 1 : x == (0x8000u | T::kInfinity) ? 2 : 3;
      u |= (is != kind ? 0u : kind == 0 ? x : T::kOne) << (16 * h);
    }
    r[i] = u;
  }
  return r;
}

// A workgroup of WAVES waves owns 32 * WAVES consecutive queries of one sequence and head, 32 a wave.
// Scores are made transposed, K Q^T, so that a lane holds 32 of a tile's 64 scores of ONE query: maxima and sums are taken
// inside the lane, but for one exchange with the lane 32 apart, and what the matrix instruction leaves is, rounded to 16 bits, the operand P^T
// of the second product V^T P^T, whose contraction slots are numbered accordingly: slots of lane half h in step t are keys
// 16 t + 4 h + {0 .. 3, 8 .. 11}.  V^T comes from transpose reads.
template <typename T, int D, int WAVES, bool CAUSAL>
__global__ __launch_bounds__(64 * WAVES, 2) void prompt_attention_kernel(const PromptArgs p, int tiles, int blocks) {
  constexpr int kQueries = 32 * WAVES, kPieces = D / 8, kTile = kKeys * D * 2;
  constexpr int kSteps = D / 16, kParts = D / 32;  // steps of the first product; parts of 32 features of the second
  constexpr int kLoads = kTile / (64 * WAVES * 16);  // pieces of 16 bytes of a tile that a thread fetches
  __shared__ __align__(16) unsigned char lds[4 * kTile];  // K, V, K, V
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // ---- which queries
  int tile, head;
  {
    const int group = p.heads / p.kv_heads;
    if (p.kv_heads % 8 == 0) {
      // Workgroup ids go round-robin to the 8 XCDs: a head of k and v stays with one of them and its L2.
      const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3, per = tiles * group;
      const int kv = (i / per) * 8 + xcd, j = i % per;
      tile = j / group;
      head = kv * group + j % group;
    } else {
      tile = blockIdx.x / p.heads;
      head = blockIdx.x % p.heads;
    }
  }
  if ((int)blockIdx.x >= blocks) return;
  int first = 0, length = -1, q0 = 0;  // the sequence's first row and rows, the workgroup's first query in it
  for (int b0 = 0, base = 0; b0 < p.sequences; b0 += 64) {
    const int b = b0 + lane;
    int lo = 0, hi = 0;
    if (b < p.sequences) {
      lo = max(0, min(p.offsets[b], p.tokens));
      hi = max(lo, min(p.offsets[b + 1], p.tokens));
    }
    const int count = (int)(((long long)(hi - lo) + kQueries - 1) / kQueries);
    const int upto = base + (int)wave_inclusive_sum((uint32_t)count);
    const unsigned long long found = __ballot(upto > tile);
    if (found != 0) {
      const int at = __builtin_ctzll(found);
      first = __builtin_amdgcn_readlane(lo, at);
      length = __builtin_amdgcn_readlane(hi, at) - first;
      // (the last queries first: with a causal mask these have the most keys)
      q0 = (__builtin_amdgcn_readlane(upto, at) - 1 - tile) * kQueries;
      break;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
  }
  if (length < 0) return;  // (there are fewer tiles than the host could exclude)

  const int kv_head = head / (p.heads / p.kv_heads);
  const int my = q0 + 32 * wave + n;  // this lane's query
  const int seen = CAUSAL ? min(my + 1, length) : length;  // keys it sees: those below
  const int all_see = CAUSAL ? min(q0 + 32 * wave + 1, length) : length;  // (every query of the wave sees those below this)
  const int most = CAUSAL ? min(q0 + 32 * wave + 32, length) : length;  // (and none of them one from here on)
  const int last = CAUSAL ? min(q0 + kQueries, length) : length;
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
  uint32_t k_at[kLoads], v_at[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int piece = (i * WAVES + wave) * 64 + lane, r = piece / kPieces, c = piece % kPieces;
    k_at[i] = r * k_pitch + (c ^ swizzle_k<D>(r)) * 16;
    v_at[i] = r * v_pitch + (c ^ swizzle_v<D>(r)) * 16;
  }
  const auto fetch = [&](int t) {
    const int rows = min(kKeys, length - t * kKeys);
    const uint16_t *const k = k0 + (long long)t * kKeys * p.k_row, *const v = v0 + (long long)t * kKeys * p.v_row;
    unsigned char *const to = lds + (t & 1) * 2 * kTile + wave * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds(k, (rows - 1) * k_pitch + D * 2, k_at[i], to + i * WAVES * 1024);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds(v, (rows - 1) * v_pitch + D * 2, v_at[i], to + kTile + i * WAVES * 1024);
  };

  floatx16 o[kParts];  // lane (n, half): features 32 part + 8 (i / 4) + 4 half + i % 4 of its query
#pragma unroll
  for (int part = 0; part < kParts; ++part)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[part][i] = 0.f;
  float run_max = -3.0e38f, run_sum = 0.f;  // of the scaled scores; this lane's share of the sum
  const float c = p.scale_log2e;

  fetch(0);
  for (int t = 0; t < key_tiles; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // tile t is there, and nobody reads tile t - 1 any more
    if (t + 1 < key_tiles) fetch(t + 1);
    const int key0 = t * kKeys;
    if (key0 >= most) continue;  // (the barrier above is in every wave's path)
    const unsigned char *const k_tile = lds + (t & 1) * 2 * kTile, *const v_tile = k_tile + kTile;

    floatx16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
      const int r = 32 * kt + n;
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        const uintx4 k = *reinterpret_cast<const uintx4 *>(k_tile + r * (D * 2) + (((2 * step + half) ^ swizzle_k<D>(r)) * 16));
        s[kt] = T::mfma_32x32x16(k, q[step], s[kt]);
      }
    }
    const bool cut = key0 + kKeys > all_see;  // uniform in the wave
    if (cut) {
      const int left = seen - key0 - 4 * half;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * kt + 8 * (i / 4) + i % 4 >= left) s[kt][i] = -INFINITY;
    }
    float most_here = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) most_here = fmaxf(most_here, s[kt][i]);
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most_here), __float_as_uint(most_here), false, false);
      most_here = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    // The reference point moves only when some query's maximum has grown by more than 2^8: until then probabilities are up to 2^8
    // too large, which either type holds, and the accumulators stay as they are.
    const float new_max = fmaxf(run_max, most_here * c);
    if (__ballot(new_max - run_max > 8.0f) != 0) {
      const float alpha = __builtin_amdgcn_exp2f(fmaxf(run_max - new_max, -126.0f));
      run_max = new_max;
      run_sum *= alpha;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[part][i] *= alpha;
    }
    uintx4 pt[4];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = __builtin_amdgcn_exp2f(fmaf(s[kt][i], c, -run_max)), b = __builtin_amdgcn_exp2f(fmaf(s[kt][i + 1], c, -run_max));
        run_sum += a + b;  // (of the exponentials, not of what 16 bits make of them)
        pt[2 * kt + i / 8][(i % 8) / 2] = T::pack(a, b);
      }

    const auto read_v = [&](int part, int step) {
      const int r = 16 * step + 4 * half + ((lane & 15) >> 2), piece = 4 * part + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const unsigned char *const at = v_tile + r * (D * 2) + ((piece ^ swizzle_v<D>(r)) * 16) + (lane & 1) * 8;
      const uintx2 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * (D * 2));  // (swizzle_v is the same eight rows on)
      return uintx4{lo[0], lo[1], hi[0], hi[1]};
    };
    bool bad = false;
    if (cut) {
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int step = 0; step < 4; ++step) bad |= not_finite<T>(read_v(part, step));
      bad = __ballot(bad) != 0;
    }
    if (!__builtin_expect(bad, 0)) {
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int step = 0; step < 4; ++step) o[part] = T::mfma_32x32x16(read_v(part, step), pt[step], o[part]);
    } else {
      // A masked key's probability is zero, but zero times an infinity or a NaN in its v is NaN.  Finite values as ever; of the others,
      // those that a query sees are counted by the same instruction, kind by kind.
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int step = 0; step < 4; ++step) o[part] = T::mfma_32x32x16(of_kind<T>(read_v(part, step), 0), pt[step], o[part]);
      uintx4 sees[4];
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = 16 * step + 4 * half + 8 * (j >> 1) + 2 * (j & 1), left = seen - key0;
          sees[step][j] = (key < left ? T::kOne : 0u) | (key + 1 < left ? T::kOne << 16 : 0u);
        }
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        for (int kind = 1; kind < 4; ++kind) {
          floatx16 count;
#pragma unroll
          for (int i = 0; i < 16; ++i) count[i] = 0.f;
#pragma unroll
          for (int step = 0; step < 4; ++step) count = T::mfma_32x32x16(of_kind<T>(read_v(part, step), kind), sees[step], count);
          const float what = kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
#pragma unroll
          for (int i = 0; i < 16; ++i) o[part][i] += count[i] > 0.f ? what : 0.f;
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

template <typename T, int D, int WAVES>
hipError_t launch(bool causal, const PromptArgs &a, hipStream_t stream) {
  const long long tiles = (long long)a.tokens / (32 * WAVES) + a.sequences, blocks = tiles * a.heads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (causal)
    hipLaunchKernelGGL((prompt_attention_kernel<T, D, WAVES, true>), dim3((unsigned)blocks), dim3(64 * WAVES), 0, stream, a, (int)tiles, (int)blocks);
  else
    hipLaunchKernelGGL((prompt_attention_kernel<T, D, WAVES, false>), dim3((unsigned)blocks), dim3(64 * WAVES), 0, stream, a, (int)tiles, (int)blocks);
  return hipGetLastError();
}

template <typename T>
hipError_t launch(int d, bool causal, const PromptArgs &a, hipStream_t stream) {
  return d == 128 ? launch<T, 128, 4>(causal, a, stream) : d == 64 ? launch<T, 64, 4>(causal, a, stream) : launch<T, 32, 4>(causal, a, stream);
}

}  // namespace

hipError_t launch_prompt_attention(int type, int d, bool causal, const PromptArgs &args, hipStream_t stream) {
  return type == 0 ? launch<Fp16>(d, causal, args, stream) : launch<Bf16>(d, causal, args, stream);
}

}  // namespace sspmm
