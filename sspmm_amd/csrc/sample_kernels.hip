// Tokens drawn from rows of logits l with given uniform numbers u.  With z_i = (max l - l_i) / T a token's weight is w_i = exp(-z_i); kept are those with
// w_i >= min_p, of these the top_k first in the order of falling logits (equal ones in the order of their indices), of these the shortest run whose weights
// reach top_p of all of theirs.  The token is the first in that order at which the running sum of the weights exceeds u times their sum.
//
// Weights are whole numbers, in units of 2^-unit_bits of the largest: sums of them are exact in any order, so that atomics and lanes give the same token every
// time.  Vocabularies of 2^17 leave 45 bits; what weighs less than half a unit is never drawn.  No row is sorted: a row is put into bins by z, which is to say
// by weight, and where a count or a sum ends inside a bin that bin alone is split by its logits until one logit is left.
#include "sample_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 4096, kFine = 1024;  // of the whole row, and of a range of logits

struct F32 {};

template <typename T>
struct Elements {  // of 16 bytes
  static constexpr int kCount = 8, kBytes = 2;
  static __device__ __forceinline__ void take(uintx4 w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = T::lower(w[i]);
      x[2 * i + 1] = T::upper(w[i]);
    }
  }
  static __device__ __forceinline__ float one(const void *p) { return T::lower(*static_cast<const uint16_t *>(p)); }
};
template <>
struct Elements<F32> {
  static constexpr int kCount = 4, kBytes = 4;
  static __device__ __forceinline__ void take(uintx4 w, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ float one(const void *p) { return *static_cast<const float *>(p); }
};

// Numbers in the order of the logits; -0 and 0 are one logit.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

typedef unsigned long long u64;

// What a workgroup knows of its row.
struct Row {
  float most;            // the largest logit
  double per_logit;      // 1 / T
  double farthest;       // largest z of a token that is kept
  double unit;           // weight of the largest
  // (monotone in x, so that bins and ranges of logits never cross)
  __device__ __forceinline__ bool candidate(float x, double &z) const {
    z = x == most ? 0.0 : ((double)most - (double)x) * per_logit;
    return x > -INFINITY && (x == most || most < INFINITY) && z <= farthest;
  }
  __device__ __forceinline__ u64 weight(double z) const { return (u64)(exp(-z) * unit + 0.5); }
};

struct Shared {
  u64 weights[kBins];
  uint32_t counts[kBins];
  u64 fine_weights[kFine];
  uint32_t fine_counts[kFine];
  u64 wave_weights[kWaves];
  uint32_t wave_counts[kWaves];
  uint32_t low, high;
  int found, token;
  u64 before_weight, at_weight;
  uint32_t before_count, at_count;
};

// A place in the order: the logit, what lies before its first token, its tokens and the weight of each.
struct Place {
  uint32_t key, before_count, tokens;
  u64 before_weight, weight;
};

template <typename T>
struct Reader {
  typedef Elements<T> E;
  const unsigned char *blocks;  // 16-byte aligned, at or before the row's first element
  int lead, vocab, first, end;  // elements before the row in its first block, of the row; the wave's blocks
  __device__ __forceinline__ Reader(const void *row, int vocab_) : vocab(vocab_) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    blocks = reinterpret_cast<const unsigned char *>(at & ~(uintptr_t)15);
    lead = (int)(at & 15) / E::kBytes;
    const int all = (lead + vocab + E::kCount - 1) / E::kCount, each = (all + kThreads - 1) / kThreads * 64;
    first = min(all, (int)(threadIdx.x >> 6) * each);
    end = min(all, first + each);
  }
  // The elements of block b; those outside the row are -infinity, and so is NaN.
  __device__ __forceinline__ void read(int b, float (&x)[E::kCount]) const {
    const int at = b * E::kCount - lead;
    if (at >= 0 && at + E::kCount <= vocab) {
      E::take(*reinterpret_cast<const uintx4 *>(blocks + (long long)b * 16), x);
    } else {
#pragma unroll
      for (int i = 0; i < E::kCount; ++i)
        x[i] = at + i >= 0 && at + i < vocab ? E::one(blocks + (long long)b * 16 + i * E::kBytes) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < E::kCount; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
  }
  // f(x) of every element of the wave's share, in any order
  template <typename F>
  __device__ __forceinline__ void each(const F &f) const {
    for (int b = first + (threadIdx.x & 63); b < end; b += 64) {
      float x[E::kCount];
      read(b, x);
#pragma unroll
      for (int i = 0; i < E::kCount; ++i) f(x[i]);
    }
  }
};

// Counts and weights of BINS bins become sums of those up to and with each.  Ends with a barrier.
template <int BINS>
__device__ __forceinline__ void running_sums(u64 (&weights)[BINS], uint32_t (&counts)[BINS], Shared &s) {
  constexpr int kEach = BINS / kThreads;
  const int tid = threadIdx.x, wave = tid >> 6;
  u64 w[kEach], w_sum = 0;
  uint32_t c[kEach], c_sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    w[i] = w_sum += weights[tid * kEach + i];
    c[i] = c_sum += counts[tid * kEach + i];
  }
  u64 w_before = wave_inclusive_sum(w_sum);
  uint32_t c_before = wave_inclusive_sum(c_sum);
  if ((tid & 63) == 63) {
    s.wave_weights[wave] = w_before;
    s.wave_counts[wave] = c_before;
  }
  w_before -= w_sum;
  c_before -= c_sum;
  __syncthreads();
  for (int i = 0; i < wave; ++i) {
    w_before += s.wave_weights[i];
    c_before += s.wave_counts[i];
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    weights[tid * kEach + i] = w_before + w[i];
    counts[tid * kEach + i] = c_before + c[i];
  }
  __syncthreads();
}

// The first bin up to whose end there are `amount` tokens, or as much weight: into s.found, with what lies before it and in it.  Ends with a barrier.
template <int BINS>
__device__ __forceinline__ void find(const u64 (&weights)[BINS], const uint32_t (&counts)[BINS], bool by_count, u64 amount, Shared &s) {
  for (int b = threadIdx.x; b < BINS; b += kThreads) {
    const u64 w0 = b ? weights[b - 1] : 0, w1 = weights[b];
    const uint32_t c0 = b ? counts[b - 1] : 0, c1 = counts[b];
    if (by_count ? c0 < amount && amount <= c1 : w0 < amount && amount <= w1) {
      s.found = b;
      s.before_weight = w0;
      s.before_count = c0;
      s.at_weight = w1 - w0;
      s.at_count = c1 - c0;
    }
  }
  __syncthreads();
}

// The logit at which the running count, or the running sum of the weights, reaches `amount` (at least one, and no more than there is).
template <typename T>
__device__ Place locate(const Reader<T> &reader, const Row &row, float to_bin, bool by_count, u64 amount, Shared &s) {
  if (threadIdx.x == 0) {
    s.low = 0xffffffffu;
    s.high = 0;
  }
  find(s.weights, s.counts, by_count, amount, s);
  const int bin = s.found;
  Place place;
  place.before_count = s.before_count;
  place.before_weight = s.before_weight;
  place.tokens = s.at_count;
  u64 inside = s.at_weight;
  uint32_t low = 0xffffffffu, high = 0;
  reader.each([&](float x) {
    double z;
    if (row.candidate(x, z) && min((int)((float)z * to_bin), kBins - 1) == bin) {
      low = min(low, key_of(x));
      high = max(high, key_of(x));
    }
  });
  if (low <= high) {
    atomicMin(&s.low, low);
    atomicMax(&s.high, high);
  }
  __syncthreads();
  low = s.low;
  high = s.high;
  __syncthreads();
  while (low < high) {
    const int shift = max(0, 22 - (int)__builtin_clz(high - low));  // (high - low) >> shift is below kFine
    for (int b = threadIdx.x; b < kFine; b += kThreads) {
      s.fine_weights[b] = 0;
      s.fine_counts[b] = 0;
    }
    __syncthreads();
    reader.each([&](float x) {
      double z;
      const uint32_t key = key_of(x);
      if (key >= low && key <= high && row.candidate(x, z)) {
        const uint32_t b = (high - key) >> shift;
        atomicAdd(&s.fine_counts[b], 1u);
        atomicAdd(&s.fine_weights[b], row.weight(z));
      }
    });
    __syncthreads();
    running_sums(s.fine_weights, s.fine_counts, s);
    find(s.fine_weights, s.fine_counts, by_count, by_count ? amount - place.before_count : amount - place.before_weight, s);
    place.before_count += s.before_count;
    place.before_weight += s.before_weight;
    place.tokens = s.at_count;
    inside = s.at_weight;
    const uint32_t from = high - ((uint32_t)s.found << shift), rest = (1u << shift) - 1u;
    high = from;
    low = max(low, from - min(from, rest));
    __syncthreads();
  }
  place.key = low;
  place.weight = inside / place.tokens;  // (tokens of one logit weigh the same)
  return place;
}

// The index of the token number `which` among those of one logit.
template <typename T>
__device__ int index_of(const Reader<T> &reader, uint32_t key, uint32_t which, Shared &s) {
  constexpr int kCount = Elements<T>::kCount;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t mine = 0;
  reader.each([&](float x) { mine += x > -INFINITY && key_of(x) == key; });
  mine = wave_inclusive_sum(mine);
  if (lane == 63) s.wave_counts[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s.wave_counts[i];
  if (which >= before && which < before + s.wave_counts[wave]) {
    uint32_t left = which - before;
    for (int b = reader.first; b < reader.end; b += 64) {
      float x[kCount];
      uint32_t here = 0;
      if (b + lane < reader.end) {
        reader.read(b + lane, x);
#pragma unroll
        for (int i = 0; i < kCount; ++i) here += x[i] > -INFINITY && key_of(x[i]) == key;
      }
      const uint32_t upto = wave_inclusive_sum(here), all = from_last_lane(upto);
      if (left < all) {
        uint32_t skip = left - (upto - here);  // (of this lane's)
        if (left >= upto - here && left < upto) {
#pragma unroll
          for (int i = 0; i < kCount; ++i)
            if (x[i] > -INFINITY && key_of(x[i]) == key && skip-- == 0) s.token = (b + lane) * kCount - reader.lead + i;
        }
        break;
      }
      left -= all;
    }
  }
  __syncthreads();
  return s.token;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_tokens_kernel(const SampleArgs p) {
  __shared__ Shared s;
  const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const Reader<T> reader(static_cast<const unsigned char *>(p.logits) + (long long)r * p.stride * Elements<T>::kBytes, p.vocab);
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float u = fminf(fmaxf(p.uniform[r], 0.f), 0x1.fffffep-1f);  // (NaN: 0)

  for (int b = tid; b < kBins; b += kThreads) {
    s.weights[b] = 0;
    s.counts[b] = 0;
  }
  float most = -INFINITY;
  reader.each([&](float x) { most = fmaxf(most, x); });
  most = wave_max_all(most);
  if ((tid & 63) == 0) s.wave_counts[wave] = __float_as_uint(most);
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) most = fmaxf(most, __uint_as_float(s.wave_counts[i]));
  __syncthreads();

  int token = -1;
  float probability = 0.f;
  if (most == -INFINITY) {  // (nothing may be drawn)
  } else if (!(temperature > 0.f) || top_k == 1) {
    token = index_of(reader, key_of(most), 0, s);
    probability = 1.f;
  } else {
    const int unit_bits = min(52, 31 + __builtin_clz(max(p.vocab - 1, 1)) - 1);  // vocab << unit_bits is no more than 2^62
    Row row;
    row.most = most;
    row.per_logit = 1.0 / (double)temperature;
    row.unit = (double)(1ull << unit_bits);
    const double all = (unit_bits + 1) * 0.6931471805599453;
    row.farthest = min_p > 0.f ? fmin(all, -log((double)fminf(min_p, 1.f))) : all;
    const float to_bin = (float)(kBins / all);
    reader.each([&](float x) {
      double z;
      if (row.candidate(x, z)) {
        const int b = min((int)((float)z * to_bin), kBins - 1);
        atomicAdd(&s.counts[b], 1u);
        atomicAdd(&s.weights[b], row.weight(z));
      }
    });
    __syncthreads();
    running_sums(s.weights, s.counts, s);
    u64 total = s.weights[kBins - 1];
    // sums of `amount` and more end at the place's first tokens that reach it
    const auto upto = [&](const Place &place, u64 amount) {
      const u64 n = (amount - place.before_weight + place.weight - 1) / place.weight;
      return place.before_weight + min(n, (u64)place.tokens) * place.weight;
    };
    if (top_k > 0 && (uint32_t)top_k < s.counts[kBins - 1]) {
      const Place place = locate(reader, row, to_bin, true, (u64)top_k, s);
      total = place.before_weight + (u64)((uint32_t)top_k - place.before_count) * place.weight;
    }
    if (top_p < 1.f) {
      const u64 amount = min(max((u64)ceil((double)fmaxf(top_p, 0.f) * (double)total), (u64)1), total);
      total = upto(locate(reader, row, to_bin, false, amount, s), amount);
    }
    const u64 amount = min((u64)((double)u * (double)total) + 1, total);
    const Place place = locate(reader, row, to_bin, false, amount, s);
    token = index_of(reader, place.key, (uint32_t)((amount - place.before_weight - 1) / place.weight), s);
    probability = (float)((double)place.weight / (double)total);
  }
  if (tid == 0) {
    p.tokens[r] = token;
    if (p.probabilities) p.probabilities[r] = probability;
  }
}

template <typename T>
hipError_t launch(const SampleArgs &a, hipStream_t stream) {
  hipLaunchKernelGGL((sample_tokens_kernel<T>), dim3(a.rows), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample_tokens(int type, const SampleArgs &args, hipStream_t stream) {
  return type == 0 ? launch<Fp16>(args, stream) : type == 1 ? launch<Bf16>(args, stream) : launch<F32>(args, stream);
}

}  // namespace sspmm
