// Tokens drawn from rows of logits l with given uniform numbers u.  With z_i = (max l - l_i) / T a token's weight is w_i = exp(-z_i); kept are those with
// w_i >= min_p, of these the top_k first in the order of falling logits (equal ones in the order of their indices), of these the shortest run whose weights
// reach top_p of all of theirs.  The token is the first in that order at which the running sum of the weights exceeds u times their sum.
//
// Weights are 2^-(n / 16) times whole numbers, n the nearest to 16 z log2(e): the whole numbers, in units of 2^-unit_bits, are summed for each n, in bins, and a bin's sum is
// brought to units of the largest's weight as a whole. Sums of whole numbers are exact in any order, so that atomics and lanes give the same token every time.
// Vocabularies of 2^17 leave 45 bits.
//
// No row is sorted.  With a top_k of some hundred, the largest logit of every thread's share gives a logit that enough others reach; those that reach it become a list
// in LDS, and the draw is the list's.  Else the row is put into bins by z, which is to say by weight; where a sum ends is then known up to a bin, and the logits of the few
// bins that matter become the list.  A bin is split by its logits until one logit is left, and equal logits by their indices.  Where the list has no room, the row
// in memory stands in its place.
//
// What bounds it: a row is read three times (its largest logit, its bins, its list), the second and third time from the caches; 256 rows of 2^17 bf16 logits, a row a CU: 18 us
// greedy (3.7 TB/s), 79 us with no limit, of which the weights in 64 bits and their atomics are some 26 (22 and 9 cycles a CU for 64 logits); 92 us with top_p, whose second
// sum reads its list again; 29 with a top_k of 50, which needs no bins of the row and reads it once, 53 with one of 1000, which reads it twice.  Few rows are bound by the chain of steps: a row of 2000
// takes 5 us greedy, 10 with no limit, 13 with top_p and top_k.
#include "sample_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

typedef unsigned long long u64;

// Threads of a workgroup (N, below).
constexpr int kThreads = 512, kManyThreads = 1024;
constexpr int kBins = 1024;                // of a row or its list, the last one for what weighs nothing
constexpr int kList = 6144;                // logits of a list
// The largest top_k that the threads' four large ones give a bound for; above it rows have bins.  By a list and by bins, us: 30 rows of 5000 logits, top_k of 1200 28 and 25, 30 of 20000
// 32 and 31, 200 of 50000 37 and 43, 64 of 131072 37 and 61, 384 of 100003 (fp32) 91 and 126; top_k of 2000 34 and 25, 42 and 33, 44 and 45, 41 and 62, 115 and 127.
constexpr int kMostTopK = 1200;

struct F32 {};

template <typename T>
struct Elements {  // of 16 bytes
  static constexpr int kCount = 8, kBytes = 2;
  static constexpr int kGrain = __is_same(T, Bf16) ? 16 : 13;  // bits at the end that are the same in all logits of one sign, taken as 32 bits
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
  static constexpr int kCount = 4, kBytes = 4, kGrain = 0;
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
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key ^ ((uint32_t)((int32_t)~key >> 31) | 0x80000000u)); }

// What a row is drawn with.
struct Setting {
  float temperature, top_p, min_p;
  int top_k;  // 0: all
  int unit_bits;
  bool greedy;
  __device__ __forceinline__ Setting(const SampleArgs &p, int r) {
    temperature = p.temperature ? p.temperature[r] : p.temperature_all;
    top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    if (top_k < 0 || top_k >= p.vocab) top_k = 0;
    greedy = !(temperature > 0.f) || top_k == 1;
    if (greedy) top_k = 1;
    unit_bits = min(50, 30 + __builtin_clz(max(p.vocab - 1, 1)));  // vocab << unit_bits is no more than 2^62
  }
  __device__ __forceinline__ bool few() const { return top_k > 0 && top_k <= kMostTopK; }
};

struct Weights {
  double most, per_logit, farthest;  // the largest logit; 16 log2(e) / T; largest 16 z log2(e) of a token that is kept
  double unit;                       // 2^unit_bits
  bool infinite, everything;
  __device__ __forceinline__ Weights(const Setting &s, float largest) {
    most = (double)largest;
    per_logit = 16.0 * 1.4426950408889634 / (double)s.temperature;
    unit = (double)(1ull << s.unit_bits);
    everything = !(s.min_p > 0.f);
    farthest = everything ? (double)(kBins - 1) : -16.0 * log2((double)fminf(s.min_p, 1.f));
    infinite = largest == INFINITY;
  }
  // 16 z log2(e).  (Monotone in x, so that bins and ranges of logits never cross; -infinity, NaN and what is farther than 2^-63 go to the last bin.)
  __device__ __forceinline__ double distance(float x) const {
    const double y = fmin((most - (double)x) * per_logit, (double)(kBins - 1));
    return everything || y <= farthest ? y : (double)(kBins - 1);
  }
  // Its bin, and in it 2^(n - y) / 16) in units: with f = n - y, 1 + f g(f), g a polynomial through its Chebyshev points in -1/2 .. 1/2, off by 2^-46.  Adding 2^52 leaves the
  // whole number in the lower bits.
  __device__ __forceinline__ int units(double y, u64 &w) const {
    const double shifted = y + 0x1.8p52, n = shifted - 0x1.8p52, f = n - y;
    double g = 0x1.5d893e591a8aap-30 * unit;
    g = fma(g, f, 0x1.3b2c4ac7da6fep-23 * unit);
    g = fma(g, f, 0x1.c6b08d6faa1acp-17 * unit);
    g = fma(g, f, 0x1.ebfbdff6988c8p-11 * unit);
    g = fma(g, f, 0x1.62e42fefa39efp-5 * unit);
    w = (u64)__double_as_longlong(fma(g, f, unit + 0x1p52)) - 0x4330000000000000ull;
    return (int)(uint32_t)__double_as_longlong(shifted);
  }
  // The same of any logit (where the largest is infinite, it alone weighs something).
  __device__ __forceinline__ int of(float x, u64 &w) const {
    const double y = distance(x);
    return units(infinite ? ((double)x == most ? 0.0 : (double)(kBins - 1)) : y, w);
  }
  // A bin's units as units of the largest's weight.
  __device__ __forceinline__ double share(int bin) const { return exp2(-(double)bin / 16.0); }
  __device__ __forceinline__ u64 whole(int bin, u64 inside) const { return (u64)rint((double)inside * share(bin)); }
  // A logit that no logit of bin b and those before it is below (or, from the side of 0, above), whatever was rounded on the way.
  __device__ __forceinline__ float lowest(int b) const {
    if (infinite) return -INFINITY;
    const double x = most - ((double)b + 0.5) * 1.000001 / per_logit;
    return (float)(x - (fabs(x) * 0x1p-22 + 1e-44));
  }
  __device__ __forceinline__ float highest(int b) const {
    if (b == 0 || infinite) return INFINITY;
    const double x = most - ((double)b - 0.5) * 0.999999 / per_logit;
    return (float)(x + (fabs(x) * 0x1p-22 + 1e-44));
  }
};

// A logit that none which weighs something beside the largest is below: z of the last bin but one ends at (kBins - 3/2) / (16 log2(e)), 44.3.
__device__ __forceinline__ float least_of(const Setting &s, float largest) {
  const float x = fmaf(-44.4f, s.temperature, largest);
  return s.greedy ? largest : largest == INFINITY ? -INFINITY : x - fmaf(fabsf(x), 0x1p-20f, 1e-44f);
}

struct Bins {
  u64 inside[kBins];   // units of the bin
  u64 weights[kBins];  // units of the largest, of this bin and those before
  uint32_t counts[kBins];
};
template <int N>
struct Shared {
  Bins bins;
  u64 fine_weights[N];  // of a range of logits, or of indices
  __align__(16) uint32_t fine_counts[N];
  uint32_t keys[kList], indices[kList];
  u64 wave_weights[N / 64];
  uint32_t wave_counts[N / 64];
  uint32_t low, high, listed, alike;
  int at;
  u64 before_weight, at_weight;
  uint32_t before_count, at_count;
};
// How far a range that ends `span` further is shifted to leave numbers below N.
template <int N>
__device__ __forceinline__ int shift_of(uint32_t span) {
  return max(0, 32 - __builtin_ctz(N) - (int)__builtin_clz(span));
}

// A row in memory, or one of the parts that its lines of 128 bytes are dealt to in turn: tokens that are likely often stand side by side, a vocabulary's first ones for
// instance, and a part that had them all would list too few of them (64 rows of 131072 whose first tokens are likely, top_k of 100: 22 us, by parts of one stretch each 114).
template <typename T>
struct RowReader {
  typedef Elements<T> E;
  static constexpr int kGrain = E::kGrain;
  static constexpr int kLine = 8;  // blocks of 16 bytes of a line
  static constexpr int kLineLogits = kLine * E::kCount;
  const unsigned char *row;  // aligned to an element
  int vocab, lead;           // elements; those in front of the row in the line that holds its first one, from where on blocks are counted
  int first, end;            // of the part's blocks, counted as if they lay side by side, those that lie whole in the row
  int part, parts;
  __device__ __forceinline__ RowReader(const void *row_, int vocab_, int part_, int parts_) {
    row = static_cast<const unsigned char *>(row_);
    vocab = vocab_;
    part = part_;
    parts = parts_;
    lead = (int)(reinterpret_cast<uintptr_t>(row_) & (16 * kLine - 1)) / E::kBytes;
    const int whole = (int)(((long long)vocab + lead) / E::kCount), lines = whole / kLine;
    first = part == 0 ? (lead + E::kCount - 1) / E::kCount : 0;  // (a line's at most)
    end = max(first, (lines - part + parts - 1) / parts * kLine + (lines % parts == part ? whole % kLine : 0));
  }
  // Where the part's block number i lies.
  __device__ __forceinline__ int place(int i) const { return parts == 1 ? i : (i / kLine * parts + part) * kLine + i % kLine; }
  __device__ __forceinline__ float one(int i) const { return E::one(row + (long long)i * E::kBytes); }
  // f(logit, index, place in its block) of the elements of the part's block number i
  template <typename F>
  __device__ __forceinline__ void block(int i, const F &f) const {
    const int b = place(i);
    float x[E::kCount];
    E::take(*reinterpret_cast<const uintx4 *>(row - lead * E::kBytes + (long long)b * 16), x);
#pragma unroll
    for (int j = 0; j < E::kCount; ++j) f(x[j], b * E::kCount - lead + j, j);
  }
  // of what lies in front of the row's whole blocks and behind them, an element a thread: the first part's
  template <typename F>
  __device__ __forceinline__ void edge(const F &f) const {
    if (part != 0) return;
    const int blocks = (lead + E::kCount - 1) / E::kCount, whole = (int)(((long long)vocab + lead) / E::kCount);
    const int tid = threadIdx.x, head_end = min(vocab, blocks * E::kCount - lead), tail = max(head_end, whole * E::kCount - lead);
    const int i = tid < head_end ? tid : tail + tid - head_end;
    if (i < vocab) f(one(i), i, 0);
  }
  // and of every element, in any order
  template <int UNROLL = 1, typename F>
  __device__ __forceinline__ void each(const F &f) const {
#pragma unroll UNROLL
    for (int i = first + (int)threadIdx.x; i < end; i += (int)blockDim.x) block(i, f);
    edge(f);
  }
};

template <typename T>
struct ListReader {
  static constexpr int kGrain = Elements<T>::kGrain;
  const uint32_t *keys, *indices;
  int count;
  template <int UNROLL = 1, typename F>
  __device__ __forceinline__ void each(const F &f) const {
    for (int i = threadIdx.x; i < count; i += (int)blockDim.x) f(logit_of(keys[i]), (int)indices[i], 0);
  }
};

// Sum of v over the threads in front of the own one; and, in `all`, over all.  Two barriers.
template <typename V, int W>
__device__ __forceinline__ V sum_before(V v, V (&waves)[W], V &all) {
  const int wave = threadIdx.x >> 6;
  const V upto = wave_inclusive_sum(v);
  if ((threadIdx.x & 63) == 63) waves[wave] = upto;
  __syncthreads();
  V before = upto - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const V w = waves[i];
    before += i < wave ? w : 0;
    all += w;
  }
  __syncthreads();
  return before;
}

// Sums of weights and counts up to and with each bin, of given weights and the counts that stand there.  Ends with a barrier.
template <int BINS, int N>
__device__ __forceinline__ void running_sums(const u64 (&given)[BINS / N], u64 (&weights)[BINS], uint32_t (&counts)[BINS], Shared<N> &s) {
  constexpr int kOwn = BINS / N;
  const int tid = threadIdx.x, wave = tid >> 6;
  u64 w[kOwn], w_sum = 0;
  uint32_t c[kOwn], c_sum = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    w[i] = w_sum += given[i];
    c[i] = c_sum += counts[tid * kOwn + i];
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
#pragma unroll
  for (int i = 0; i < N / 64; ++i) {
    w_before += i < wave ? s.wave_weights[i] : 0;
    c_before += i < wave ? s.wave_counts[i] : 0;
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    weights[tid * kOwn + i] = w_before + w[i];
    counts[tid * kOwn + i] = c_before + c[i];
  }
  __syncthreads();
}
// Of a row's bins.
template <int N>
__device__ __forceinline__ void sum_bins(const Weights &weights, Shared<N> &s) {
  u64 whole[kBins / N];
#pragma unroll
  for (int i = 0; i < kBins / N; ++i) {
    const int b = threadIdx.x * (kBins / N) + i;
    whole[i] = weights.whole(b, s.bins.inside[b]);
  }
  running_sums<kBins>(whole, s.bins.weights, s.bins.counts, s);
}

// The first bin up to whose end there are `amount` tokens, or as much weight: into s.at, with what lies before it and in it.  Ends with a barrier.
template <int BINS, int N>
__device__ __forceinline__ void find(const u64 (&weights)[BINS], const uint32_t (&counts)[BINS], bool by_count, u64 amount, Shared<N> &s) {
  for (int b = threadIdx.x; b < BINS; b += N) {
    const u64 w0 = b ? weights[b - 1] : 0, w1 = weights[b];
    const uint32_t c0 = b ? counts[b - 1] : 0, c1 = counts[b];
    if (by_count ? c0 < amount && amount <= c1 : w0 < amount && amount <= w1) {
      s.at = b;
      s.before_weight = w0;
      s.before_count = c0;
      s.at_weight = w1 - w0;
      s.at_count = c1 - c0;
    }
  }
  __syncthreads();
}

// A place in the order: the logit, its bin, what lies before its first token (tokens; units before the bin, and units of the bin), its tokens, and units of the bin of each.
struct Place {
  uint32_t key, before_count, tokens;
  int bin;
  u64 before_bin, before_inside, weight;
};
// A place after so many of its tokens: weight of all up to there, and units of its bin.
struct End {
  int bin;
  u64 total, inside;
};
__device__ __forceinline__ End end_at(const Weights &weights, const Place &place, u64 tokens) {
  const u64 inside = place.before_inside + tokens * place.weight;
  return {place.bin, place.before_bin + weights.whole(place.bin, inside), inside};
}

// The logit at which the running count, or the running sum of the weights, reaches `amount` (at least one, and no more than there is), and how much that is in units of its bin, which
// are at least one, and no more than there are: in the bin, or in what is kept of it.
template <typename Reader, int N>
__device__ __forceinline__ Place locate(const Reader &reader, const Weights &weights, bool by_count, u64 amount, const End &kept, u64 &inside, Shared<N> &s) {
  __syncthreads();
  if (threadIdx.x == 0) {
    s.low = 0xffffffffu;
    s.high = 0;
  }
  find(s.bins.weights, s.bins.counts, by_count, amount, s);
  Place place;
  place.bin = s.at;
  place.before_count = s.before_count;
  place.before_bin = s.before_weight;
  place.before_inside = 0;
  u64 in_all = s.bins.inside[place.bin];
  if (by_count) {
    inside = 0;
  } else {
    // (units of the largest's weight are the first bin's own: as they are, since 53 bits lose the one that u times equal weights is to be exceeded by)
    const u64 rest = amount - place.before_bin;
    inside = place.bin == 0 ? rest : max((u64)ceil((double)rest / weights.share(place.bin)), (u64)1);
    inside = min(inside, place.bin == kept.bin ? min(kept.inside, in_all) : in_all);
  }
  uint32_t low = 0xffffffffu, high = 0, count = 0;
  const float from = weights.lowest(place.bin), to = weights.highest(place.bin);
  reader.template each<2>([&](float x, int, int) {
    if (x >= from && x <= to) {
      u64 w;
      if (weights.of(x, w) == place.bin) {
        low = min(low, key_of(x));
        high = max(high, key_of(x));
        ++count;
      }
    }
  });
  if (low <= high) {
    atomicMin(&s.low, low);
    atomicMax(&s.high, high);
  }
  sum_before(count, s.wave_counts, place.tokens);  // (two barriers)
  low = s.low;
  high = s.high;
  while (low < high) {
    // (no finer than the type: with 16 bits a bin has few logits, and one round finds the right one)
    const int shift = max(shift_of<N>(high - low), Reader::kGrain);
    s.fine_weights[threadIdx.x] = 0;
    s.fine_counts[threadIdx.x] = 0;
    __syncthreads();
    reader.each([&](float x, int, int) {
      const uint32_t key = key_of(x);
      if (key >= low && key <= high) {
        u64 w;
        if (weights.of(x, w) == place.bin) {
          atomicAdd(&s.fine_counts[(high - key) >> shift], 1u);
          atomicAdd(&s.fine_weights[(high - key) >> shift], w);
        }
      }
    });
    __syncthreads();
    const u64 fine[1] = {s.fine_weights[threadIdx.x]};
    running_sums<N>(fine, s.fine_weights, s.fine_counts, s);
    find(s.fine_weights, s.fine_counts, by_count, by_count ? amount - place.before_count : inside - place.before_inside, s);
    place.before_count += s.before_count;
    place.before_inside += s.before_weight;
    place.tokens = s.at_count;
    in_all = s.at_weight;
    const uint32_t first = high - ((uint32_t)s.at << shift), rest = (1u << shift) - 1u;
    if (shift == Reader::kGrain) {  // one logit (a negative one ends in ones, the others in zeros)
      low = high = Reader::kGrain > 0 && first < 0x80000000u && (first & rest) == 0 ? first - 1 : first;
    } else {
      high = first;
      low = max(low, first - min(first, rest));
    }
    __syncthreads();
  }
  place.key = low;
  place.weight = in_all / place.tokens;  // (tokens of one logit weigh the same)
  return place;
}

constexpr uint32_t kFewAlike = 256;  // (ranked by the first four waves at a time; 512 by eight cost 256 rows of 131072 83 us instead of 78)
// The index of the token number `which` among those of one logit: of few, by counting the smaller ones; else the range of indices is split as ranges of logits are.
template <typename Reader, int N>
__device__ __forceinline__ int index_of(const Reader &reader, uint32_t key, uint32_t which, int vocab, Shared<N> &s) {
  s.fine_counts[threadIdx.x] = 0xffffffffu;
  if (threadIdx.x == 0) s.alike = 0;
  __syncthreads();
  reader.each([&](float x, int i, int) {
    if (key_of(x) == key) {
      const uint32_t at = atomicAdd(&s.alike, 1u);
      if (at < N) s.fine_counts[at] = (uint32_t)i;
    }
  });
  __syncthreads();
  const uint32_t those = s.alike;
  if (those <= kFewAlike) {
    if (threadIdx.x < those) {
      const uint32_t own = s.fine_counts[threadIdx.x];
      uint32_t smaller = 0;
      for (uint32_t i = 0; i < those; i += 4) {
        const uintx4 four = *reinterpret_cast<const uintx4 *>(&s.fine_counts[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) smaller += four[j] < own;
      }
      if (smaller == which) s.at = (int)own;
    }
    __syncthreads();
    return s.at;
  }
  uint32_t low = 0, high = (uint32_t)vocab - 1;
  while (low < high) {
    const int shift = shift_of<N>(high - low);
    s.fine_counts[threadIdx.x] = 0;
    __syncthreads();
    reader.each([&](float x, int i, int) {
      if (key_of(x) == key && (uint32_t)i >= low && (uint32_t)i <= high) atomicAdd(&s.fine_counts[((uint32_t)i - low) >> shift], 1u);
    });
    __syncthreads();
    uint32_t all;
    const uint32_t own = s.fine_counts[threadIdx.x], before = sum_before(own, s.wave_counts, all);
    if (which >= before && which < before + own) {
      s.at = threadIdx.x;
      s.before_count = before;
    }
    __syncthreads();
    which -= s.before_count;
    const uint32_t from = low + ((uint32_t)s.at << shift);
    high = min(high, from + ((1u << shift) - 1u));
    low = from;
    __syncthreads();
  }
  return (int)low;
}

// The reader's logits into the bins.  counted: tokens, too.  Ends with a barrier.
template <typename Reader, int N>
__device__ __forceinline__ void fill_bins(const Reader &reader, const Weights &weights, bool counted, Shared<N> &s) {
  for (int b = threadIdx.x; b < kBins; b += N) {
    s.bins.inside[b] = 0;
    s.bins.counts[b] = 0;
  }
  __syncthreads();
  if (counted || weights.infinite)
    reader.each([&](float x, int, int) {
      u64 w;
      const int b = weights.of(x, w);
      if (b < kBins - 1) {
        atomicAdd(&s.bins.counts[b], 1u);
        atomicAdd(&s.bins.inside[b], w);
      }
    });
  else
    reader.each([&](float x, int, int) {
      u64 w;
      const int b = weights.units(weights.distance(x), w);
      if (b < kBins - 1) atomicAdd(&s.bins.inside[b], w);
    });
  __syncthreads();
}

__device__ __forceinline__ u64 top_p_amount(float top_p, u64 total) { return min(max((u64)ceil((double)fmaxf(top_p, 0.f) * (double)total), (u64)1), total); }
__device__ __forceinline__ u64 drawn_amount(float u, u64 total) { return min((u64)((double)u * (double)total) + 1, total); }

// The draw, with the row's sums in s.bins; of the bins in which the sums that it asks for end, the reader has the logits.
template <typename Reader, int N>
__device__ __forceinline__ void draw(const Reader &reader, const Setting &setting, const Weights &weights, float u, int vocab, Shared<N> &s, int &token, float &probability) {
  End kept = {-1, s.bins.weights[kBins - 1], 0};
  u64 inside;
  if (setting.top_k > 0 && (uint32_t)setting.top_k < s.bins.counts[kBins - 1]) {
    const Place place = locate(reader, weights, true, (u64)setting.top_k, kept, inside, s);
    kept = end_at(weights, place, (u64)((uint32_t)setting.top_k - place.before_count));
  }
  if (setting.top_p < 1.f) {
    const Place place = locate(reader, weights, false, top_p_amount(setting.top_p, kept.total), kept, inside, s);
    // (the first of its tokens that reaches the amount is the last one kept)
    kept = end_at(weights, place, (inside - place.before_inside + place.weight - 1) / place.weight);
  }
  const Place place = locate(reader, weights, false, drawn_amount(u, kept.total), kept, inside, s);
  token = index_of(reader, place.key, (uint32_t)((inside - place.before_inside - 1) / place.weight), vocab, s);
  probability = (float)((double)place.weight * weights.share(place.bin) / (double)kept.total);
}

// A logit onto the list, as far as it has room; s.listed counts all.
template <int N>
__device__ __forceinline__ void list(float x, int i, Shared<N> &s) {
  const uint32_t at = atomicAdd(&s.listed, 1u);
  if (at < kList) {
    s.keys[at] = key_of(x);
    s.indices[at] = (uint32_t)i;
  }
}

// Ranges of logits.
struct Ranges {
  float from[3], to[3];
};

// Those of the bins in which what draw() asks for may end, as far as the sums in s.bins say.  Ends with a barrier.
template <int N>
__device__ __forceinline__ Ranges ends_of(const Setting &setting, const Weights &weights, float u, Shared<N> &s) {
  Ranges r = {{INFINITY, INFINITY, INFINITY}, {-INFINITY, -INFINITY, -INFINITY}};
  u64 least = s.bins.weights[kBins - 1], most = least;  // that the kept tokens weigh
  const auto ends = [&](float &from, float &to, bool by_count, u64 first, u64 last) {  // bins in which sums of first .. last end
    find(s.bins.weights, s.bins.counts, by_count, first, s);
    const int low = s.at;
    least = max(s.before_weight, (u64)1);
    __syncthreads();
    find(s.bins.weights, s.bins.counts, by_count, last, s);
    const int high = s.at;
    most = s.before_weight + s.at_weight;
    __syncthreads();
    from = weights.lowest(high);
    to = weights.highest(low);
  };
  if (setting.top_k > 0 && (uint32_t)setting.top_k < s.bins.counts[kBins - 1]) ends(r.from[0], r.to[0], true, (u64)setting.top_k, (u64)setting.top_k);
  if (setting.top_p < 1.f) ends(r.from[1], r.to[1], false, top_p_amount(setting.top_p, least), top_p_amount(setting.top_p, most));
  ends(r.from[2], r.to[2], false, drawn_amount(u, least), drawn_amount(u, most));
  return r;
}

// The reader's logits in these ranges become the list.  Ends with a barrier.
template <typename Reader, int N>
__device__ __forceinline__ void list_ranges(const Reader &reader, const Ranges &r, Shared<N> &s) {
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  reader.template each<4>([&](float x, int i, int) {
    const bool a = x >= r.from[0] && x <= r.to[0], b = x >= r.from[1] && x <= r.to[1], c = x >= r.from[2] && x <= r.to[2];
    if (a || b || c) list(x, i, s);
  });
  __syncthreads();
}

// The largest of the reader's logits, -infinity if there is none.
template <typename Reader, int N>
__device__ __forceinline__ float largest_of(const Reader &reader, Shared<N> &s) {
  float most = -INFINITY;
  reader.template each<4>([&](float x, int, int) { most = fmaxf(most, x); });
  most = wave_max_all(most);
  if ((threadIdx.x & 63) == 0) s.wave_counts[threadIdx.x >> 6] = __float_as_uint(most);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N / 64; ++i) most = fmaxf(most, __uint_as_float(s.wave_counts[i]));
  __syncthreads();
  return most;
}

// The first `wanted` of the reader's logits, and others, onto the list: those that reach a logit which so many of the threads' largest reach, but for what weighs nothing beside
// the largest (tokens ruled out by a low number instead of -infinity would fill it: 64 rows of 131072 with some 20 others, top_k of 50 23 us instead of 146; with -infinity 17).  Its number, or
// 0 where the list has all that weighs something.  Ends with a barrier.
template <typename T, int N>
__device__ __forceinline__ uint32_t list_first(const RowReader<T> &reader, const Setting &setting, uint32_t wanted, float &largest, Shared<N> &s) {
  const int tid = threadIdx.x;
  constexpr int kPairs = 2;  // (the largest and the one behind it, of the even and of the odd places of all blocks)
  // (Where first ones stand side by side, a list has all logits of as many blocks, and the parts' lists have to fit one: 64 sorted rows of 131072 in bf16, top_k of 200, 38 us, and
  // 288 with lists that do not.  In any order one a thread takes 21.7 us there and four 25.1.)
  const bool one = wanted <= min(N / 4, (kList - kFewAlike) / (RowReader<T>::E::kCount * reader.parts));
  float large[2 * kPairs];
#pragma unroll
  for (float &x : large) x = -INFINITY;
  if (one)
    reader.template each<4>([&](float x, int, int) { large[0] = fmaxf(large[0], x); });
  else
    reader.template each<2>([&](float x, int, int place) {
      x = x == x ? x : -INFINITY;
      float &first = large[2 * (place % kPairs)], &second = large[2 * (place % kPairs) + 1];
      second = fmaxf(second, fminf(first, x));
      first = fmaxf(first, x);
    });
  // ---- bins of equal width from the smallest of these to the largest
  if (tid == 0) {
    s.low = s.high = 0;
    s.at = N;
    s.listed = 0;
  }
  s.fine_counts[tid] = 0;
  __syncthreads();
  float most = -INFINITY, least = INFINITY;  // of the finite ones
#pragma unroll
  for (float x : large) {
    most = fmaxf(most, x);
    least = x > -INFINITY ? fminf(least, x) : least;
  }
  most = wave_max_all(most);
  least = -wave_max_all(-least);
  if ((tid & 63) == 0) {
    atomicMax(&s.high, key_of(most));
    atomicMax(&s.low, ~key_of(least));
  }
  __syncthreads();
  const float top = logit_of(s.high), bottom = logit_of(~s.low);
  const float scale = (float)(N - 1) / fmaxf(top - bottom, 1e-30f);
  const auto bin = [&](float x) { return (int)fminf(fmaxf((top - x) * scale, 0.f), (float)(N - 1)); };
#pragma unroll
  for (float x : large)
    if (x > -INFINITY) atomicAdd(&s.fine_counts[bin(x)], 1u);
  __syncthreads();
  uint32_t all;
  const uint32_t own = s.fine_counts[tid], before = sum_before(own, s.wave_counts, all);
  if (before < wanted && wanted <= before + own) s.at = tid;
  if (tid == 0) {
    s.low = 0xffffffffu;
    s.high = 0;
  }
  __syncthreads();
  const int last = s.at;
  if (last < N) {
#pragma unroll
    for (float x : large)
      if (x > -INFINITY && bin(x) <= last) atomicMin(&s.low, key_of(x));
  }
  __syncthreads();
  const float reached = last < N ? logit_of(s.low) : -INFINITY, weighs = least_of(setting, top);
  const uint32_t from = last < N && reached >= weighs ? s.low : 0;
  const float reaches = fmaxf(reached, weighs);
  const auto take = [&](float x, int i, int) {
    if (x >= reaches && x > -INFINITY) list(x, i, s);
  };
  // Where few threads' largest reach it, those threads' blocks are all that has to be read again, by all threads (256 rows of
  // 131072 in bf16, greedy 18 us instead of 27, top_k of 50 29 instead of 38, of 128 34 instead of 38).
  bool few = one && last < N;
  if (few) {
    if (large[0] >= reaches) s.fine_counts[atomicAdd(&s.high, 1u)] = (uint32_t)tid;
    __syncthreads();
    few = s.high <= N / 4;
  }
  if (few) {
    const int threads = (int)s.high, blocks = (reader.end - reader.first + N - 1) / N * threads;
    for (int j = tid; j < blocks; j += N) {
      const int i = reader.first + (int)s.fine_counts[j % threads] + N * (j / threads);
      if (i < reader.end) reader.block(i, take);
    }
    reader.edge(take);
  } else {
    reader.template each<2>(take);
  }
  __syncthreads();
  largest = top;
  return from;
}

template <typename T>
__device__ __forceinline__ const unsigned char *row_at(const SampleArgs &p, int r) {
  return static_cast<const unsigned char *>(p.logits) + (long long)r * p.stride * Elements<T>::kBytes;
}

__device__ __forceinline__ void result(const SampleArgs &p, int r, int token, float probability) {
  if (threadIdx.x == 0) {
    p.tokens[r] = token;
    if (p.probabilities) p.probabilities[r] = probability;
  }
}
__device__ __forceinline__ float uniform_of(const SampleArgs &p, int r) { return fminf(fmaxf(p.uniform[r], 0.f), 0x1.fffffep-1f); }  // (NaN: 0)

// The row's token, and it is written: from the list in s, of some bins of those in s.bins (binned) or of the row's first logits; or where there were too many for it, from the row itself.
template <typename T, int N>
__device__ __forceinline__ void finish(const SampleArgs &p, const Setting &setting, int r, const RowReader<T> &reader, float most, bool binned, bool fits, Shared<N> &s) {
  const Weights weights(setting, most);
  const ListReader<T> listed = {s.keys, s.indices, (int)s.listed};
  int token;
  float probability = 1.f;
  if (setting.greedy) {
    token = fits ? index_of(listed, key_of(most), 0, p.vocab, s) : index_of(reader, key_of(most), 0, p.vocab, s);
  } else {
    if (!binned) {
      if (fits) fill_bins(listed, weights, true, s);
      else fill_bins(reader, weights, true, s);
      sum_bins(weights, s);
    }
    if (fits) draw(listed, setting, weights, uniform_of(p, r), p.vocab, s, token, probability);
    else draw(reader, setting, weights, uniform_of(p, r), p.vocab, s, token, probability);
  }
  result(p, r, token, probability);
}

// A workgroup a row.
template <typename T, int N>
__global__ __launch_bounds__(N, 4) void sample_tokens_kernel(const SampleArgs p) {
  __shared__ Shared<N> s;
  const int r = blockIdx.x;
  const unsigned char *const row = row_at<T>(p, r);
  const RowReader<T> reader(row, p.vocab, 0, 1);
  const Setting setting(p, r);
  float most;
  if (setting.few()) list_first(reader, setting, (uint32_t)setting.top_k, most, s);
  else most = largest_of(reader, s);
  if (most == -INFINITY) {  // (nothing may be drawn)
    result(p, r, -1, 0.f);
    return;
  }
  if (!setting.few()) {
    const Weights weights(setting, most);
    fill_bins(reader, weights, setting.top_k > 0, s);
    sum_bins(weights, s);
    list_ranges(reader, ends_of(setting, weights, uniform_of(p, r), s), s);
  }
  finish(p, setting, r, reader, most, !setting.few(), s.listed <= kList, s);
}

// ---- The same where rows are few: p.parts workgroups a row, four launches, or the first and the last where no row has bins.  What they leave for each other:
constexpr int kMostParts = 8;  // (the third launch's workgroups go over all parts' bins)
struct Part {
  float most;
  uint32_t from;   // its list has the logits whose numbers are this and more
  uint32_t count;  // of its list, or more than kList
};
struct Between {
  Part *parts;          // [rows, parts]
  u64 *weights;         // [rows, parts, kBins]
  uint32_t *counts;     // the same
  uint32_t *keys, *indices;  // [rows, parts, kList]
  __host__ __device__ Between(unsigned char *at, long long rows_, int parts_) {
    weights = reinterpret_cast<u64 *>(at);
    counts = reinterpret_cast<uint32_t *>(weights + rows_ * parts_ * kBins);
    keys = counts + rows_ * parts_ * kBins;
    indices = keys + rows_ * parts_ * kList;
    parts = reinterpret_cast<Part *>(indices + rows_ * parts_ * kList);
  }
  __host__ __device__ size_t bytes(long long rows_, int parts_) const {
    return reinterpret_cast<unsigned char *>(parts + rows_ * parts_) - reinterpret_cast<unsigned char *>(weights);
  }
};

template <typename T>
__device__ __forceinline__ RowReader<T> part_of(const SampleArgs &p, int r, int part) {
  return RowReader<T>(row_at<T>(p, r), p.vocab, part, p.parts);
}
template <typename T>
__device__ __forceinline__ RowReader<T> all_of(const SampleArgs &p, int r) {
  return RowReader<T>(row_at<T>(p, r), p.vocab, 0, 1);
}
// (a lane a part)
__device__ __forceinline__ Part part_here(const SampleArgs &p, const Part *parts) {
  const int lane = threadIdx.x & 63;
  return lane < p.parts ? parts[lane] : Part{-INFINITY, 0, 0};
}
__device__ __forceinline__ float largest_of_parts(const SampleArgs &p, const Part *parts) { return wave_max_all(part_here(p, parts).most); }

// The list in s to memory.
template <int N>
__device__ __forceinline__ void leave_list(const Between &b, long long at, const Shared<N> &s) {
  const int count = min((int)s.listed, kList);
  for (int i = threadIdx.x; i < count; i += N) {
    b.keys[at * kList + i] = s.keys[i];
    b.indices[at * kList + i] = s.indices[i];
  }
}
// The parts' lists as one in s, but for logits that some part's list does not hold, and parts whose largest is below `least`; false if some part's, or all together, are too many, or
// fewer than `wanted`.  Ends with a barrier.
template <int N>
__device__ __forceinline__ bool take_lists(const SampleArgs &p, const Between &b, int r, uint32_t wanted, float least, Shared<N> &s) {
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  Part mine = part_here(p, b.parts + (long long)r * p.parts);
  if (mine.most < least) mine = {mine.most, 0, 0};
  const uint32_t from = from_last_lane(wave_inclusive_max(mine.from));
  bool fits = from_last_lane(wave_inclusive_max(mine.count)) <= (uint32_t)kList;
  const uint32_t behind = wave_inclusive_sum(min(mine.count, (uint32_t)kList)), all = from_last_lane(behind);
  const long long first = (long long)r * p.parts * kList;
#pragma unroll 2
  for (uint32_t i = threadIdx.x; i < all; i += N) {
    int part = 0;
    uint32_t before = 0;
#pragma unroll
    for (int j = 0; j < kMostParts - 1; ++j) {
      const uint32_t end = (uint32_t)__builtin_amdgcn_readlane((int)behind, j);
      part += i >= end;
      before = i >= end ? end : before;
    }
    const long long at = first + (long long)part * kList + (i - before);
    const uint32_t key = b.keys[at], index = b.indices[at];
    if (key >= from) list(logit_of(key), (int)index, s);
  }
  __syncthreads();
  return fits && s.listed <= kList && (from == 0 || s.listed >= wanted);
}

// The row's sums from its parts' bins.  Ends with a barrier.
template <int N>
__device__ __forceinline__ void take_bins(const SampleArgs &p, const Between &b, int r, const Weights &weights, bool counted, Shared<N> &s) {
  const long long first = (long long)r * p.parts * kBins;
  for (int i = threadIdx.x; i < kBins; i += N) {
    u64 weight = 0;
    uint32_t count = 0;
#pragma unroll
    for (int j = 0; j < kMostParts; ++j) {
      const long long at = first + (long long)min(j, p.parts - 1) * kBins + i;
      const u64 w = b.weights[at];
      weight += j < p.parts ? w : 0;
      if (counted) count += j < p.parts ? b.counts[at] : 0;
    }
    s.bins.inside[i] = weight;
    s.bins.counts[i] = count;
  }
  __syncthreads();
  sum_bins(weights, s);
}

// First: every part's largest, and where top_k is small a list of its first.
template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_first_kernel(const SampleArgs p) {
  __shared__ Shared<kThreads> s;
  const int part = blockIdx.x, r = blockIdx.y;
  const Between b(p.workspace, p.rows, p.parts);
  const RowReader<T> reader = part_of<T>(p, r, part);
  const Setting setting(p, r);
  const long long at = (long long)r * p.parts + part;
  Part mine = {-INFINITY, 0, 0};
  if (setting.few()) {
    // (its share and a line, which no part exceeds of first ones that stand side by side; half as many again, and some, of logits in any order)
    const int share = max((setting.top_k + p.parts - 1) / p.parts + RowReader<T>::kLineLogits, 3 * setting.top_k / (2 * p.parts) + 48);
    mine.from = list_first(reader, setting, (uint32_t)min(setting.top_k, share), mine.most, s);
    mine.count = s.listed;
    leave_list(b, at, s);
  } else {
    mine.most = largest_of(reader, s);
  }
  if (threadIdx.x == 0) b.parts[at] = mine;
}

// Second: every part's bins, where it has no such list.
template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_bins_kernel(const SampleArgs p) {
  __shared__ Shared<kThreads> s;
  const int part = blockIdx.x, r = blockIdx.y;
  const Between b(p.workspace, p.rows, p.parts);
  const Setting setting(p, r);
  const float most = largest_of_parts(p, b.parts + (long long)r * p.parts);
  if (setting.few() || most == -INFINITY) return;
  const bool counted = setting.top_k > 0;
  fill_bins(part_of<T>(p, r, part), Weights(setting, most), counted, s);
  const long long own = ((long long)r * p.parts + part) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    b.weights[own + i] = s.bins.inside[i];
    if (counted) b.counts[own + i] = s.bins.counts[i];
  }
}

// Third: from all parts' bins the ranges of logits that matter, and every part's list of its own in these.
template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_ends_kernel(const SampleArgs p) {
  __shared__ Shared<kThreads> s;
  const int part = blockIdx.x, r = blockIdx.y;
  const Between b(p.workspace, p.rows, p.parts);
  const Setting setting(p, r);
  const long long at = (long long)r * p.parts + part;
  const float most = largest_of_parts(p, b.parts + (long long)r * p.parts);
  if (setting.few() || most == -INFINITY) return;
  const Weights weights(setting, most);
  take_bins(p, b, r, weights, setting.top_k > 0, s);
  list_ranges(part_of<T>(p, r, part), ends_of(setting, weights, uniform_of(p, r), s), s);
  leave_list(b, at, s);
  if (threadIdx.x == 0) b.parts[at].count = s.listed;
}

// Fourth: the draw from the lists.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(const SampleArgs p) {
  __shared__ Shared<kThreads> s;
  const int r = blockIdx.x;
  const Between b(p.workspace, p.rows, p.parts);
  const Setting setting(p, r);
  const float most = largest_of_parts(p, b.parts + (long long)r * p.parts);
  if (most == -INFINITY) {
    result(p, r, -1, 0.f);
    return;
  }
  if (!setting.few()) take_bins(p, b, r, Weights(setting, most), setting.top_k > 0, s);
  const bool fits = take_lists(p, b, r, (uint32_t)setting.top_k, setting.few() ? least_of(setting, most) : -INFINITY, s);
  finish(p, setting, r, all_of<T>(p, r), most, !setting.few(), fits, s);
}

// Rows that are too few for the chip's 512 places for workgroups are taken in five parts or more, of 16384 logits or more: four launches, which cost some 9 us.  (bf16, us in
// parts and as a row each: one row of 131072 logits with no limit 31 and 51, top_k 28 and 35; 64 rows in eight parts 52 and 64, 39 and 46, top_p 67 and 78; 128 rows in four 65
// and 65, 46 and 46, all settings mixed 77 and 73; one row of 50000 in three 30 and 29, 23 and 20.)
int parts_of(int rows, int vocab) {
  const int parts = min(min(kMostParts, 512 / rows), vocab / 16384);
  return parts < 5 ? 1 : parts;
}

template <typename T>
hipError_t launch(const SampleArgs &a, hipStream_t stream) {
  if (a.parts == 1) {
    // Where a row has a CU of its own, 1024 threads, unless it is short, when their barriers cost more (us with 1024 and with 512 threads, no limit: 1 row of 2000 11.7 and 9.8, of
    // 20000 17.9 and 17.5, of 32000 20.7 and 21.8; 200 rows of 50000 36 and 39; 256 rows of 131072 79 and 93).  More rows have two workgroups a CU.
    if (a.rows <= 256 && a.vocab > 24576) hipLaunchKernelGGL((sample_tokens_kernel<T, kManyThreads>), dim3(a.rows), dim3(kManyThreads), 0, stream, a);
    else hipLaunchKernelGGL((sample_tokens_kernel<T, kThreads>), dim3(a.rows), dim3(kThreads), 0, stream, a);
  } else {
    const dim3 grid(a.parts, a.rows);
    // (settings that the host knows may say that no row has bins: 64 rows of 131072, top_k of 50 23.5 -> 20.3 us)
    const bool no_bins = (!a.top_k && a.top_k_all > 0 && a.top_k_all <= kMostTopK) || (!a.temperature && !(a.temperature_all > 0.f));
    hipLaunchKernelGGL((sample_first_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    if (!no_bins) {
      hipLaunchKernelGGL((sample_bins_kernel<T>), grid, dim3(kThreads), 0, stream, a);
      hipLaunchKernelGGL((sample_ends_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    }
    hipLaunchKernelGGL((sample_draw_kernel<T>), dim3(a.rows), dim3(kThreads), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(int rows, int vocab) {
  const int parts = parts_of(rows, vocab);
  return parts == 1 ? 0 : Between(nullptr, rows, parts).bytes(rows, parts);
}

hipError_t launch_sample_tokens(int type, SampleArgs args, hipStream_t stream) {
  args.parts = parts_of(args.rows, args.vocab);
  return type == 0 ? launch<Fp16>(args, stream) : type == 1 ? launch<Bf16>(args, stream) : launch<F32>(args, stream);
}

}  // namespace sspmm
