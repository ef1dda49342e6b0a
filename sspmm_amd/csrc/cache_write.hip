// Keys and values of new tokens into the paged cache: one scale for the tokens of a page and head,
//   scale = max |x| times 1 / 127 in 32 bits (int8) or the smallest power of two with max |x| / scale <= 448 (e4m3),  code = round(x / scale).
// A page that already holds tokens keeps its scale unless the new ones need a larger one; its codes are then brought to it.
#include "cache_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

// Both formats' rules; an infinity or a NaN among the values makes the scale NaN, and NaN stays.
template <int FORMAT>
__device__ __forceinline__ float scale_for(uint32_t most) {  // most: the bits of the largest magnitude
  if (most >= 0x7f800000u) return NAN;
  if (FORMAT == 0) return __uint_as_float(most) * (1.0f / 127.0f);
  if (most == 0) return 0.f;
  // 448 = 1.75 * 2^8.  (Below the normal numbers' range the exponent is out of the clamp's reach anyway.)
  const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}
__device__ __forceinline__ float larger_scale(float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }

// four quotients x / scale as codes; scale zero (a block of zeros) or NaN: zeros
template <int FORMAT>
__device__ __forceinline__ uint32_t codes(float x0, float x1, float x2, float x3, float scale) {
  if (!(scale > 0.f)) return 0u;
  if constexpr (FORMAT == 0) {
    const auto one = [&](float x) { return (uint32_t)(int)fminf(fmaxf(rintf(x / scale), -127.f), 127.f) & 0xffu; };
    return one(x0) | one(x1) << 8 | one(x2) << 16 | one(x3) << 24;
  } else {
    const float inv = 1.0f / scale;  // (a power of two)
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x0 * inv, x1 * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2 * inv, x3 * inv, r, true);
  }
}
template <int FORMAT>
__device__ __forceinline__ floatx4 values_of(uint32_t c) {
  if constexpr (FORMAT == 0) {
    return floatx4{(float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24)};
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return floatx4{lo[0], lo[1], hi[0], hi[1]};
  }
}
// codes at an old scale, at the new one
template <int FORMAT>
__device__ __forceinline__ uint32_t rescaled(uint32_t c, float before, float now) {
  const floatx4 x = values_of<FORMAT>(c);
  return codes<FORMAT>(x[0] * before, x[1] * before, x[2] * before, x[3] * before, now);
}

// Four words of four bytes, a token each, to a feature each.
__device__ __forceinline__ void turn(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
  // v_perm: selectors 0 .. 3 are bytes of the second operand, 4 .. 7 of the first
  const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x05010400u), ab2 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x05010400u), cd2 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  a = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
  b = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
  c = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
  d = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}

// Pages that the call's tokens lie in at most, in other words than that each has one.
__host__ __device__ __forceinline__ long long most_pages(const CacheWriteArgs &p) { return (long long)p.tokens / p.pool.page_size + 2ll * p.sequences; }

// A workgroup owns the keys (blockIdx.z = 0) or values of `heads_each` heads in one page that gets new tokens, one head after the other.  A thread takes four places
// of the page and eight features, side by side with threads of other features (keys) or other places (values, which lie transposed in the page), so that
// either's stores are whole lines and nothing passes through LDS.
//
// Bound by its bytes when there are many: 128 sequences of 1000 tokens, 8 heads of 128 features in bf16 191 us, 4.1 TB/s of reads and writes; 8084 tokens 12.6 us,
// 3.9 TB/s; and by the chain of loads that finds a page, its scale and its tokens when there are few: 48 sequences of one token, 8 heads of 64 features 4.9 us.
// A thread per item (64 to 256 a workgroup) instead of 256 always: 64 features, 4096 sequences of 64 tokens 504 -> 376 us, 8 of 1000 tokens 38 -> 31.
// kMost: of these a thread takes, the page's places / 4 times D / 8 over the threads.
template <typename T, int FORMAT, int D, int kThreads, int kMost>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(const CacheWriteArgs p, int heads_each) {
  constexpr int kPer = D / 8;  // threads for the features
  __shared__ uint32_t largest[2][kThreads / 64];  // of one head and of the next
  const int lane = threadIdx.x & 63, page_size = p.pool.page_size, quads = page_size / 4, items = quads * kPer;
  const int values = blockIdx.z;

  // ---- which page: the blockIdx.x-th of those that the sequences touch
  int row = -1, slot = 0, from = 0, upto = 0;
  long long token0 = 0;  // the token at the page's place `from`
  // (Numbers from `base` on are those of 64 sequences: as many as they have tokens, or a page for each page_size of these and two a sequence, as the host
  // counts.  Summing up the pages of the sequences before: 4096 of a token, 8 heads of 64 features 915 us instead of 175.)
  const bool by_tokens = p.tokens <= most_pages(p);
  const auto base = [&](int chunk) {
    const int tokens = max(0, min(p.offsets[64 * chunk], p.tokens));
    return by_tokens ? tokens : tokens / page_size + 128 * chunk;
  };
  const int chunk = last_not_above((p.sequences + 63) / 64, (int)blockIdx.x, base), left = (int)blockIdx.x - base(chunk);
  if (left >= 0) {
    const int b = 64 * chunk + lane;
    int lo = 0, hi = 0, start = 0;
    if (b < p.sequences) {
      lo = max(0, min(p.offsets[b], p.tokens));
      hi = max(lo, min(p.offsets[b + 1], p.tokens));
      start = p.starts[b];
      if (start < 0) hi = lo;
    }
    const long long end = (long long)start + (hi - lo);
    const int count = hi > lo ? (int)((end - 1) / page_size - start / page_size + 1) : 0;
    const int until = (int)wave_inclusive_sum((uint32_t)count);
    const unsigned long long found = __ballot(until > left);
    if (found != 0) {
      const int at = __builtin_ctzll(found);
      const int s = __builtin_amdgcn_readlane(start, at), n = __builtin_amdgcn_readlane(hi, at) - __builtin_amdgcn_readlane(lo, at);
      const int i = left - (__builtin_amdgcn_readlane(until, at) - __builtin_amdgcn_readlane(count, at));
      row = 64 * chunk + at;
      slot = s / page_size + i;
      const long long page0 = (long long)slot * page_size;
      from = (int)max(0ll, (long long)s - page0);
      upto = (int)min((long long)page_size, (long long)s + n - page0);
      token0 = __builtin_amdgcn_readlane(lo, at) + (page0 + from - s);
    }
  }
  if (row < 0 || slot >= p.pool.slots) return;
  const int page = p.pool.table[(long long)row * p.pool.slots + slot];
  if (page < 0 || page >= p.pool.pages) return;

#pragma unroll 1
  for (int head = blockIdx.y * heads_each; head < min(p.pool.kv_heads, ((int)blockIdx.y + 1) * heads_each); ++head) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (else all places are kept in registers from one head to the next: 187 instead of 104)
    float *const scale_at = p.pool.scales + ((long long)page * 2 + values) * p.pool.kv_heads + head;
    const float before = from > 0 ? *scale_at : 0.f;

    // ---- the new tokens, in registers
    const long long pitch = values ? p.v_row : p.k_row;
    const uint16_t *const src = (values ? p.v + (long long)head * p.v_head : p.k + (long long)head * p.k_head) + (token0 - from) * pitch;  // place 0
    const int bits = 31 - __builtin_clz(quads);
    unsigned char *const block = (values ? p.pool.values : p.pool.keys) + ((long long)page * p.pool.kv_heads + head) * ((long long)page_size * D);
    uintx4 x[kMost][4];
    uint32_t old[kMost][8] = {};  // (values) words with both new places and others, as they are
    uint32_t most = 0;
  #pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int at = i * kThreads + tid;
      const int quad = values ? at & (quads - 1) : at / kPer, octet = values ? at >> bits : at % kPer;
  #pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int place = 4 * quad + j;
        x[i][j] = uintx4{0, 0, 0, 0};
        if (at < items && place >= from && place < upto) x[i][j] = *reinterpret_cast<const uintx4 *>(src + place * pitch + 8 * octet);
      }
      if (values && at < items && 4 * quad < upto && 4 * quad + 4 > from && (4 * quad < from || 4 * quad + 4 > upto)) {
  #pragma unroll
        for (int f = 0; f < 8; ++f) old[i][f] = *reinterpret_cast<const uint32_t *>(block + (8 * octet + f) * page_size + 4 * quad);
      }
    }
  #pragma unroll
    for (int i = 0; i < kMost; ++i)
  #pragma unroll
      for (int j = 0; j < 4; ++j)
  #pragma unroll
        for (int w = 0; w < 4; ++w) {
          // (bits of magnitudes order as the magnitudes do, infinities and NaN above all)
          most = max(most, max(__float_as_uint(T::lower(x[i][j][w])) & 0x7fffffffu, __float_as_uint(T::upper(x[i][j][w])) & 0x7fffffffu));
        }
    most = from_last_lane(wave_inclusive_max(most));
    if (lane == 0) largest[head & 1][tid >> 6] = most;
    __syncthreads();  // (behind it every wave has read the scale, too, that is about to be replaced)
  #pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) most = max(most, largest[head & 1][i]);

    const float needed = scale_for<FORMAT>(most);
    const float scale = from > 0 ? larger_scale(before, needed) : needed;
    const bool grown = from > 0 && scale > before;  // (a NaN scale: what is there does not matter any more)
    if (tid == 0 && (from == 0 || scale != before)) *scale_at = scale;

  #pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int at = i * kThreads + tid;
      const int quad = values ? at & (quads - 1) : at / kPer, octet = values ? at >> bits : at % kPer, place = 4 * quad;
      if (at >= items || place >= upto || (place + 4 <= from && !grown)) continue;
      uint32_t c[4][2];
  #pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j][0] = c[j][1] = 0;
        if (place + j < from || place + j >= upto) continue;  // (a division is a dozen instructions: a single token does one of four)
  #pragma unroll
        for (int w = 0; w < 2; ++w)
          c[j][w] = codes<FORMAT>(T::lower(x[i][j][2 * w]), T::upper(x[i][j][2 * w]), T::lower(x[i][j][2 * w + 1]), T::upper(x[i][j][2 * w + 1]), scale);
      }
      if (!values) {
        uintx2 *to[4];
        uintx2 kept[4];
  #pragma unroll
        for (int j = 0; j < 4; ++j) {
          to[j] = reinterpret_cast<uintx2 *>(block + (place + j) * D + 8 * octet);
          kept[j] = grown && place + j < from ? *to[j] : uintx2{0, 0};
        }
  #pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (place + j >= from) {
            if (place + j < upto) *to[j] = uintx2{c[j][0], c[j][1]};
          } else if (grown) {
            *to[j] = uintx2{rescaled<FORMAT>(kept[j][0], before, scale), rescaled<FORMAT>(kept[j][1], before, scale)};
          }
        }
      } else {
  #pragma unroll
        for (int w = 0; w < 2; ++w) turn(c[0][w], c[1][w], c[2][w], c[3][w]);  // c[j][w]: feature 4 w + j, a byte a place
        if (place + 4 <= from) {  // (all of it kept, at a scale that has grown)
  #pragma unroll
          for (int f = 0; f < 8; ++f) old[i][f] = *reinterpret_cast<const uint32_t *>(block + (8 * octet + f) * page_size + place);
        }
        uint32_t keep = 0, stale = 0;  // the bytes in front of the new places and behind them
  #pragma unroll
        for (int j = 0; j < 4; ++j) {
          keep |= place + j < from ? 0xffu << (8 * j) : 0u;
          stale |= place + j >= upto ? 0xffu << (8 * j) : 0u;
        }
  #pragma unroll
        for (int f = 0; f < 8; ++f) {
          const uint32_t moved = grown && keep != 0 ? rescaled<FORMAT>(old[i][f], before, scale) : old[i][f];
          *reinterpret_cast<uint32_t *>(block + (8 * octet + f) * page_size + place) = (moved & keep) | (old[i][f] & stale) | (c[f % 4][f / 4] & ~(keep | stale));
        }
      }
    }
  }
}

template <typename T, int FORMAT, int D, int kThreads, int kMost = 1>
hipError_t launch(const CacheWriteArgs &a, hipStream_t stream) {
  const long long most = min(most_pages(a), (long long)a.tokens);
  if (most >= (1ll << 32) / kThreads) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads along x)
  // A workgroup takes a head, or several one after the other where there are more of them than the chip has places for, some 2000 to 8000: each page has
  // to be found, and that is a chain of loads of its own.  4096 sequences of a token, 8 heads of 64 features 102 us with a head each, 81 so; of
  // 64 tokens 447 and 376; 128 of 1000 tokens, 128 features 207 and 191; 300 of 100 tokens 65 and 68.
  const int kv = a.pool.kv_heads, heads_each = (int)max(1ll, min(most * kv * 2 / 4096, (long long)kv));
  const dim3 grid((unsigned)most, (kv + heads_each - 1) / heads_each, 2);
  hipLaunchKernelGGL((cache_write_kernel<T, FORMAT, D, kThreads, kMost>), grid, dim3(kThreads), 0, stream, a, heads_each);
  return hipGetLastError();
}

template <typename T, int FORMAT>
hipError_t launch(const CacheWriteArgs &a, hipStream_t stream) {
  const int page = a.pool.page_size;
  switch (a.pool.d) {
    case 128: return page == 128 ? launch<T, FORMAT, 128, 256, 2>(a, stream) : page == 64 ? launch<T, FORMAT, 128, 256>(a, stream) : launch<T, FORMAT, 128, 128>(a, stream);
    case 64: return page == 128 ? launch<T, FORMAT, 64, 256>(a, stream) : page == 64 ? launch<T, FORMAT, 64, 128>(a, stream) : launch<T, FORMAT, 64, 64>(a, stream);
    default: return page == 128 ? launch<T, FORMAT, 32, 128>(a, stream) : launch<T, FORMAT, 32, 64>(a, stream);
  }
}

}  // namespace

hipError_t launch_cache_write(int type, int format, const CacheWriteArgs &a, hipStream_t stream) {
  if (type == 0) return format == 0 ? launch<Fp16, 0>(a, stream) : launch<Fp16, 1>(a, stream);
  return format == 0 ? launch<Bf16, 0>(a, stream) : launch<Bf16, 1>(a, stream);
}

}  // namespace sspmm
