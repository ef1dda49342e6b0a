// Keys and values of new tokens into the paged cache: one scale for the tokens of a page and head,
//   scale = max |x| / 127 (int8) or the smallest power of two with max |x| / scale <= 448 (e4m3),  code = round(x / scale).
// A page that already holds tokens keeps its scale unless the new ones need a larger one; its codes are then brought to it.
#include "cache_kernels.h"

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

namespace {

constexpr int kThreads = 256;

// Both formats' rules; an infinity or a NaN among the values makes the scale NaN, and NaN stays.
template <int FORMAT>
__device__ __forceinline__ float scale_for(uint32_t most) {  // most: the bits of the largest magnitude
  if (most >= 0x7f800000u) return NAN;
  if (FORMAT == 0) return __uint_as_float(most) / 127.0f;
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

// A workgroup owns one block: the keys (blockIdx.z = 0) or values of one head in one page that gets new tokens.  Values lie transposed in the
// page, so their codes pass through LDS.
template <typename T, int FORMAT, int D>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(const CacheWriteArgs p) {
  constexpr int kPer = D / 8;  // pieces of eight elements of a token
  constexpr int kMost = 128 * kPer / kThreads;  // of a thread, in the largest page
  __shared__ __align__(16) unsigned char turned[D * 128];
  __shared__ uint32_t largest[kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, page_size = p.pool.page_size;
  const int head = blockIdx.y, values = blockIdx.z;

  // ---- which page: the blockIdx.x-th of those that the sequences touch
  int row = -1, slot = 0, from = 0, upto = 0;
  long long token0 = 0;  // the token at the page's place `from`
  for (int b0 = 0, base = 0; b0 < p.sequences; b0 += 64) {
    const int b = b0 + lane;
    int lo = 0, hi = 0, start = 0;
    if (b < p.sequences) {
      lo = max(0, min(p.offsets[b], p.tokens));
      hi = max(lo, min(p.offsets[b + 1], p.tokens));
      start = p.starts[b];
      if (start < 0) hi = lo;
    }
    const long long end = (long long)start + (hi - lo);
    const int count = hi > lo ? (int)((end - 1) / page_size - start / page_size + 1) : 0;
    const int until = base + (int)wave_inclusive_sum((uint32_t)count);
    const unsigned long long found = __ballot(until > (int)blockIdx.x);
    if (found != 0) {
      const int at = __builtin_ctzll(found);
      const int s = __builtin_amdgcn_readlane(start, at), n = __builtin_amdgcn_readlane(hi, at) - __builtin_amdgcn_readlane(lo, at);
      const int i = (int)blockIdx.x - (__builtin_amdgcn_readlane(until, at) - __builtin_amdgcn_readlane(count, at));
      row = b0 + at;
      slot = s / page_size + i;
      const long long page0 = (long long)slot * page_size;
      from = (int)max(0ll, (long long)s - page0);
      upto = (int)min((long long)page_size, (long long)s + n - page0);
      token0 = __builtin_amdgcn_readlane(lo, at) + (page0 + from - s);
      break;
    }
    base = __builtin_amdgcn_readlane(until, 63);
  }
  if (row < 0 || slot >= p.pool.slots) return;
  const int page = p.pool.table[(long long)row * p.pool.slots + slot];
  if (page < 0 || page >= p.pool.pages) return;

  // ---- the new tokens, in registers
  const uint16_t *const src = values ? p.v + token0 * p.v_row + (long long)head * p.v_head : p.k + token0 * p.k_row + (long long)head * p.k_head;
  const long long pitch = values ? p.v_row : p.k_row;
  const int pieces = (upto - from) * kPer;
  uintx4 x[kMost];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int at = i * kThreads + tid;
    x[i] = uintx4{0, 0, 0, 0};
    if (at < pieces) x[i] = *reinterpret_cast<const uintx4 *>(src + (at / kPer) * pitch + (at % kPer) * 8);
  }
#pragma unroll
  for (int i = 0; i < kMost; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (bits of magnitudes order as the magnitudes do, infinities and NaN above all)
      most = max(most, max(__float_as_uint(T::lower(x[i][j])) & 0x7fffffffu, __float_as_uint(T::upper(x[i][j])) & 0x7fffffffu));
    }
  most = from_last_lane(wave_inclusive_max(most));
  if (lane == 0) largest[tid >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) most = max(most, largest[i]);

  float *const scale_at = p.pool.scales + ((long long)page * 2 + values) * p.pool.kv_heads + head;
  const float needed = scale_for<FORMAT>(most), before = from > 0 ? *scale_at : 0.f;
  const float scale = from > 0 ? larger_scale(before, needed) : needed;
  const bool grown = from > 0 && scale > before;  // (a NaN scale: what is there does not matter any more)
  __syncthreads();  // (every wave has read the scale that is about to be replaced)
  if (tid == 0 && (from == 0 || scale != before)) *scale_at = scale;

  unsigned char *const block = (values ? p.pool.values : p.pool.keys) + ((long long)page * p.pool.kv_heads + head) * ((long long)page_size * D);
  if (!values) {
    if (grown)
      for (int at = tid; at < from * kPer; at += kThreads) {
        uintx2 *const c = reinterpret_cast<uintx2 *>(block + at * 8);
        const uintx2 old = *c;
        *c = uintx2{rescaled<FORMAT>(old[0], before, scale), rescaled<FORMAT>(old[1], before, scale)};
      }
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int at = i * kThreads + tid;
      if (at < pieces)
        *reinterpret_cast<uintx2 *>(block + (from * kPer + at) * 8) =
            uintx2{codes<FORMAT>(T::lower(x[i][0]), T::upper(x[i][0]), T::lower(x[i][1]), T::upper(x[i][1]), scale),
                   codes<FORMAT>(T::lower(x[i][2]), T::upper(x[i][2]), T::lower(x[i][3]), T::upper(x[i][3]), scale)};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int at = i * kThreads + tid;
    if (at < pieces) {
      const uint32_t a = codes<FORMAT>(T::lower(x[i][0]), T::upper(x[i][0]), T::lower(x[i][1]), T::upper(x[i][1]), scale);
      const uint32_t b = codes<FORMAT>(T::lower(x[i][2]), T::upper(x[i][2]), T::lower(x[i][3]), T::upper(x[i][3]), scale);
      unsigned char *const to = turned + (at % kPer) * 8 * page_size + from + at / kPer;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        to[j * page_size] = (unsigned char)(a >> (8 * j));
        to[(4 + j) * page_size] = (unsigned char)(b >> (8 * j));
      }
    }
  }
  __syncthreads();
  const int words = page_size / 4;
  for (int at = tid; at < D * words; at += kThreads) {
    const int place = (at % words) * 4;
    if (place >= upto || (place + 4 <= from && !grown)) continue;
    uint32_t w = *reinterpret_cast<const uint32_t *>(turned + at * 4);
    uint32_t *const to = reinterpret_cast<uint32_t *>(block + at * 4);
    if (place < from || place + 4 > upto) {
      uint32_t old = *to;
      const uint32_t moved = grown ? rescaled<FORMAT>(old, before, scale) : old;
      uint32_t r = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t m = 0xffu << (8 * j);
        r |= (place + j < from ? moved : place + j < upto ? w : old) & m;
      }
      w = r;
    }
    *to = w;
  }
}

template <typename T, int FORMAT>
hipError_t launch(const CacheWriteArgs &a, hipStream_t stream) {
  const long long most = (long long)a.tokens / a.pool.page_size + 2ll * a.sequences;
  const dim3 grid((unsigned)min(most, (long long)a.tokens), a.pool.kv_heads, 2);
  switch (a.pool.d) {
    case 128: hipLaunchKernelGGL((cache_write_kernel<T, FORMAT, 128>), grid, dim3(kThreads), 0, stream, a); break;
    case 64: hipLaunchKernelGGL((cache_write_kernel<T, FORMAT, 64>), grid, dim3(kThreads), 0, stream, a); break;
    default: hipLaunchKernelGGL((cache_write_kernel<T, FORMAT, 32>), grid, dim3(kThreads), 0, stream, a); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_write(int type, int format, const CacheWriteArgs &a, hipStream_t stream) {
  if (type == 0) return format == 0 ? launch<Fp16, 0>(a, stream) : launch<Fp16, 1>(a, stream);
  return format == 0 ? launch<Bf16, 0>(a, stream) : launch<Bf16, 1>(a, stream);
}

}  // namespace sspmm
