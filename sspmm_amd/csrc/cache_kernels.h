// Launch interface of the paged cache in 8 bits: writing, attention, pages.
#ifndef SSPMM_AMD_CACHE_KERNELS_H
#define SSPMM_AMD_CACHE_KERNELS_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sspmm {

// keys [pages, kv_heads, page_size, d] and values [pages, kv_heads, d, page_size] in 8 bits, scales [pages, 2, kv_heads] (keys, values),
// table [rows, slots]: the page that holds positions slot * page_size .. of a row.  All of it dense, keys and values 16-byte aligned.
struct CachePool {
  unsigned char *keys, *values;
  float *scales;
  const int32_t *table;
  int pages, kv_heads, page_size, d, slots;
};

// Rows offsets[b] .. offsets[b + 1] - 1 of k and v ([tokens, kv_heads, d], strides in elements, multiples of 8, 16-byte aligned) to positions
// starts[b] on of table row b.  type: 0 fp16, 1 bf16; format: 0 int8, 1 e4m3.
struct CacheWriteArgs {
  CachePool pool;
  const uint16_t *k, *v;
  long long k_row, k_head, v_row, v_head;
  const int32_t *offsets, *starts;
  int sequences, tokens;
};
hipError_t launch_cache_write(int type, int format, const CacheWriteArgs &args, hipStream_t stream);

// out[b, i, h] = attention of q[b, i, h] over positions 0 .. lengths[b] - queries + i of table row b.
struct CacheAttentionArgs {
  CachePool pool;
  const uint16_t *q;
  uint16_t *out;
  long long q_seq, q_row, q_head, out_seq, out_row, out_head;
  const int32_t *lengths;
  int sequences, queries, heads;
  float scale_log2e;
  float *partial;  // cache_attention_workspace floats
  int splits;      // (the launch's own)
};
// longest: positions that a row of the table has room for
size_t cache_attention_workspace(int sequences, int queries, int heads, int kv_heads, int d, long long longest);  // floats
hipError_t launch_cache_attention(int type, int format, CacheAttentionArgs args, hipStream_t stream);

}  // namespace sspmm
#endif
