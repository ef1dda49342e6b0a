// Launch interface of the attention over the paged cache for rows that share leading pages.
#ifndef SSPMM_AMD_PREFIX_KERNELS_H
#define SSPMM_AMD_PREFIX_KERNELS_H

#include "cache_kernels.h"

namespace sspmm {

constexpr int kMostPlanRows = 1024;

// What the sizes alone say of a plan and of the workspace of the attention that follows it.
struct PrefixShape {
  long long tiles, jobs;  // no plan has more
  long long state_rows;   // of the states that the jobs leave, for each head of the cache
  int target;             // jobs, about, of many units
  int row_queries;        // queries x heads of a group, of a row
};
PrefixShape prefix_shape(int rows, int queries, int heads, int kv_heads);
size_t prefix_plan_ints(const PrefixShape &shape, int rows);
size_t prefix_attention_floats(const PrefixShape &shape, int kv_heads, int d);

// table [rows, slots], lengths [rows]; plan: prefix_plan_ints, 16-byte aligned
hipError_t launch_plan_prefixes(const PrefixShape &shape, const int32_t *table, int rows, int slots, const int32_t *lengths, int page_size, int queries, int32_t *plan,
                                hipStream_t stream);

// out[b, i, h] = attention of q[b, i, h] over positions 0 .. length - queries + i of table row b, length as the plan has it.
struct PrefixAttentionArgs {
  CachePool pool;
  const uint16_t *q;
  uint16_t *out;
  long long q_seq, q_row, q_head, out_seq, out_row, out_head;
  const int32_t *plan;
  int rows, queries, heads;
  float scale_log2e;
  float *partial;  // prefix_attention_floats
  PrefixShape shape;
};
hipError_t launch_prefix_attention(int type, int format, const PrefixAttentionArgs &args, hipStream_t stream);

}  // namespace sspmm
#endif
