// Launch interface of the attention over whole prompts, and of that of packed queries over packed states.
#ifndef SSPMM_AMD_PROMPT_KERNELS_H
#define SSPMM_AMD_PROMPT_KERNELS_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sspmm {

// Sequence b is rows offsets[b] .. offsets[b + 1] - 1 of q, out ([tokens, heads, d]) and k, v ([tokens, kv_heads, d]), or rows
// key_offsets[b] .. key_offsets[b + 1] - 1 of these ([key_tokens, kv_heads, d]).  Row i, head h of x
// is at x + i * x_row + h * x_head elements; 16-byte aligned, strides multiples of 8 elements, rows at least d apart.
struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int32_t *offsets;
  const int32_t *key_offsets;  // null: the queries' sequences are those of the keys, and key_tokens is tokens
  long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  int sequences, tokens, key_tokens, heads, kv_heads;
  float scale_log2e;
};
// d: 32, 64 or 128; type: 0 fp16, 1 bf16; causal only without key_offsets
hipError_t launch_prompt_attention(int type, int d, bool causal, const PromptArgs &args, hipStream_t stream);

// The attention with key_offsets: by the above, or by workgroups that share out a sequence's keys where it has few queries.
size_t cross_attention_workspace(int sequences, int tokens, int key_tokens, int heads, int kv_heads, int d);  // floats
hipError_t launch_cross_attention(int type, int d, const PromptArgs &args, float *workspace, hipStream_t stream);

}  // namespace sspmm
#endif
