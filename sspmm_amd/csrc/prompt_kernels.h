// Launch interface of the attention over whole prompts.
#ifndef SSPMM_AMD_PROMPT_KERNELS_H
#define SSPMM_AMD_PROMPT_KERNELS_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sspmm {

// Sequence b is rows offsets[b] .. offsets[b + 1] - 1 of q, out ([tokens, heads, d]) and k, v ([tokens, kv_heads, d]).  Row i, head h of x
// is at x + i * x_row + h * x_head elements; 16-byte aligned, strides multiples of 8 elements, rows at least d apart.
struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int32_t *offsets;
  long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  int sequences, tokens, heads, kv_heads;
  float scale_log2e;
};
// d: 32, 64 or 128; type: 0 fp16, 1 bf16
hipError_t launch_prompt_attention(int type, int d, bool causal, const PromptArgs &args, hipStream_t stream);

}  // namespace sspmm
#endif
