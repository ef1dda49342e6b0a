// Launch interface of drawing tokens from logits.
#ifndef SSPMM_AMD_SAMPLE_KERNELS_H
#define SSPMM_AMD_SAMPLE_KERNELS_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sspmm {

// Row i of the logits is `vocab` elements from logits + i * stride on (aligned to an element).  Of temperature, top_k, top_p and min_p there is one value a row,
// or one for all where the pointer is null.
struct SampleArgs {
  const void *logits;
  long long stride;
  int rows, vocab;
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int32_t *tokens;
  float *probabilities;  // may be null
  unsigned char *workspace;  // sample_workspace_bytes, 8-byte aligned
  int parts;  // (the launch's own)
};
size_t sample_workspace_bytes(int rows, int vocab);
// type: 0 fp16, 1 bf16, 2 fp32
hipError_t launch_sample_tokens(int type, SampleArgs args, hipStream_t stream);

}  // namespace sspmm
#endif
