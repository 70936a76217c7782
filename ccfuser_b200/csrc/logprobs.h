// Entry points of the log-probability kernels (logprobs.cu), as torch_tokens.cpp and ops/logprobs.py call them.
#pragma once

#define CCF_LOGPROBS_MAX_TOP 32

// One call over logits [rows, width] (`ld` elements between rows) of which the first `vocab` columns count. `stats`: three floats per row
// (largest logit, sum, entropy) that the backward pass reads. The gradients may be null. The rows of `dx`
// begin as far from a 16-byte boundary as those of `x` do: `dx_ld` differs from `ld` by a multiple of 16 bytes where there are several.
struct CcfLogprobs {
  const void* x;
  const void* targets;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  long long* top_ids;
  float* stats;
  const float* d_logprobs;
  const float* d_entropy;
  const float* d_top;
  void* dx;
  int* status;
  long long rows;
  long long ld;
  long long dx_ld;
  long long ignore;
  int vocab;
  int width;
  int top_k;
  int type;           // 0 bf16, 1 fp16, 2 fp32
  int wide;           // targets are 64 bits wide
  float inv_t;        // 1 / temperature
};

#ifdef __cplusplus
extern "C" {
#endif
int ccf_sizeof_logprobs();
int ccf_logprobs_fwd(const CcfLogprobs* a, void* stream);
int ccf_logprobs_bwd(const CcfLogprobs* a, void* stream);
#ifdef __cplusplus
}
#endif
