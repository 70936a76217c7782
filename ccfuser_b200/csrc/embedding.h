// Entry points of the embedding kernels (embedding.cu), as torch_tokens.cpp and ops/embedding.py call them.
#pragma once

#define CCF_EMBED_TABLES 3
#define CCF_EMBED_MAX_D (1 << 24)
#define CCF_EMBED_MAX_TOKENS (1 << 26)   // merging sorted chunks takes time with the square of their number: seconds there

// One table of a sum of lookups. `ids`: an index per token (32 or 64 bits), or null for the token's place in its sequence
// (token % seq). `grad`, `scratch`, `skip` belong to the backward pass: the dense gradient [rows, d], its scratch memory and the row that
// gets none (-1: every row gets one).
struct CcfEmbedTable {
  const void* weight;
  const void* ids;
  void* grad;
  void* scratch;
  long long rows;
  long long ld;       // elements between rows of `weight`; rows of `grad` are d apart
  long long skip;
  float scale;
  int wide;           // ids are 64 bits wide
};

struct CcfEmbed {
  CcfEmbedTable table[CCF_EMBED_TABLES];
  long long tokens;
  long long seq;
  int tables;
  int d;
  int type;           // 0 bf16, 1 fp16, 2 fp32
  int pad0;
};

#ifdef __cplusplus
extern "C" {
#endif
int ccf_sizeof_embed();
int ccf_embedding_fwd(const CcfEmbed* e, void* y, int* status, void* stream);
long long ccf_embedding_scratch(long long tokens, long long seq, long long rows, int d, int sorted);
int ccf_embedding_bwd(const CcfEmbed* e, const void* dy, int* status, void* stream);
#ifdef __cplusplus
}
#endif
