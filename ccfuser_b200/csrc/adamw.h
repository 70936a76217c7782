// Entry points of adamw.cu: one AdamW step over many tensors.
#pragma once

#define CCF_ADAMW_BLOCK 256   // weights that share the exponents of their 8-bit moments

#ifdef __cplusplus
extern "C" {
#endif

// One tensor: `rows` rows of n / rows weights each, contiguous. 8-bit moments are cut into blocks of CCF_ADAMW_BLOCK within a row (the last one of a row may be
// shorter), with two exponents a block.
typedef struct CcfAdamwTensor {
  void* p;
  const void* g;          // of p's type
  void* m;                // float, or uint8 codes
  void* v;
  unsigned char* e;       // [rows, blocks of a row, 2], or null: moments in fp32
  long long n, rows;
  long long number;       // of the tensor in its call: tensors round to 8 bits with hashes of their own
} CcfAdamwTensor;

typedef struct CcfAdamw {
  const CcfAdamwTensor* tensors;   // on the host
  int count, type;                 // type: elements.cuh's, of every tensor
  double lr, beta1, beta2, eps, weight_decay;
  unsigned long long seed;         // of the roundings to 8 bits
  long long step;                  // number of this step, from 1
  const void* scalars;             // of ccf_adamw_scalars, on the device, in the place of lr, weight_decay, seed and step; or null
} CcfAdamw;

#define CCF_ADAMW_SCALARS 32       // bytes, on a 16-byte boundary

int ccf_sizeof_adamw();
int ccf_sizeof_adamw_tensor();
// launches made, or a negative code (-2: arguments, nothing was launched). Either all tensors have 8-bit moments or none.
int ccf_adamw(const CcfAdamw* a, void* stream);
// What a step reads from the device: the counter there is raised by one and is the number of this step; lr comes from `device_lr` unless that is null
int ccf_adamw_scalars(const CcfAdamw* a, long long* counter, const float* device_lr, void* scalars, void* stream);
// the values of n = rows * (n / rows) codes: first moment, or the second; type: elements.cuh's, of the result
int ccf_state_values(const void* codes, const unsigned char* e, void* out, long long n, long long rows, int second, int type, void* stream);

#ifdef __cplusplus
}
#endif
