// Element types of the kernels between token ids and logits (embedding.cu, logprobs.cu, dropout.cu): 16 bytes of bf16, fp16 or fp32
// to floats and back, and what their launchers share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dispatch.cuh"   // pack2 / unpack2, report_status
#include "sm100.cuh"

namespace ccf {

enum ElemType { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

template <int kType>
constexpr int kElemBytes = kType == kFp32 ? 4 : 2;
template <int kType>
constexpr int kElemsPer16 = 16 / kElemBytes<kType>;

template <int kType>
__device__ __forceinline__ void unpack16(const uint4& q, float (&f)[kElemsPer16<kType>]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kType == kFp32) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (kType == kBf16) {   // a bf16 is the upper half of a float
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = unpack2(w[i], kType == kFp16);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

template <int kType>
__device__ __forceinline__ uint4 pack16(const float (&f)[kElemsPer16<kType>]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kType == kFp32) w[i] = __float_as_uint(f[i]);
    else w[i] = pack2(f[2 * i], f[2 * i + 1], kType == kFp16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// one element by its index
template <int kType>
__device__ __forceinline__ float load_elem(const void* p, long long i) {
  if constexpr (kType == kFp32) return __ldg(reinterpret_cast<const float*>(p) + i);
  else if constexpr (kType == kFp16) return __half2float(__ldg(reinterpret_cast<const __half*>(p) + i));
  else return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
}
template <int kType>
__device__ __forceinline__ void store_elem(void* p, long long i, float v) {
  if constexpr (kType == kFp32) reinterpret_cast<float*>(p)[i] = v;
  else if constexpr (kType == kFp16) reinterpret_cast<__half*>(p)[i] = __float2half(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
}

// 16 bytes that this kernel reads once: not kept in L1
__device__ __forceinline__ uint4 load16_once(const void* p) {
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
  return q;
}

// an index of a 32- or 64-bit array
__device__ __forceinline__ long long load_index(const void* p, long long i, int wide) {
  return wide ? __ldg(reinterpret_cast<const long long*>(p) + i) : static_cast<long long>(__ldg(reinterpret_cast<const int*>(p) + i));
}

// An id out of its table, at this token (or row of logits). The status word has 23 bits for it: the last number stands for all from there on.
__device__ __forceinline__ void report_index(int* status, uint32_t token) {
  report_status(status, CCF_ERR_INDEX, static_cast<int>(min(token, 0x7fffffu)));
}

inline int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

inline int launch_result() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -static_cast<int>(e);
}

}  // namespace ccf
