// Dropout, alone or with the addition of the residual stream: y = residual + (kept ? x / (1 - p) : 0). Whether element i is kept follows from
// 16 bits of a counter-based generator, Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", 2011): key = the seed, counter = (i / 8, call, step). No mask is stored: the backward pass draws the same bits again. The
// reference's Transformer-XL drops activations at these places with torch's dropout
// (mix_moe/mix_moe/examples/transformer-xl/mem_transformer_mix_moe.py).
//
// Bound by reading x (and the residual) and writing y once. 16 bits an element, eight elements a block of the generator: ten integer operations an
// element next to 4 or 6 bytes. p is rounded to a multiple of 2^-16, and 1 / (1 - p) is that of the rounded p, so that the mean stays.
#include "dropout.h"
#include "elements.cuh"

namespace ccf {

constexpr int kDropThreads = 256;

struct Philox {
  uint32_t k0, k1, call, step;
  // bits of the eight elements of a group, 16 each: element 2 i + h in half h of word i
  __device__ __forceinline__ uint4 operator()(uint64_t group) const {
    uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = call, c3 = step, a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const uint64_t p = static_cast<uint64_t>(0xD2511F53u) * c0, q = static_cast<uint64_t>(0xCD9E8D57u) * c2;
      c0 = static_cast<uint32_t>(q >> 32) ^ c1 ^ a;
      c1 = static_cast<uint32_t>(q);
      c2 = static_cast<uint32_t>(p >> 32) ^ c3 ^ b;
      c3 = static_cast<uint32_t>(p);
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

template <int kType>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const void* __restrict__ x, const void* __restrict__ residual, void* __restrict__ y,
                                                               const long long* __restrict__ state, long long* __restrict__ state_copy,
                                                               uint32_t call, uint32_t drop, float scale, long long n) {
  constexpr int kE = kElemsPer16<kType>, kQ = 8 / kE;   // 16-byte pieces of a group
  const unsigned long long seed = state[0], step = state[1];
  if (state_copy != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    state_copy[0] = seed;
    state_copy[1] = step;
  }
  const Philox bits{static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), call, static_cast<uint32_t>(step)};
  const long long groups = (n + 7) / 8;
  for (long long g = static_cast<long long>(blockIdx.x) * kDropThreads + threadIdx.x; g < groups; g += static_cast<long long>(gridDim.x) * kDropThreads) {
    if (g * 8 + 8 <= n) {
      uint4 xv[kQ], rv[kQ];
#pragma unroll
      for (int i = 0; i < kQ; ++i) xv[i] = load16_once(reinterpret_cast<const uint4*>(x) + g * kQ + i);
      if (residual != nullptr) {
#pragma unroll
        for (int i = 0; i < kQ; ++i) rv[i] = load16_once(reinterpret_cast<const uint4*>(residual) + g * kQ + i);
      }
      const uint4 b = bits(g);
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        float f[kE], r[kE] = {};
        unpack16<kType>(xv[i], f);
        if (residual != nullptr) unpack16<kType>(rv[i], r);
#pragma unroll
        for (int j = 0; j < kE; ++j) {
          const int e = i * kE + j;
          const uint32_t v = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
          f[j] = v >= drop ? fmaf(f[j], scale, r[j]) : r[j];
        }
        reinterpret_cast<uint4*>(y)[g * kQ + i] = pack16<kType>(f);
      }
    } else {
      const uint4 b = bits(g);
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const long long at = g * 8 + e;
        if (at >= n) continue;
        const uint32_t v = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
        const float r = residual != nullptr ? load_elem<kType>(residual, at) : 0.f;
        store_elem<kType>(y, at, v >= drop ? fmaf(load_elem<kType>(x, at), scale, r) : r);
      }
    }
  }
}

template <int kType>
static int launch_dropout(const void* x, const void* residual, void* y, const long long* state, long long* state_copy, uint32_t call,
                          uint32_t drop, long long n, cudaStream_t st) {
  const long long need = ((n + 7) / 8 + kDropThreads - 1) / kDropThreads, wave = 8ll * sm_count();
  const float scale = drop < 65536u ? 65536.f / static_cast<float>(65536u - drop) : 0.f;
  dropout_kernel<kType><<<static_cast<unsigned>(need < wave ? need : wave), kDropThreads, 0, st>>>(x, residual, y, state, state_copy, call, drop,
                                                                                                  scale, n);
  return launch_result();
}

}  // namespace ccf

extern "C" {

// y[i] = residual[i] + (r_i >= drop ? x[i] * 65536 / (65536 - drop) : 0) with the 16 bits r_i of (seed, i, call, step); state: {seed, step} on the
// device, copied to `state_copy` where that is given. residual may be null. The backward pass is the same call on dy without a residual.
// x, residual and y on 16-byte boundaries, n elements.
int ccf_dropout(const void* x, const void* residual, void* y, const long long* state, long long* state_copy, unsigned int call,
                unsigned int drop, long long n, int type, void* stream) {
  using namespace ccf;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
  if (x == nullptr || y == nullptr || state == nullptr || n < 1 || drop > 65536u || type < 0 || type > 2 || (at & 15) != 0) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (type == kBf16) return launch_dropout<kBf16>(x, residual, y, state, state_copy, call, drop, n, st);
  if (type == kFp16) return launch_dropout<kFp16>(x, residual, y, state, state_copy, call, drop, n, st);
  return launch_dropout<kFp32>(x, residual, y, state, state_copy, call, drop, n, st);
}

}  // extern "C"
