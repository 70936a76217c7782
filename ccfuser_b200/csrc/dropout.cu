// Dropout, alone or with the addition of the residual stream: y = residual + (kept ? x / (1 - p) : 0). Whether element i is kept follows from
// 16 bits of a counter-based generator, Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", 2011): key = the seed, counter = (i / 8, call, step). No mask is stored: the backward pass draws the same bits again. The
// reference's Transformer-XL drops activations at these places with torch's dropout
// (mix_moe/mix_moe/examples/transformer-xl/mem_transformer_mix_moe.py).
//
// Bound by reading x (and the residual) and writing y once. 16 bits an element, eight elements a block of the generator: ten integer operations an
// element next to 4 or 6 bytes. p is rounded to a multiple of 2^-16, and 1 / (1 - p) is that of the rounded p, so that the mean stays. One rounding, of
// the sum in fp32. 16384 x 4096 bf16 with the residual 66 us (6.1 TB/s), without 51 (5.3 TB/s; with one round of the generator instead of ten 48).
#include "dropout.h"
#include "elements.cuh"

namespace ccf {

// Blocks per SM: one wave, each thread walks the groups a grid apart. Sum of both passes at that size with 3, 4, 5 and 6 blocks: 124, 118, 122 and 121 us.
constexpr int kDropThreads = 256, kDropBlocks = 4;
template <int kType, bool kResidual>
constexpr int kDropGroups = kType != kFp32 && !kResidual ? 4 : 2;   // groups that a thread has in flight: 64 bytes

struct Philox {
  uint32_t a[10], b[10];   // the keys of the rounds
  uint32_t call, step;
  __device__ __forceinline__ Philox(uint64_t seed, uint32_t call_, uint32_t step_) : call(call_), step(step_) {
    a[0] = static_cast<uint32_t>(seed);
    b[0] = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 1; r < 10; ++r) {
      a[r] = a[r - 1] + 0x9E3779B9u;
      b[r] = b[r - 1] + 0xBB67AE85u;
    }
  }
  // bits of the eight elements of a group, 16 each: element 2 i + h in half h of word i
  __device__ __forceinline__ void operator()(uint64_t group, uint32_t (&w)[4]) const {
    uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = call, c3 = step;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const uint64_t p = static_cast<uint64_t>(0xD2511F53u) * c0, q = static_cast<uint64_t>(0xCD9E8D57u) * c2;
      c0 = static_cast<uint32_t>(q >> 32) ^ c1 ^ a[r];
      c1 = static_cast<uint32_t>(q);
      c2 = static_cast<uint32_t>(p >> 32) ^ c3 ^ b[r];
      c3 = static_cast<uint32_t>(p);
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
  }
};

// Element e of a group is kept: its 16 bits are at least `drop`. `high` = drop << 16: below the compared half nothing counts.
__device__ __forceinline__ bool kept(const uint32_t (&w)[4], int e, uint32_t high) { return (e & 1 ? w[e / 2] : w[e / 2] << 16) >= high; }

// scale 0: nothing is kept, which `high` cannot say.
template <int kType, bool kResidual>
__global__ void __launch_bounds__(kDropThreads, kDropBlocks)
    dropout_kernel(const void* __restrict__ x, const void* __restrict__ residual, void* __restrict__ y, const long long* __restrict__ state,
                   long long* __restrict__ state_copy, uint32_t call, uint32_t high, float scale, long long n) {
  constexpr int kE = kElemsPer16<kType>, kQ = 8 / kE;   // 16-byte pieces of a group
  constexpr int kGroups = kDropGroups<kType, kResidual>;
  const unsigned long long seed = state[0], step = state[1];
  if (state_copy != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    state_copy[0] = seed;
    state_copy[1] = step;
  }
  const Philox bits(seed, call, static_cast<uint32_t>(step));
  const bool none = scale == 0.f;
  const long long whole = n / 8, stride = static_cast<long long>(gridDim.x) * kDropThreads;
  const long long first = static_cast<long long>(blockIdx.x) * kDropThreads + threadIdx.x;
  for (long long g0 = first; g0 < whole; g0 += kGroups * stride) {
    uint4 xv[kGroups][kQ], rv[kGroups][kQ];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const long long g = g0 + k * stride;
      if (k > 0 && g >= whole) break;
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        xv[k][i] = load16_once(reinterpret_cast<const uint4*>(x) + g * kQ + i);
        if constexpr (kResidual) rv[k][i] = load16_once(reinterpret_cast<const uint4*>(residual) + g * kQ + i);
      }
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const long long g = g0 + k * stride;
      if (k > 0 && g >= whole) break;
      uint32_t w[4];
      bits(g, w);
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        float f[kE], r[kE] = {};
        unpack16<kType>(xv[k][i], f);
        if constexpr (kResidual) unpack16<kType>(rv[k][i], r);
#pragma unroll
        for (int j = 0; j < kE; ++j)
          if (kept(w, i * kE + j, high) && !none) r[j] = fmaf(f[j], scale, r[j]);
        reinterpret_cast<uint4*>(y)[g * kQ + i] = pack16<kType>(r);
      }
    }
  }
  if (first == 0 && n % 8 != 0) {   // the last group
    uint32_t w[4];
    bits(whole, w);
    for (int e = 0; e < n % 8; ++e) {
      const long long at = whole * 8 + e;
      const float r = kResidual ? load_elem<kType>(residual, at) : 0.f;
      const uint32_t v = (e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu) << 16;
      store_elem<kType>(y, at, v >= high && !none ? fmaf(load_elem<kType>(x, at), scale, r) : r);
    }
  }
}

template <int kType>
static int launch_dropout(const void* x, const void* residual, void* y, const long long* state, long long* state_copy, uint32_t call,
                          uint32_t drop, long long n, cudaStream_t st) {
  const long long need = (n / 8 + kDropThreads - 1) / kDropThreads, wave = static_cast<long long>(kDropBlocks) * sm_count();
  const unsigned blocks = static_cast<unsigned>(need < 1 ? 1 : need < wave ? need : wave);
  const float scale = drop < 65536u ? 65536.f / static_cast<float>(65536u - drop) : 0.f;   // 0: nothing is kept, and `high` does not count
  const auto kern = residual != nullptr ? dropout_kernel<kType, true> : dropout_kernel<kType, false>;
  kern<<<blocks, kDropThreads, 0, st>>>(x, residual, y, state, state_copy, call, drop << 16, scale, n);
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
