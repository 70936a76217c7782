// AdamW over many tensors in one launch (Loshchilov, Hutter: "Decoupled weight decay regularization", 2019):
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32 whatever the weights' type, rounded once. Moments lie in fp32 or in 8 bits.
//
// 8 bits: CCF_ADAMW_BLOCK weights share a power of two 2^E per moment, the binade of the block's largest value (one byte, E + 127, at least 40; 255: the block
// holds something that is not finite, or above 1.875 2^127, and all of it is NaN from then on). A code is a small float relative to it: sign, 4 bits of exponent and 3 of mantissa
// for m (17 binades down to the smallest), 5 and 3 for v (33 binades), with gradual underflow. A scale that is a power of two makes a code the upper
// bits of a float, so that coding is an integer addition and a shift. What counts for training is the rounding: with b2 = 0.999 a step changes v by 0.1 %
// where codes lie 6 to 12 % apart, and rounding to nearest would lose every such change. A value is rounded up or down by 20 bits of a hash, up as often as
// it is near, so that the mean of what is stored is the value, for m at every size and for v down to the smallest code, some 2^-33 of its block's largest value. A positive v
// never becomes 0 (m / sqrt(v) would be without bound): below that it is held as the smallest code, which is more than it is, and its weights move less.
// The hash: MurmurHash3's last step (Appleby, 2011) of the weight's number plus a key of (seed, step, tensor), which comes from SplitMix64
// (Steele, Lea, Flood: "Fast splittable pseudorandom number generators", 2014).
//
// m, v and their codes are computed with one rounding an operation, so that they are the same bits as torch's operations give.
#include <cmath>

#include "adamw.h"
#include "elements.cuh"

namespace ccf {

constexpr int kAdamThreads = 256;
constexpr int kAdamPer = 8;                                   // weights of a thread at a time
constexpr int kAdamChunk = kAdamThreads * kAdamPer;           // of a block
constexpr int kAdamMost = 400;                                // tensors of a launch: kernel arguments end at 32 KB
constexpr int kAdamFew = 32;
// 8-bit moments. Blocks per SM: as many as leave the registers in place (16-bit weights: four 470, five 424, six 415 us for 200 M; fp32 518, 477, 489)
template <int kType>
constexpr int kAdam8Blocks = kType == kFp32 ? 5 : 6;
// Blocks of weights that a warp takes one after another, while two waves of thread blocks are left: what a thread block does first (its tensor, its constants) is a tenth of
// one turn. 285 M weights of 14 tensors with one, four, eight and sixteen turns 710, 599, 581 and 561 us. Not fp32 weights: the loop does not fit their registers (738 -> 845).
constexpr int kAdam8Turns = 16;

struct AdamScalars {
  float decay, rate, inv_root, pad0;   // lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned key, pad1, pad2, pad3;
};
static_assert(sizeof(AdamScalars) == 32);

struct AdamEntry {
  void* p;
  const void* g;
  void* m;
  void* v;
  unsigned char* e;
  long long n, width;                  // width: weights of a row
  unsigned row_blocks;                 // blocks of CCF_ADAMW_BLOCK of a row; 0: one row alone
  unsigned first_block, key;           // key: added to the step's
  unsigned vectors;                    // 1: eight weights and their moments are read at once wherever a lane begins, 2: their gradients too
};

template <int kCount>
struct AdamTable {
  const AdamScalars* device;           // in the place of `now`
  AdamScalars now;
  float b1, one_b1, b2, one_b2, eps;
  float minus_zero;
  int count, turns;                    // turns: blocks of weights of a warp, one after another
  AdamEntry entry[kCount];
};
static_assert(sizeof(AdamTable<kAdamMost>) <= 32764);

__host__ __device__ inline unsigned long long split_mix(unsigned long long x) {
  x += 0x9E3779B97F4A7C15ull;
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

__host__ __device__ inline AdamScalars adam_scalars(double lr, double b1, double b2, double wd, unsigned long long seed, long long step) {
  AdamScalars s = {};
  const double t = static_cast<double>(step);
  s.decay = static_cast<float>(lr * wd);
  s.rate = static_cast<float>(lr / (1.0 - pow(b1, t)));
  s.inv_root = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, t)));
  s.key = static_cast<unsigned>(split_mix(split_mix(seed) ^ static_cast<unsigned long long>(step)) >> 32);
  return s;
}

__global__ void adam_scalars_kernel(AdamScalars* out, long long* counter, const float* device_lr, double lr, double b1, double b2, double wd,
                                    unsigned long long seed) {
  const long long step = ++*counter;
  *out = adam_scalars(device_lr != nullptr ? static_cast<double>(*device_lr) : lr, b1, b2, wd, seed, step);
}

__device__ __forceinline__ unsigned mix(unsigned h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// ---- 8 bits ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float(static_cast<unsigned>(exponent + 127) << 23); }

// The factors of a block's codes: 2^E of the first moments as halves, 2^(E - 4) of the second as floats of the smallest exponents (subnormal ones among
// them), which are 2^100 times as large first.
struct Scale {
  float m, v;
  __device__ __forceinline__ Scale(unsigned em, unsigned ev) {
    // a block that holds something not finite: NaN times whatever its codes are
    m = em == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(static_cast<int>(max(em, 40u)) - 127);
    v = ev == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(static_cast<int>(max(ev, 40u)) - 127 - 4);
  }
};
// the biased exponent of a block whose largest magnitude has these bits: one more where rounding up could leave its binade
__device__ __forceinline__ unsigned block_exponent(unsigned largest) {
  return largest >= 0x7f800000u ? 255u : max((largest + 0xfffffu) >> 23, 40u);
}

// ---- the step --------------------------------------------------------------------------------------------------------
// The entry of this thread block: the last one whose first block is not behind it.
template <int kCount>
__device__ __forceinline__ int find_entry(const AdamTable<kCount>& a) {
  if (a.count == 1) return 0;
  __shared__ int found;
  if (threadIdx.x == 0) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.entry[mid].first_block <= blockIdx.x) lo = mid; else hi = mid;
    }
    found = lo;
  }
  __syncthreads();
  return found;
}

struct AdamRates {
  float b1, one_b1, b2, one_b2, eps;
};

// one rounding an operation
__device__ __forceinline__ void moments(float g, float& m, float& v, const AdamRates& r) {
  m = __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.one_b1));
  v = __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.one_b2));
}
// What is taken off is added up first: 1 - lr wd of 1 - 1e-6 would be a hundredth of lr wd off in fp32, the same way in every step.
__device__ __forceinline__ float updated(float p, float m, float v, const AdamRates& r, const AdamScalars& s) {
  const float root = fmaf(sqrtf(v), s.inv_root, r.eps);
  return p - fmaf(p, s.decay, s.rate * (m / root));
}

template <int kType>
__device__ __forceinline__ void load_eight(const void* base, long long at, float (&f)[8]) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * kElemBytes<kType>);
#pragma unroll
  for (int i = 0; i < 8 / kElemsPer16<kType>; ++i) {
    float part[kElemsPer16<kType>];
    unpack16<kType>(q[i], part);
#pragma unroll
    for (int j = 0; j < kElemsPer16<kType>; ++j) f[i * kElemsPer16<kType> + j] = part[j];
  }
}
// One weight. A plain read: load_elem's is for data that nothing writes while the kernel runs, and weights are written.
template <int kType>
__device__ __forceinline__ float load_weight(const void* p, long long i) {
  if constexpr (kType == kFp32) return static_cast<const float*>(p)[i];
  else if constexpr (kType == kFp16) return __half2float(static_cast<const __half*>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <int kType>
__device__ __forceinline__ void load_gradients(const AdamEntry& e, long long at, float (&g)[8]) {
  if ((e.vectors & 2) != 0) {
    load_eight<kType>(e.g, at, g);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = load_elem<kType>(e.g, at + i);
  }
}
template <int kType>
__device__ __forceinline__ void store_eight(void* base, long long at, const float (&f)[8]) {
  uint4* q = reinterpret_cast<uint4*>(static_cast<char*>(base) + at * kElemBytes<kType>);
#pragma unroll
  for (int i = 0; i < 8 / kElemsPer16<kType>; ++i) {
    float part[kElemsPer16<kType>];
#pragma unroll
    for (int j = 0; j < kElemsPer16<kType>; ++j) part[j] = f[i * kElemsPer16<kType> + j];
    q[i] = pack16<kType>(part);
  }
}

// Moments in fp32. Bound by memory: 22 bytes a weight of bf16, 28 of fp32; 285 M weights of 14 tensors 901 us at full clocks and 960 to 1005
// in a long run, where the card holds its clock down for power (the copy rate says 960), 18.9 M fp32 weights of 96 tensors 79 to 82 us (81).
template <int kType, int kCount>
__global__ void __launch_bounds__(kAdamThreads) adamw32_kernel(const __grid_constant__ AdamTable<kCount> a) {
  const AdamEntry& e = a.entry[find_entry(a)];
  const AdamScalars s = a.device != nullptr ? *a.device : a.now;
  const AdamRates r = {a.b1, a.one_b1, a.b2, a.one_b2, a.eps};
  const long long n = e.n, at = static_cast<long long>(blockIdx.x - e.first_block) * kAdamChunk + threadIdx.x * kAdamPer;
  if (at >= n) return;
  if ((e.vectors & 1) != 0 && at + kAdamPer <= n) {
    float p[8], g[8], m[8], v[8];
    load_eight<kType>(e.p, at, p);
    load_gradients<kType>(e, at, g);
    load_eight<kFp32>(e.m, at, m);
    load_eight<kFp32>(e.v, at, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      moments(g[i], m[i], v[i], r);
      p[i] = updated(p[i], m[i], v[i], r, s);
    }
    store_eight<kType>(e.p, at, p);
    store_eight<kFp32>(e.m, at, m);
    store_eight<kFp32>(e.v, at, v);
    return;
  }
  float* const pm = static_cast<float*>(e.m);
  float* const pv = static_cast<float*>(e.v);
  for (long long i = at; i < min(at + kAdamPer, n); ++i) {
    float m = pm[i], v = pv[i];
    moments(load_elem<kType>(e.g, i), m, v, r);
    pm[i] = m;
    pv[i] = v;
    store_elem<kType>(e.p, i, updated(load_weight<kType>(e.p, i), m, v, r, s));
  }
}

// A warp has a block of CCF_ADAMW_BLOCK weights, eight a lane, as pairs: one instruction for two operations, each rounded as alone. Bound by what
// an SM does in a clock, and by nothing of it alone: no pipe is full (ALU 63 %, issue slots 73 %, 60 instructions a weight), the first stall is for memory, as nothing of a turn is read
// before the turn in front of it is stored, and the time goes with the clock: 285 M weights of 14 tensors of bf16 564 us at 1965 MHz, 602 to 618 at the 1750 that a long run is held to (436 at the
// copy rate); 722 of fp32 (697). Scalar arithmetic instead of pairs 464 us where pairs take 424, constants as pairs in the arguments 443, shifts as products 440 (200 M).
struct Place {
  long long block, at;   // of the tensor's blocks, first weight of this lane
  int here;              // its number of weights, 0 to 8
};
// `first`: the first block of this thread block
__device__ __forceinline__ Place place_of(long long first, long long n, long long width, unsigned row_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Place p;
  p.block = first + warp;
  long long left;
  if (row_blocks == 0) {
    p.at = first * CCF_ADAMW_BLOCK + threadIdx.x * kAdamPer;
    left = n - p.at;
  } else {
    const unsigned row = static_cast<unsigned>(p.block) / row_blocks;      // fewer than 2^32 blocks
    const long long in = (static_cast<unsigned>(p.block) - row * row_blocks) * static_cast<long long>(CCF_ADAMW_BLOCK) + lane * kAdamPer;
    p.at = row * width + in;
    left = p.at - lane * kAdamPer < n ? width - in : 0;
  }
  p.here = left >= kAdamPer ? kAdamPer : left > 0 ? static_cast<int>(left) : 0;
  return p;
}
// Gradients by themselves: those that lie in a bucket of many begin anywhere.
inline unsigned vectors_of(const void* p, const void* g, const void* m, const void* v, long long n, long long rows, bool eight) {
  const uintptr_t moments = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  const bool rows_too = rows == 1 || n / rows % 8 == 0;
  return (reinterpret_cast<uintptr_t>(p) % 16 == 0 && moments % (eight ? 8 : 16) == 0 && rows_too ? 1u : 0u) |
         (reinterpret_cast<uintptr_t>(g) % 16 == 0 && rows_too ? 2u : 0u);
}

// A product that is rounded before something is added to it. The compiler merges a packed product with the packed sum behind it (a code of one weight in some
// 50000 then differs), also one written as an fma with the constant -0; of a -0 that it does not know it cannot.
__device__ __forceinline__ f32x2 product2(f32x2 a, f32x2 b, f32x2 minus_zero) { return fma2(a, b, minus_zero); }
// Two codes of a word (bytes 2 k and 2 k + 1) as floats, of blocks with E = 0. The first moment's sign, 4 and 3 bits are those of a half without its highest bit of
// exponent, subnormals included; the second's 5 and 3 bits those of a bf16 (and a float) without the highest three.
__device__ __forceinline__ f32x2 first_pair(unsigned codes, int k) {
  const unsigned t = __byte_perm(codes, 0, k == 0 ? 0x4140 : 0x4342) << 7;
  const unsigned h = t + (t & 0x40004000u);      // the sign one place up
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pk2(f.x, f.y);
}
__device__ __forceinline__ f32x2 second_pair(unsigned codes, int k) {
  const unsigned t = __byte_perm(codes, 0, k == 0 ? 0x4140 : 0x4342) << 4;
  return pk2(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
}
// the largest of three magnitudes; NaN if one is
__device__ __forceinline__ float largest(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// codes from bits 20 to 27 of four words, the first moment's sign from bit 31
template <bool kSecond>
__device__ __forceinline__ unsigned four_codes(const unsigned* w) {
  const unsigned x = __byte_perm(w[0], w[1], 0x7632), y = __byte_perm(w[2], w[3], 0x7632);      // upper halves
  const unsigned codes = __byte_perm(x >> 4, y >> 4, 0x6420);
  return kSecond ? codes : codes | (__byte_perm(x, y, 0x7531) & 0x80808080u);
}
// The inverses of sqrt(v) / sqrt(1 - b2^t) + eps by the hardware's approximations; subnormal v count as 0 there, which eps covers from 1e-10 on. They are some 2^-22 of
// the update off, where moments of 3 bits of mantissa are up to an eighth off themselves; the step with moments in fp32 rounds correctly. Below 1e-10 it is rounded correctly here too.
template <bool kFast>
__device__ __forceinline__ f32x2 inverse_roots(f32x2 v2, const AdamRates& r, const AdamScalars& s) {
  float v[2], root[2];
  upk2(v2, v[0], v[1]);
  if constexpr (kFast) {
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root[0]) : "f"(v[0]));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root[1]) : "f"(v[1]));
    upk2(fma2(pk2(root[0], root[1]), bc2(s.inv_root), bc2(r.eps)), v[0], v[1]);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(root[0]) : "f"(v[0]));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(root[1]) : "f"(v[1]));
    return pk2(root[0], root[1]);
  }
  return pk2(1.f / fmaf(sqrtf(v[0]), s.inv_root, r.eps), 1.f / fmaf(sqrtf(v[1]), s.inv_root, r.eps));
}
template <bool kFast>
__device__ __forceinline__ void update_pairs(float (&p)[8], const f32x2 (&m)[4], const f32x2 (&v)[4], const AdamRates& r, const AdamScalars& s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 step = mul2(mul2(m[i], inverse_roots<kFast>(v[i], r, s)), bc2(-s.rate)), old = pk2(p[2 * i], p[2 * i + 1]);
    upk2(add2(old, fma2(old, bc2(-s.decay), step)), p[2 * i], p[2 * i + 1]);
  }
}

template <int kType, int kCount>
__global__ void __launch_bounds__(kAdamThreads, kAdam8Blocks<kType>) adamw8_kernel(const __grid_constant__ AdamTable<kCount> a) {
  const AdamEntry& e = a.entry[find_entry(a)];
  const AdamScalars s = a.device != nullptr ? *a.device : a.now;
  const AdamRates r = {a.b1, a.one_b1, a.b2, a.one_b2, a.eps};
  unsigned char* const pm = static_cast<unsigned char*>(e.m);
  unsigned char* const pv = static_cast<unsigned char*>(e.v);
  long long first = static_cast<long long>(blockIdx.x - e.first_block) * (kType == kFp32 ? 1 : a.turns) * (kAdamThreads / 32);
#pragma unroll 1
  for (int turn = 0; turn < (kType == kFp32 ? 1 : a.turns); ++turn, first += kAdamThreads / 32) {
    const Place place = place_of(first, e.n, e.width, e.row_blocks);
    const long long at = place.at, block = place.block;
    const int here = place.here;
    if (__all_sync(0xffffffffu, here == 0)) return;      // a warp behind the last block
    const bool whole = here == kAdamPer && (e.vectors & 1) != 0;
    float p[8] = {}, g[8] = {};
    uint2 cm = {}, cv = {};
    if (whole) {
      cm = *reinterpret_cast<const uint2*>(pm + at);
      cv = *reinterpret_cast<const uint2*>(pv + at);
      load_gradients<kType>(e, at, g);
      load_eight<kType>(e.p, at, p);
    } else {
      unsigned bm[2] = {}, bv[2] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= here) break;
        bm[i / 4] |= static_cast<unsigned>(pm[at + i]) << (8 * (i & 3));
        bv[i / 4] |= static_cast<unsigned>(pv[at + i]) << (8 * (i & 3));
        g[i] = load_elem<kType>(e.g, at + i);
        p[i] = load_weight<kType>(e.p, at + i);
      }
      cm = make_uint2(bm[0], bm[1]);
      cv = make_uint2(bv[0], bv[1]);
    }
    const Scale old(e.e[2 * block], e.e[2 * block + 1]);
    const f32x2 nought = bc2(a.minus_zero);
    f32x2 m[4], v[4];
    float top_m = 0.f, top_v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 g2 = pk2(g[2 * i], g[2 * i + 1]);
      m[i] = mul2(first_pair(i < 2 ? cm.x : cm.y, i & 1), bc2(old.m));
      v[i] = mul2(mul2(second_pair(i < 2 ? cv.x : cv.y, i & 1), bc2(0x1p100f)), bc2(old.v));
      m[i] = add2(product2(m[i], bc2(r.b1), nought), product2(g2, bc2(r.one_b1), nought));
      v[i] = add2(product2(v[i], bc2(r.b2), nought), product2(mul2(g2, g2), bc2(r.one_b2), nought));
      float x, y;
      upk2(m[i], x, y);
      top_m = largest(top_m, x, y);
      upk2(v[i], x, y);
      top_v = largest(top_v, x, y);
    }
    const unsigned all_m = __reduce_max_sync(0xffffffffu, __float_as_uint(top_m)), all_v = __reduce_max_sync(0xffffffffu, __float_as_uint(top_v));
    // the weights first: their registers are free for the codes then
    if (r.eps >= 1e-10f) update_pairs<true>(p, m, v, r, s);
    else update_pairs<false>(p, m, v, r, s);
    if (whole) {
      store_eight<kType>(e.p, at, p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < here) store_elem<kType>(e.p, at + i, p[i]);
    }
    const unsigned em = block_exponent(all_m), ev = block_exponent(all_v);
    const bool near = em <= 127 + 14 && ev <= 127 + 30;      // else the factors of the way back leave the range of fp32 and are two
    const f32x2 im = bc2(power_of_two(near ? 127 - 112 - static_cast<int>(em) : em == 255 ? 0 : 127 + 8 - static_cast<int>(em)));
    const f32x2 iv = bc2(power_of_two(near ? 127 - 96 - static_cast<int>(ev) : ev == 255 ? 0 : 127 + 4 - static_cast<int>(ev)));
    const unsigned key = s.key + e.key + static_cast<unsigned>(at);
    unsigned nm[2], nv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      unsigned wm[4], wv[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x2 dm = mul2(m[2 * q + i], im), dv = mul2(v[2 * q + i], iv);
        if (!near) {
          dm = mul2(dm, bc2(0x1p-120f));
          dv = mul2(dv, bc2(0x1p-100f));
        }
        float xm[2], xv[2];
        upk2(dm, xm[0], xm[1]);
        upk2(dv, xv[0], xv[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned h = mix(key + 4 * q + 2 * i + k), u = __float_as_uint(xm[k]);
          wm[2 * i + k] = u + (h << 12 >> 12);      // does not reach the sign
          wv[2 * i + k] = __float_as_uint(xv[k]) + (h >> 12);
        }
      }
      nm[q] = em == 255 ? 0u : four_codes<false>(wm);
      nv[q] = four_codes<true>(wv);
      if ((nv[q] - 0x01010101u) & ~nv[q] & 0x80808080u) {      // a code of 0: of 0 alone
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float o[2];
          upk2(v[2 * q + i / 2], o[0], o[1]);
          if ((nv[q] >> (8 * i) & 0xffu) == 0 && o[i & 1] > 0.f) nv[q] |= 1u << (8 * i);
        }
      }
      if (ev == 255) nv[q] = 0;
    }
    if (whole) {
      *reinterpret_cast<uint2*>(pm + at) = make_uint2(nm[0], nm[1]);
      *reinterpret_cast<uint2*>(pv + at) = make_uint2(nv[0], nv[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= here) break;
        pm[at + i] = static_cast<unsigned char>(nm[i / 4] >> (8 * (i & 3)));
        pv[at + i] = static_cast<unsigned char>(nv[i / 4] >> (8 * (i & 3)));
      }
    }
    if ((threadIdx.x & 31) == 0) {
      e.e[2 * block] = static_cast<unsigned char>(em);
      e.e[2 * block + 1] = static_cast<unsigned char>(ev);
    }
  }
}

// Values of codes, for those who want them in numbers. Bound by memory: 200 M codes to bf16 95 us with four blocks of weights in flight a warp (floor 92), 98 with two, 119 with
// one.
constexpr int kStateTurns = 4;
template <int kType, bool kSecond>
__global__ void __launch_bounds__(kAdamThreads)
    state_values_kernel(const unsigned char* codes, const unsigned char* ex, void* out, long long n, long long width, unsigned row_blocks, unsigned vectors) {
  Place place[kStateTurns];
  uint2 c[kStateTurns];
  unsigned e[kStateTurns][2];
#pragma unroll
  for (int k = 0; k < kStateTurns; ++k) {
    place[k] = place_of((static_cast<long long>(blockIdx.x) * kStateTurns + k) * (kAdamThreads / 32), n, width, row_blocks);
    c[k] = {};
    if (place[k].here == 0) continue;
    e[k][0] = ex[2 * place[k].block];
    e[k][1] = ex[2 * place[k].block + 1];
    if (place[k].here == kAdamPer && (vectors & 1) != 0) {
      c[k] = __ldg(reinterpret_cast<const uint2*>(codes + place[k].at));
    } else {
      unsigned b[2] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < place[k].here) b[i / 4] |= static_cast<unsigned>(codes[place[k].at + i]) << (8 * (i & 3));
      c[k] = make_uint2(b[0], b[1]);
    }
  }
#pragma unroll
  for (int k = 0; k < kStateTurns; ++k) {
    if (place[k].here == 0) continue;
    const Scale scale(e[k][0], e[k][1]);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned word = i < 2 ? c[k].x : c[k].y;
      upk2(kSecond ? mul2(mul2(second_pair(word, i & 1), bc2(0x1p100f)), bc2(scale.v)) : mul2(first_pair(word, i & 1), bc2(scale.m)), f[2 * i], f[2 * i + 1]);
    }
    if (place[k].here == kAdamPer && (vectors & 1) != 0) {
      store_eight<kType>(out, place[k].at, f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < place[k].here) store_elem<kType>(out, place[k].at + i, f[i]);
    }
  }
}

inline unsigned row_blocks_of(long long n, long long rows) {
  return rows == 1 ? 0u : static_cast<unsigned>((n / rows + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK);
}
inline long long blocks_of(const CcfAdamwTensor& t) {
  if (t.e == nullptr) return (t.n + kAdamChunk - 1) / kAdamChunk;
  const long long width = t.n / t.rows, warps = t.rows * ((width + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK);
  return (warps + kAdamThreads / 32 - 1) / (kAdamThreads / 32);
}

// blocks of the grid, and blocks of weights where they are divided into rows, in 32 bits
inline bool blocks_fit(const CcfAdamwTensor& t) {
  return blocks_of(t) <= 0x7fffffff && (t.e == nullptr || t.rows == 1 || t.rows * static_cast<long long>(row_blocks_of(t.n, t.rows)) <= 0xffffff00ll);
}

template <int kType, int kCount>
static int launch_adamw(const CcfAdamw& a, int first, int count, cudaStream_t st) {
  AdamTable<kCount> t;
  t.device = static_cast<const AdamScalars*>(a.scalars);
  t.now = a.scalars != nullptr ? AdamScalars{} : adam_scalars(a.lr, a.beta1, a.beta2, a.weight_decay, a.seed, a.step);
  t.b1 = static_cast<float>(a.beta1);
  t.one_b1 = static_cast<float>(1.0 - a.beta1);
  t.b2 = static_cast<float>(a.beta2);
  t.one_b2 = static_cast<float>(1.0 - a.beta2);
  t.eps = static_cast<float>(a.eps);
  t.minus_zero = -0.f;
  t.count = count;
  long long blocks = 0;
  for (int i = 0; i < count; ++i) blocks += blocks_of(a.tensors[first + i]);
  t.turns = 1;
  if (a.tensors[first].e != nullptr && kType != kFp32) {
    const long long wave = kAdam8Blocks<kType> * sm_count();
    while (t.turns < kAdam8Turns && blocks / (2 * t.turns) >= 2 * wave) t.turns *= 2;
  }
  blocks = 0;
  for (int i = 0; i < count; ++i) {
    const CcfAdamwTensor& from = a.tensors[first + i];
    t.entry[i] = {from.p, from.g, from.m, from.v, from.e, from.n, from.n / from.rows, row_blocks_of(from.n, from.rows), static_cast<unsigned>(blocks),
                  static_cast<unsigned>(from.number) * 0x9E3779B9u, vectors_of(from.p, from.g, from.m, from.v, from.n, from.e != nullptr ? from.rows : 1, from.e != nullptr)};
    blocks += (blocks_of(from) + t.turns - 1) / t.turns;
  }
  const auto kern = a.tensors[first].e != nullptr ? adamw8_kernel<kType, kCount> : adamw32_kernel<kType, kCount>;
  kern<<<static_cast<unsigned>(blocks), kAdamThreads, 0, st>>>(t);
  return launch_result();
}

template <int kType>
static int run_adamw(const CcfAdamw& a, cudaStream_t st) {
  constexpr long long kGrid = 0x7fffffff;
  int launches = 0;
  for (int first = 0; first < a.count; ++launches) {
    int count = 0;
    for (long long blocks = 0; first + count < a.count && count < kAdamMost; ++count) {
      blocks += blocks_of(a.tensors[first + count]);
      if (count > 0 && blocks > kGrid) break;
    }
    const int rc = count <= kAdamFew ? launch_adamw<kType, kAdamFew>(a, first, count, st) : launch_adamw<kType, kAdamMost>(a, first, count, st);
    if (rc != 0) return rc;
    first += count;
  }
  return launches;
}

}  // namespace ccf

extern "C" {

int ccf_sizeof_adamw() { return static_cast<int>(sizeof(CcfAdamw)); }
int ccf_sizeof_adamw_tensor() { return static_cast<int>(sizeof(CcfAdamwTensor)); }

static bool adamw_rates_ok(const CcfAdamw& a) {
  return a.lr >= 0.0 && a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0 && a.eps >= 0.0 && a.weight_decay >= 0.0;
}

int ccf_adamw(const CcfAdamw* a, void* stream) {
  using namespace ccf;
  if (a->tensors == nullptr || a->count < 1 || a->type < 0 || a->type > 2 || !adamw_rates_ok(*a)) return -2;
  if (a->scalars != nullptr ? (reinterpret_cast<uintptr_t>(a->scalars) & 15) != 0 : a->step < 1) return -2;
  const uintptr_t size = a->type == kFp32 ? 4 : 2;
  for (int i = 0; i < a->count; ++i) {
    const CcfAdamwTensor& t = a->tensors[i];
    if (t.p == nullptr || t.g == nullptr || t.m == nullptr || t.v == nullptr || t.n < 1 || t.n > (1ll << 40) || t.rows < 1 || t.n % t.rows != 0 ||
        (t.e != nullptr) != (a->tensors[0].e != nullptr) || (reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) % size != 0 ||
        (t.e == nullptr && (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) % 4 != 0) || !blocks_fit(t))
      return -2;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a->type == kBf16 ? run_adamw<kBf16>(*a, st) : a->type == kFp16 ? run_adamw<kFp16>(*a, st) : run_adamw<kFp32>(*a, st);
}

int ccf_adamw_scalars(const CcfAdamw* a, long long* counter, const float* device_lr, void* scalars, void* stream) {
  using namespace ccf;
  if (counter == nullptr || scalars == nullptr || (reinterpret_cast<uintptr_t>(scalars) & 15) != 0 || !adamw_rates_ok(*a)) return -2;
  adam_scalars_kernel<<<1, 1, 0, reinterpret_cast<cudaStream_t>(stream)>>>(static_cast<AdamScalars*>(scalars), counter, device_lr, a->lr, a->beta1, a->beta2,
                                                                          a->weight_decay, a->seed);
  return launch_result();
}

int ccf_state_values(const void* codes, const unsigned char* e, void* out, long long n, long long rows, int second, int type, void* stream) {
  using namespace ccf;
  if (codes == nullptr || e == nullptr || out == nullptr || n < 1 || rows < 1 || n % rows != 0 || type < 0 || type > 2) return -2;
  CcfAdamwTensor t = {};
  t.e = const_cast<unsigned char*>(e);
  t.n = n;
  t.rows = rows;
  if (!blocks_fit(t)) return -2;
  const long long blocks = (blocks_of(t) + kStateTurns - 1) / kStateTurns;
  const unsigned char* const c = static_cast<const unsigned char*>(codes);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto kern = type == kBf16   ? (second ? state_values_kernel<kBf16, true> : state_values_kernel<kBf16, false>)
                    : type == kFp16 ? (second ? state_values_kernel<kFp16, true> : state_values_kernel<kFp16, false>)
                                    : (second ? state_values_kernel<kFp32, true> : state_values_kernel<kFp32, false>);
  kern<<<static_cast<unsigned>(blocks), kAdamThreads, 0, st>>>(c, e, out, n, n / rows, row_blocks_of(n, rows), vectors_of(out, nullptr, c, nullptr, n, rows, true));
  return launch_result();
}

}  // extern "C"
