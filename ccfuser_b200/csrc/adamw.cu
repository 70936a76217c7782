// AdamW over many tensors in one launch (Loshchilov, Hutter: "Decoupled weight decay regularization", 2019):
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32 whatever the weights' type, rounded once. Moments lie in fp32 or in 8 bits.
//
// 8 bits: CCF_ADAMW_BLOCK weights share a power of two 2^E per moment, the binade of the block's largest value (one byte, E + 127, at least 40; 255: the block
// holds something that is not finite, and all of it is NaN from then on). A code is a small float relative to it: sign, 4 bits of exponent and 3 of mantissa
// for m (17 binades down to the smallest), 5 and 3 for v (33 binades), with gradual underflow. A scale that is a power of two makes a code the upper
// bits of a float, so that coding is an integer addition and a shift. What counts for training is the rounding: with b2 = 0.999 a step changes v by 0.1 %
// where codes lie 6 to 12 % apart, and rounding to nearest would lose every such change. A value is rounded up or down by 20 bits of a hash, up as often as
// it is near, so that the mean of what is stored is the value. A positive v never becomes 0: m / sqrt(v) would be without bound.
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

struct AdamScalars {
  float decay, rate, inv_root, pad0;   // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned key, pad1, pad2, pad3;
};
static_assert(sizeof(AdamScalars) == 32);

struct AdamEntry {
  CcfAdamwTensor t;
  unsigned first_block, key;           // key: added to the step's
};

template <int kCount>
struct AdamTable {
  const AdamScalars* device;           // in the place of `now`
  AdamScalars now;
  float b1, one_b1, b2, one_b2, eps;
  int count;
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
  s.decay = static_cast<float>(1.0 - lr * wd);
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

// A code's value is its bits as those of a float (of the smallest exponents: with hardware subnormals) times 2^120 2^(E - 8), or 2^100 2^(E - 4).
struct Scale {
  float m, v;
  __device__ __forceinline__ Scale(unsigned em, unsigned ev) {
    // a block that holds something not finite: NaN times whatever its codes are
    m = em == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(static_cast<int>(max(em, 40u)) - 127 - 8);
    v = ev == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(static_cast<int>(max(ev, 40u)) - 127 - 4);
  }
};
__device__ __forceinline__ float first_value(unsigned code, const Scale& s) {
  return __fmul_rn(__fmul_rn(__uint_as_float((code & 0x7fu) << 20 | (code & 0x80u) << 24), 0x1p120f), s.m);
}
__device__ __forceinline__ float second_value(unsigned code, const Scale& s) {
  return __fmul_rn(__fmul_rn(__uint_as_float(code << 20), 0x1p100f), s.v);
}
// the biased exponent of a block whose largest magnitude has these bits: one more where rounding up could leave its binade
__device__ __forceinline__ unsigned block_exponent(unsigned largest) {
  return largest >= 0x7f800000u ? 255u : max((largest + 0xfffffu) >> 23, 40u);
}
__device__ __forceinline__ unsigned first_code(float m, float inverse, unsigned bits) {
  const unsigned u = __float_as_uint(__fmul_rn(__fmul_rn(fabsf(m), inverse), 0x1p-120f));
  return ((u + bits) >> 20) | ((__float_as_uint(m) >> 24) & 0x80u);
}
__device__ __forceinline__ unsigned second_code(float v, float inverse, unsigned bits) {
  const unsigned u = __float_as_uint(__fmul_rn(__fmul_rn(v, inverse), 0x1p-100f));
  const unsigned code = (u + bits) >> 20;
  return v > 0.f ? max(code, 1u) : code;
}

// ---- the step --------------------------------------------------------------------------------------------------------
template <int kCount>
__device__ __forceinline__ int find_entry(const AdamTable<kCount>& a) {
  int lo = 0, hi = a.count;   // the last entry whose first block is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.entry[mid].first_block <= blockIdx.x) lo = mid; else hi = mid;
  }
  return lo;
}

struct AdamRates {
  float b1, one_b1, b2, one_b2, eps;
};

__device__ __forceinline__ void moments(float g, float& m, float& v, const AdamRates& r) {
  m = __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.one_b1));
  v = __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.one_b2));
}
__device__ __forceinline__ float updated(float p, float m, float v, const AdamRates& r, const AdamScalars& s) {
  const float root = fmaf(sqrtf(v), s.inv_root, r.eps);
  return fmaf(p, s.decay, -s.rate * (m / root));
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

template <int kType, int kCount>
__global__ void __launch_bounds__(kAdamThreads) adamw32_kernel(const __grid_constant__ AdamTable<kCount> a) {
  const AdamEntry& e = a.entry[find_entry(a)];
  const AdamScalars s = a.device != nullptr ? *a.device : a.now;
  const AdamRates r = {a.b1, a.one_b1, a.b2, a.one_b2, a.eps};
  const long long n = e.t.n, at = static_cast<long long>(blockIdx.x - e.first_block) * kAdamChunk + threadIdx.x * kAdamPer;
  if (at >= n) return;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(e.t.p) | reinterpret_cast<uintptr_t>(e.t.g) | reinterpret_cast<uintptr_t>(e.t.m) | reinterpret_cast<uintptr_t>(e.t.v);
  if ((bits & 15) == 0 && at + kAdamPer <= n) {
    float p[8], g[8], m[8], v[8];
    load_eight<kType>(e.t.p, at, p);
    load_eight<kType>(e.t.g, at, g);
    load_eight<kFp32>(e.t.m, at, m);
    load_eight<kFp32>(e.t.v, at, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      moments(g[i], m[i], v[i], r);
      p[i] = updated(p[i], m[i], v[i], r, s);
    }
    store_eight<kType>(e.t.p, at, p);
    store_eight<kFp32>(e.t.m, at, m);
    store_eight<kFp32>(e.t.v, at, v);
    return;
  }
  float* const pm = static_cast<float*>(e.t.m);
  float* const pv = static_cast<float*>(e.t.v);
  for (long long i = at; i < min(at + kAdamPer, n); ++i) {
    float m = pm[i], v = pv[i];
    moments(load_elem<kType>(e.t.g, i), m, v, r);
    pm[i] = m;
    pv[i] = v;
    store_elem<kType>(e.t.p, i, updated(load_elem<kType>(e.t.p, i), m, v, r, s));
  }
}

// a warp has a block of CCF_ADAMW_BLOCK weights, eight a lane
template <int kType, int kCount>
__global__ void __launch_bounds__(kAdamThreads) adamw8_kernel(const __grid_constant__ AdamTable<kCount> a) {
  const AdamEntry& e = a.entry[find_entry(a)];
  const AdamScalars s = a.device != nullptr ? *a.device : a.now;
  const AdamRates r = {a.b1, a.one_b1, a.b2, a.one_b2, a.eps};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long width = e.t.n / e.t.rows, per_row = (width + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK;
  const long long block = static_cast<long long>(blockIdx.x - e.first_block) * (kAdamThreads / 32) + warp;
  const long long row = block / per_row, begin = (block - row * per_row) * CCF_ADAMW_BLOCK;
  if (row >= e.t.rows) return;
  const int here = static_cast<int>(min(static_cast<long long>(kAdamPer), max(width - begin - lane * kAdamPer, 0ll)));   // weights of this lane
  const long long at = row * width + begin + lane * kAdamPer;
  unsigned char* const pm = static_cast<unsigned char*>(e.t.m);
  unsigned char* const pv = static_cast<unsigned char*>(e.t.v);
  const Scale scale(e.t.e[2 * block], e.t.e[2 * block + 1]);
  const uintptr_t bits = (reinterpret_cast<uintptr_t>(e.t.p) + at * kElemBytes<kType>) | (reinterpret_cast<uintptr_t>(e.t.g) + at * kElemBytes<kType>) |
                         (reinterpret_cast<uintptr_t>(pm + at) << 1) | (reinterpret_cast<uintptr_t>(pv + at) << 1);
  const bool whole = here == kAdamPer && (bits & 15) == 0;
  float p[8] = {}, g[8] = {}, m[8] = {}, v[8] = {};
  if (whole) {
    load_eight<kType>(e.t.p, at, p);
    load_eight<kType>(e.t.g, at, g);
    const uint2 cm = *reinterpret_cast<const uint2*>(pm + at), cv = *reinterpret_cast<const uint2*>(pv + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = first_value(((i < 4 ? cm.x : cm.y) >> (8 * (i & 3))) & 0xffu, scale);
      v[i] = second_value(((i < 4 ? cv.x : cv.y) >> (8 * (i & 3))) & 0xffu, scale);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= here) break;
      p[i] = load_elem<kType>(e.t.p, at + i);
      g[i] = load_elem<kType>(e.t.g, at + i);
      m[i] = first_value(pm[at + i], scale);
      v[i] = second_value(pv[at + i], scale);
    }
  }
  unsigned top_m = 0, top_v = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    moments(g[i], m[i], v[i], r);
    top_m = max(top_m, __float_as_uint(m[i]) & 0x7fffffffu);
    top_v = max(top_v, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  const unsigned em = block_exponent(__reduce_max_sync(0xffffffffu, top_m)), ev = block_exponent(__reduce_max_sync(0xffffffffu, top_v));
  const float im = power_of_two(em == 255 ? 0 : 127 + 8 - static_cast<int>(em)), iv = power_of_two(ev == 255 ? 0 : 127 + 4 - static_cast<int>(ev));
  const unsigned key = s.key + e.key + static_cast<unsigned>(at);
  unsigned cm[8], cv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned h = mix(key + i);
    cm[i] = em == 255 ? 0u : first_code(m[i], im, h & 0xfffffu);
    cv[i] = ev == 255 ? 0u : second_code(v[i], iv, h >> 12);
    p[i] = updated(p[i], m[i], v[i], r, s);
  }
  if (whole) {
    store_eight<kType>(e.t.p, at, p);
    *reinterpret_cast<uint2*>(pm + at) = make_uint2(cm[0] | cm[1] << 8 | cm[2] << 16 | cm[3] << 24, cm[4] | cm[5] << 8 | cm[6] << 16 | cm[7] << 24);
    *reinterpret_cast<uint2*>(pv + at) = make_uint2(cv[0] | cv[1] << 8 | cv[2] << 16 | cv[3] << 24, cv[4] | cv[5] << 8 | cv[6] << 16 | cv[7] << 24);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= here) break;
      store_elem<kType>(e.t.p, at + i, p[i]);
      pm[at + i] = static_cast<unsigned char>(cm[i]);
      pv[at + i] = static_cast<unsigned char>(cv[i]);
    }
  }
  if (lane == 0) {
    e.t.e[2 * block] = static_cast<unsigned char>(em);
    e.t.e[2 * block + 1] = static_cast<unsigned char>(ev);
  }
}

template <int kType, bool kSecond>
__global__ void __launch_bounds__(kAdamThreads) state_values_kernel(const unsigned char* codes, const unsigned char* ex, void* out, long long width, long long rows) {
  const int lane = threadIdx.x & 31;
  const long long per_row = (width + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK;
  const long long block = static_cast<long long>(blockIdx.x) * (kAdamThreads / 32) + (threadIdx.x >> 5);
  const long long row = block / per_row, begin = (block - row * per_row) * CCF_ADAMW_BLOCK;
  if (row >= rows) return;
  const int here = static_cast<int>(min(static_cast<long long>(kAdamPer), max(width - begin - lane * kAdamPer, 0ll)));
  const long long at = row * width + begin + lane * kAdamPer;
  const Scale scale(ex[2 * block], ex[2 * block + 1]);
  const uintptr_t bits = (reinterpret_cast<uintptr_t>(codes + at) << 1) | (reinterpret_cast<uintptr_t>(out) + at * kElemBytes<kType>);
  float f[8];
  if (here == kAdamPer && (bits & 15) == 0) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned x = ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xffu;
      f[i] = kSecond ? second_value(x, scale) : first_value(x, scale);
    }
    store_eight<kType>(out, at, f);
  } else {
    for (int i = 0; i < here; ++i) store_elem<kType>(out, at + i, kSecond ? second_value(codes[at + i], scale) : first_value(codes[at + i], scale));
  }
}

inline long long blocks_of(const CcfAdamwTensor& t) {
  if (t.e == nullptr) return (t.n + kAdamChunk - 1) / kAdamChunk;
  const long long width = t.n / t.rows, warps = t.rows * ((width + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK);
  return (warps + kAdamThreads / 32 - 1) / (kAdamThreads / 32);
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
  t.count = count;
  long long blocks = 0;
  for (int i = 0; i < count; ++i) {
    t.entry[i].t = a.tensors[first + i];
    t.entry[i].first_block = static_cast<unsigned>(blocks);
    t.entry[i].key = static_cast<unsigned>(a.tensors[first + i].number) * 0x9E3779B9u;
    blocks += blocks_of(a.tensors[first + i]);
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
        (t.e == nullptr && (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) % 4 != 0) || blocks_of(t) > 0x7fffffff)
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
  const long long blocks = blocks_of(t);
  if (blocks > 0x7fffffff) return -2;
  const unsigned char* const c = static_cast<const unsigned char*>(codes);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto kern = type == kBf16   ? (second ? state_values_kernel<kBf16, true> : state_values_kernel<kBf16, false>)
                    : type == kFp16 ? (second ? state_values_kernel<kFp16, true> : state_values_kernel<kFp16, false>)
                                    : (second ? state_values_kernel<kFp32, true> : state_values_kernel<kFp32, false>);
  kern<<<static_cast<unsigned>(blocks), kAdamThreads, 0, st>>>(c, e, out, n / rows, rows);
  return launch_result();
}

}  // extern "C"
