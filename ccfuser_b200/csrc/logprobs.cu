// Log probabilities of given tokens, with the entropy and the best alternatives of every row of logits, and their gradient: the loss of the
// example models (mix_moe/mix_moe/examples/models/moe_gpt.py and transformer-xl/mem_transformer_mix_moe.py take torch's cross-entropy) and the scores
// of a sampled or a given text.
//
// With z = x / T over the first `vocab` columns, M the largest x, u_j = (x_j - M) / (T ln 2), S = sum 2^u_j, Q = sum 2^u_j u_j:
//   lp_j = (x_j - M) / T - ln S        H = ln S - ln 2 * Q / S        (both terms of H are >= 0: nothing cancels)
//   dx_j = 1/T * ( g [j = t] + sum_k g_k [j = top_k] - p_j (g + sum_k g_k + g_H (lp_j + H)) ),   p_j = 2^u_j / S
// One pass over the logits with running M, S and Q forward; one pass that reads them and writes the gradient backward. Both are bound by those
// bytes; next to them stand one exponential and about five more instructions an element. Statistics in fp32: a sum of V terms has V / 512 to V / 64
// additions in a row, and the terms' relative error of 2^-22 averages out; the gradient is rounded once, to the logits' type.
#include <cooperative_groups.h>

#include "elements.cuh"
#include "logprobs.h"

namespace ccf {

constexpr int kUnroll = 4;                 // 16-byte pieces that a thread has in flight
constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;
constexpr float kFloorU = -1000.f;         // 2^kFloorU is 0, and 0 * kFloorU is 0 where 0 * -inf would be NaN
constexpr uint32_t kNanOrder = 0xfffffffeu;

__device__ __forceinline__ float exp2_fast(float u) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// A whole number in the order of the floats; NaN above all, as in torch.topk; -0 is 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return kNanOrder;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return order == kNanOrder ? __int_as_float(0x7fc00000) : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// Larger value first, then lower index; 0 is no element.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t index) { return static_cast<uint64_t>(order_of(v)) << 32 | (0xffffffffu - index); }

template <int kType>
constexpr uint32_t kNegInf2 = kType == kBf16 ? 0xff80ff80u : kType == kFp16 ? 0xfc00fc00u : 0xff800000u;
// Elements are raised to this before the arithmetic, so that -inf needs no care there (0 * -inf): -1e30 in bf16 and fp32, the lowest fp16.
template <int kType>
constexpr uint32_t kFloorBits = kType == kBf16 ? 0xf14af14au : kType == kFp16 ? 0xfbfffbffu : 0xf149f2cau;
template <int kType>
constexpr float kFloor = kType == kFp16 ? -65504.f : -1e30f;

template <int kType>
struct Pair {
  using T = typename std::conditional<kType == kFp16, __half2, __nv_bfloat162>::type;
  static __device__ __forceinline__ T of(uint32_t w) { return *reinterpret_cast<T*>(&w); }
  static __device__ __forceinline__ uint32_t bits(T v) { return *reinterpret_cast<uint32_t*>(&v); }
};

template <int kType>
__device__ __forceinline__ uint32_t raise_word(uint32_t w) {
  if constexpr (kType == kFp32) return __float_as_uint(fmaxf(__uint_as_float(w), __uint_as_float(kFloorBits<kType>)));
  else return Pair<kType>::bits(__hmax2(Pair<kType>::of(w), Pair<kType>::of(kFloorBits<kType>)));
}
template <int kType>
__device__ __forceinline__ uint4 raised(const uint4& q) {
  return make_uint4(raise_word<kType>(q.x), raise_word<kType>(q.y), raise_word<kType>(q.z), raise_word<kType>(q.w));
}

// largest of the elements of kUnroll pieces; NaN if one is
template <int kType>
__device__ __forceinline__ float max_of(const uint4 (&q)[kUnroll]) {
  if constexpr (kType == kFp32) {
    float m = neg_inf();
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      m = max_nan(m, max_nan(max_nan(__uint_as_float(q[k].x), __uint_as_float(q[k].y)), max_nan(__uint_as_float(q[k].z), __uint_as_float(q[k].w))));
    return m;
  } else {
    using P = Pair<kType>;
    typename P::T m = P::of(kNegInf2<kType>);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(P::of(q[k].x), P::of(q[k].y)), __hmax2_nan(P::of(q[k].z), P::of(q[k].w))));
    const float2 f = unpack2(P::bits(m), kType == kFp16);
    return max_nan(f.x, f.y);
  }
}

// How the elements of a row lie: up to a 16-byte boundary single ones, then whole pieces, then single ones again.
template <int kType>
struct RowShape {
  static constexpr int kE = kElemsPer16<kType>;
  int head, pieces, tail;
  __device__ __forceinline__ RowShape(const uint8_t* p, int n) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / kElemBytes<kType>;
    head = min((kE - off) % kE, n);
    pieces = (n - head) / kE;
    tail = n - head - pieces * kE;
  }
};

// u_j = x_j c - m c, with m c rounded once and the same for all of a row: one fused operation, whose rounding of m c cancels in every quotient. That
// holds where raised elements vanish and where m c is at most 2^20: the largest element's u is what the rounding left out, here at most 2^-5, but 256 at
// 2^33, and 2^256 is no number. Elsewhere (rows of the type's lowest value, large logits, an extreme temperature) u_j = (x_j - m) c.
// Products are rounded where they are taken (__fmul_rn): one that the compiler drew into a following subtraction would be another number.
constexpr float kMostMc = 1048576.f;
template <int kType>
__device__ __forceinline__ bool fused_ok(float mc, float c) {
  const float low = __fmul_rn(kFloor<kType>, c), least = low > -1e38f ? fmaxf(low + 200.f, -kMostMc) : kMostMc;
  return mc > least && mc < kMostMc;
}
// The exponents are relative to m c, rounded where they come from the fused operation and exact elsewhere: m c and what its rounding left out of it. Sums under several
// maxima meet by the difference of both: without the second, fp32 logits around 1e6 would be a hundredth off.
template <int kType>
__device__ __forceinline__ float rest_of(float m, float mc, float c) { return fused_ok<kType>(mc, c) ? 0.f : fmaf(m, c, -mc); }

struct RowStats {
  float m, s, q;
};
// the same sums relative to a larger m
template <int kType>
__device__ __forceinline__ void rescale(RowStats& a, float m, float c) {
  const float from = __fmul_rn(a.m, c), to = __fmul_rn(m, c), d = (from - to) + (rest_of<kType>(a.m, from, c) - rest_of<kType>(m, to, c));
  const float u = a.m == m ? 0.f : fmaxf(d, kFloorU), f = exp2_fast(u);
  a.q = fmaf(a.s, u, a.q) * f;
  a.s *= f;
  a.m = m;
}
template <int kType, int kLanes>
__device__ __forceinline__ void reduce_lanes(RowStats& a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  rescale<kType>(a, m, c);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o /= 2) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.q += __shfl_xor_sync(0xffffffffu, a.q, o);
  }
}

// running statistics of one thread; with kTop also the place of the turn that holds its largest element, and the largest of the other turns
template <int kType, bool kTop>
struct Running {
  float m = neg_inf(), mc = neg_inf(), rest = 0.f, second = neg_inf();
  int at = 0;
  f32x2 s = 0, q = 0;
  __device__ __forceinline__ void turn(float largest, int v, float c) {
    if constexpr (kTop) {
      second = max_nan(second, fminf(m, largest));   // NaN stands above all
      if (largest > m || largest != largest) at = v;
    }
    raise(largest, c);
  }
  __device__ __forceinline__ void raise(float to, float c) {   // before elements up to `to`
    if (to <= m) return;
    m = max_nan(m, to);
    const float next = __fmul_rn(m, c), next_rest = rest_of<kType>(m, next, c);
    const float d = fmaxf((mc - next) + (rest - next_rest), kFloorU), f = exp2_fast(d);   // NaN, from infinite products: the floor
    q = mul2(fma2(s, bc2(d), q), bc2(f));
    s = mul2(s, bc2(f));
    mc = next;
    rest = next_rest;
  }
  __device__ __forceinline__ void add(f32x2 u) {
    float u0, u1;
    upk2(u, u0, u1);
    const f32x2 e = pk2(exp2_fast(u0), exp2_fast(u1));
    s = add2(s, e);
    q = fma2(e, u, q);
  }
  __device__ __forceinline__ void piece(const uint4& v, float c, bool fused) {
    constexpr int kE = kElemsPer16<kType>;
    float f[kE];
    if (fused) {
      unpack16<kType>(raised<kType>(v), f);
#pragma unroll
      for (int i = 0; i < kE; i += 2) add(fma2(pk2(f[i], f[i + 1]), bc2(c), bc2(-mc)));
    } else {
      unpack16<kType>(v, f);
#pragma unroll
      for (int i = 0; i < kE; i += 2) add(pk2(fmaxf((f[i] - m) * c, kFloorU), fmaxf((f[i + 1] - m) * c, kFloorU)));
    }
  }
  __device__ __forceinline__ RowStats done() const {
    float a, b, x, y;
    upk2(s, a, b);
    upk2(q, x, y);
    return {m, a + b, x + y};
  }
};
template <int kThreads>
constexpr int kListLen = kThreads == 32 ? 256 : 1024;
template <int kThreads>
struct RowShared {
  RowStats part[kThreads / 32];
  RowStats all;
  __align__(16) uint32_t group[kThreads < 128 ? kThreads : 128];   // largest element of a group of threads
  uint64_t top[CCF_LOGPROBS_MAX_TOP];
  uint64_t best[kThreads / 32];
  uint64_t list[kListLen<kThreads>];
  int listed;
};
template <int kThreads>
struct RowSharedPlain {   // without alternatives
  RowStats part[kThreads / 32];
  RowStats all;
};

template <int kThreads>
__device__ __forceinline__ void row_sync() {
  if constexpr (kThreads == 32) __syncwarp();
  else __syncthreads();
}

// sh.list[0, n) by rank into sh.top, the k largest
template <int kStep, typename Shared>
__device__ __forceinline__ void rank_list(Shared& sh, int n, int k, int first) {
  for (int i = first; i < n; i += kStep) {
    const uint64_t key = sh.list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sh.list[j] > key;
    if (key != 0 && rank < k) sh.top[rank] = key;
  }
}

// Groups whose largest elements bound the k-th largest: more than k of them keep the bound tight.
template <int kThreads>
__device__ __forceinline__ int log_group(int k) {   // log2 of the threads in a group
  constexpr int kLog = kThreads == 32 ? 5 : kThreads == 128 ? 7 : 8;
  return max(0, min(min(5, kLog - 2), kLog - 1 - (32 - __clz(k))));
}

// Before the row's first barrier: what select_top starts from.
template <int kThreads>
__device__ __forceinline__ uint32_t group_maxima(RowShared<kThreads>& sh, float m, int tid, int k) {
  const uint32_t mine = m == neg_inf() ? 0u : order_of(m);
  const int log = log_group<kThreads>(k);
  uint32_t g = mine;
  for (int o = 1 << log >> 1; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if ((tid & ((1 << log) - 1)) == 0) sh.group[tid >> log] = g;
  if (tid == 0) sh.listed = 0;
  if (tid < CCF_LOGPROBS_MAX_TOP) sh.top[tid] = 0;
  return mine;
}

// The k largest elements of this block's share of a row, in order, into sh.top. The largest elements of groups of threads are elements themselves: the k-th
// largest of those bounds the k-th largest element from below. Only threads whose own largest element reaches the bound look at elements again (a few more than
// k), for most of them those of the one turn that held it, an element a lane; and only elements that reach the bound are listed. Should they
// not fit the list (many equal elements), they are taken one after the other instead, each the largest below the one before: 4 rows of 50257 with five columns above
// the type's lowest value and twenty alternatives 113 us, not 10.
template <int kType, int kThreads>
__device__ __forceinline__ void select_top(RowShared<kThreads>& sh, const uint8_t* p, const RowShape<kType>& shape, int first, int last,
                                           const Running<kType, true>& run, uint32_t largest, float edge, int edge_index, int k) {
  constexpr int kE = kElemsPer16<kType>;
  const int tid = kThreads == 32 ? lane_id() : threadIdx.x, lane = lane_id();
  const uint4* pieces = reinterpret_cast<const uint4*>(p + shape.head * kElemBytes<kType>);
  const int groups = kThreads >> log_group<kThreads>(k);
  uint32_t bound = 0;   // every warp finds it by itself: cheaper than a barrier
  for (int j = lane; j < groups; j += 32) {
    const uint32_t g = sh.group[j];
    int above = 0, from = 0;
#pragma unroll 2
    for (int i = 0; i < groups; i += 4) {   // at least four groups
      const uint4 o = *reinterpret_cast<const uint4*>(sh.group + i);
      above += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
      from += (o.x >= g) + (o.y >= g) + (o.z >= g) + (o.w >= g);
    }
    if (above < k && k <= from) bound = g;   // the k-th largest
  }
  bound = max(1u, __reduce_max_sync(0xffffffffu, bound));   // fewer elements than that: every finite one counts
  auto list = [&](float v, int index) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < kListLen<kThreads>) sh.list[at] = top_key(v, index);
  };
  auto consider = [&](float v, int index) {
    if (v != neg_inf() && order_of(v) >= bound) list(v, index);
  };
  if (edge_index >= 0) consider(edge, edge_index);
  uint32_t wide = __ballot_sync(0xffffffffu, run.second != neg_inf() && order_of(run.second) >= bound);
  uint32_t owners = __ballot_sync(0xffffffffu, largest >= bound) & ~wide;
  while (owners != 0) {   // four of them at a time, so that their elements come together
    float f[4];
    int index[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int owner = __ffs(owners) - 1;
      const int v = __shfl_sync(0xffffffffu, run.at, owner & 31) + lane / kE * kThreads;
      index[u] = shape.head + v * kE + lane % kE;
      f[u] = owner >= 0 && lane < kUnroll * kE && v < last ? load_elem<kType>(p, index[u]) : neg_inf();
      owners &= owners - 1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) consider(f[u], index[u]);
  }
  for (; wide != 0; wide &= wide - 1) {
    for (int v = first + tid - lane + __ffs(wide) - 1 + lane * kThreads; v < last; v += 32 * kThreads) {
      float f[kE];
      unpack16<kType>(__ldg(pieces + v), f);
#pragma unroll
      for (int i = 0; i < kE; ++i) consider(f[i], shape.head + v * kE + i);
    }
  }
  row_sync<kThreads>();
  const int n = sh.listed;
  if (n <= kListLen<kThreads>) {   // the first warp's work, and what is written from it too
    if (tid < 32) rank_list<32>(sh, n, k, lane);
    __syncwarp();
    return;
  }
  uint64_t below = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    auto look = [&](float v, int index) {
      const uint64_t key = v == neg_inf() ? 0 : top_key(v, index);
      if (key < below && key > best) best = key;
    };
    for (int v = first + tid; v < last; v += kThreads) {
      float f[kE];
      unpack16<kType>(__ldg(pieces + v), f);
#pragma unroll
      for (int i = 0; i < kE; ++i) look(f[i], shape.head + v * kE + i);
    }
    if (edge_index >= 0) look(edge, edge_index);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if constexpr (kThreads > 32) {
      if (lane == 0) sh.best[threadIdx.x >> 5] = best;
      __syncthreads();
#pragma unroll 1
      for (int w = 0; w < kThreads / 32; ++w) best = sh.best[w] > best ? sh.best[w] : best;
      __syncthreads();
    }
    if (tid == 0) sh.top[r] = best;
    if (best == 0) break;
    below = best;
  }
  row_sync<kThreads>();
}

// kThreads per row; a warp per row, eight rows a block, where rows are short. Rows of wide vocabularies may be shared by a cluster of 2^log_split blocks,
// each with its part of the columns, whose statistics and alternatives the first one joins: a few rows would leave most of the card idle.
// 8192 rows of 50257 bf16 133 us (6.2 TB/s), 4099 with five alternatives 84 (4.9 TB/s: choosing them takes a quarter more instructions), 4 rows with twenty 10.
// Bound by the memory in the first, by the arithmetic's latency in the second (55 % of the issue slots). Rows by bulk copies into shared memory, over the ends
// of rows, took 167 to 230 us: what their buffers leave room for is too few warps.
template <int kType, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : kThreads) logprobs_fwd_kernel(const __grid_constant__ CcfLogprobs a, int log_split) {
  namespace cg = cooperative_groups;
  constexpr int kE = kElemsPer16<kType>, kRows = kThreads == 32 ? 8 : 1;
  using Shared = typename std::conditional<kTop, RowShared<kThreads>, RowSharedPlain<kThreads>>::type;
  __shared__ Shared shared[kRows];
  const int warp = threadIdx.x >> 5, lane = lane_id(), tid = kThreads == 32 ? lane : threadIdx.x;
  const int split = 1 << log_split, rank = static_cast<int>(blockIdx.x) & (split - 1);
  const long long row = kThreads == 32 ? blockIdx.x * 8ll + warp : static_cast<long long>(blockIdx.x >> log_split);
  if (kThreads == 32 && row >= a.rows) return;
  Shared& sh = shared[kThreads == 32 ? warp : 0];
  const uint8_t* p = reinterpret_cast<const uint8_t*>(a.x) + static_cast<size_t>(row) * a.ld * kElemBytes<kType>;
  const RowShape<kType> shape(p, a.vocab);
  const int first = static_cast<int>(static_cast<unsigned>(shape.pieces) * rank >> log_split);   // at most 2^28 pieces and 4 blocks
  const int last = static_cast<int>(static_cast<unsigned>(shape.pieces) * (rank + 1) >> log_split);
  const uint4* pieces = reinterpret_cast<const uint4*>(p + shape.head * kElemBytes<kType>);
  const float c = a.inv_t * kLog2e;
  long long target = 0;
  float logit = 0.f;
  if (rank == 0 && tid == 0) {
    target = load_index(a.targets, row, a.wide);
    if (target >= 0 && target < a.vocab) logit = load_elem<kType>(p, target);
  }
  // single elements in front of and behind the whole pieces: one for each of the first threads
  int edge_index = -1;
  if (rank == 0 && tid < shape.head) edge_index = tid;
  if (rank == split - 1 && tid >= shape.head && tid < shape.head + shape.tail) edge_index = tid + shape.pieces * kE;
  const float edge = edge_index >= 0 ? load_elem<kType>(p, edge_index) : neg_inf();
  Running<kType, kTop> run;
  int v = first + tid;
  auto turn = [&](const uint4(&q)[kUnroll]) {
    run.turn(max_of<kType>(q), v, c);
    const bool fused = fused_ok<kType>(run.mc, c);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) run.piece(q[u], c, fused);
  };
  for (; v + (kUnroll - 1) * kThreads < last; v += kUnroll * kThreads) {
    uint4 q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = load16_once(pieces + v + u * kThreads);
    turn(q);
  }
  if (v < last) {
    uint4 q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      q[u] = make_uint4(kNegInf2<kType>, kNegInf2<kType>, kNegInf2<kType>, kNegInf2<kType>);
      if (v + u * kThreads < last) q[u] = load16_once(pieces + v + u * kThreads);
    }
    turn(q);
  }
  // of the whole pieces; a single element is taken as it is
  const float own = run.m;
  run.raise(edge, c);
  run.add(pk2(fmaxf(fused_ok<kType>(run.mc, c) ? fmaf(edge, c, -run.mc) : (edge - run.m) * c, kFloorU), kFloorU));
  RowStats st = run.done();
  uint32_t largest = 0;
  if constexpr (kTop) largest = group_maxima<kThreads>(sh, own, tid, a.top_k);
  reduce_lanes<kType, 32>(st, c);
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    if (lane == 0) sh.part[warp] = st;
    __syncthreads();
    st = sh.part[lane % kWarps];
    reduce_lanes<kType, kWarps>(st, c);
  } else {
    __syncwarp();
  }
  if constexpr (kTop) select_top<kType, kThreads>(sh, p, shape, first, last, run, largest, edge, edge_index, a.top_k);
  if constexpr (kThreads > 32) {
    if (split > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (tid == 0) sh.all = st;
      cluster.sync();
      if (rank == 0) {
        st = RowStats{neg_inf(), 0.f, 0.f};
        if (lane < split) st = *cluster.map_shared_rank(&sh.all, lane);
        reduce_lanes<kType, 32>(st, c);
        if constexpr (kTop) {
          const int n = split * a.top_k;
          for (int i = tid; i < n; i += kThreads) sh.list[i] = cluster.map_shared_rank(sh.top, i / a.top_k)[i % a.top_k];
          __syncthreads();
          if (tid < CCF_LOGPROBS_MAX_TOP) sh.top[tid] = 0;
          __syncthreads();
          rank_list<kThreads>(sh, n, a.top_k, tid);
          __syncthreads();
        }
      }
      cluster.sync();   // nobody leaves while its shared memory is read
      if (rank != 0) return;
    }
    if (tid >= 32) return;   // the first warp has what is left
  }
  const float log_s = logf(st.s), mc = __fmul_rn(st.m, c);
  // lp_j = (x_j - M) / T - log_sum: the sum stands relative to the rounded M c, so the rounding is taken out of it
  const float log_sum = fused_ok<kType>(mc, c) ? fmaf(-kLn2, fmaf(st.m, c, -mc), log_s) : log_s;
  const bool none = st.m == neg_inf(), bad = !(st.m < __int_as_float(0x7f800000));
  const float nan = __int_as_float(0x7fc00000);
  if (tid == 0) {
    const float h = bad ? nan : none ? 0.f : fmaf(-kLn2, st.q / st.s, log_s);
    float lp = bad ? nan : none ? neg_inf() : (logit - st.m) * a.inv_t - log_sum;
    if (target == a.ignore) {
      lp = 0.f;
    } else if (target < 0 || target >= a.vocab) {
      report_index(a.status, static_cast<uint32_t>(row));
      lp = nan;
    }
    a.logprobs[row] = lp;
    a.entropy[row] = h;
    if (a.stats != nullptr) {
      a.stats[row * 3] = st.m;
      a.stats[row * 3 + 1] = st.s;
      a.stats[row * 3 + 2] = h;
    }
  }
  if constexpr (kTop) {
    if (tid < a.top_k) {
      const uint64_t key = sh.top[tid];
      const float v = value_of(static_cast<uint32_t>(key >> 32));
      a.top_ids[row * a.top_k + tid] = key != 0 ? static_cast<long long>(0xffffffffu - static_cast<uint32_t>(key)) : -1ll;
      a.top_logprobs[row * a.top_k + tid] = key == 0 ? neg_inf() : bad ? nan : (v - st.m) * a.inv_t - log_sum;
    }
  }
}

// The coefficients of a row: dx_j = hot_j - 2^u_j (w0 + w1 u_j).
struct RowGrad {
  float m, w0, w1, g;
  bool zero;
};
template <int kType>
__device__ __forceinline__ RowGrad row_grad(const CcfLogprobs& a, long long row, long long target) {
  RowGrad r;
  const float s = a.stats[row * 3 + 1], h = a.stats[row * 3 + 2];
  r.m = a.stats[row * 3];
  r.g = a.d_logprobs != nullptr && target != a.ignore && target >= 0 && target < a.vocab ? a.d_logprobs[row] : 0.f;
  const float gh = a.d_entropy != nullptr ? a.d_entropy[row] : 0.f;
  float all = r.g;
  bool any = r.g != 0.f || gh != 0.f;
  if (a.d_top != nullptr) {
    for (int k = 0; k < a.top_k; ++k) {
      if (a.top_ids[row * a.top_k + k] < 0) continue;
      const float gk = a.d_top[row * a.top_k + k];
      all += gk;
      any = any || gk != 0.f;
    }
  }
  r.zero = !any || r.m == neg_inf();
  const float scale = a.inv_t / s;
  r.w0 = scale * fmaf(gh, h - logf(s), all);
  r.w1 = scale * gh * kLn2;
  if (!(r.m < __int_as_float(0x7f800000))) r.w0 = __int_as_float(0x7fc00000);
  return r;
}

// kThreads per row and part of its columns (blockIdx.y of gridDim.y), a warp per row where rows are short. Bound by reading the logits and writing
// the gradient once: 8192 rows of 50304 bf16 258 us, 6.4 TB/s.
template <int kType, int kThreads>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : kThreads) logprobs_bwd_kernel(const __grid_constant__ CcfLogprobs a) {
  constexpr int kE = kElemsPer16<kType>;
  const int warp = threadIdx.x >> 5, tid = kThreads == 32 ? lane_id() : threadIdx.x;
  const long long row = kThreads == 32 ? blockIdx.x * 8ll + warp : static_cast<long long>(blockIdx.x);
  if (kThreads == 32 && row >= a.rows) return;
  const int split = static_cast<int>(gridDim.y), rank = static_cast<int>(blockIdx.y);
  const uint8_t* p = reinterpret_cast<const uint8_t*>(a.x) + static_cast<size_t>(row) * a.ld * kElemBytes<kType>;
  uint8_t* o = reinterpret_cast<uint8_t*>(a.dx) + static_cast<size_t>(row) * a.dx_ld * kElemBytes<kType>;
  const RowShape<kType> shape(p, a.width);
  const int first = static_cast<int>(static_cast<long long>(shape.pieces) * rank / split);
  const int last = static_cast<int>(static_cast<long long>(shape.pieces) * (rank + 1) / split);
  const uint4* pieces = reinterpret_cast<const uint4*>(p + shape.head * kElemBytes<kType>);
  uint4* out = reinterpret_cast<uint4*>(o + shape.head * kElemBytes<kType>);
  const long long target = load_index(a.targets, row, a.wide);
  const RowGrad r = row_grad<kType>(a, row, target);
  const float c = a.inv_t * kLog2e;
  int edge_index = -1;
  if (rank == 0 && tid < shape.head) edge_index = tid;
  if (rank == split - 1 && tid >= shape.head && tid < shape.head + shape.tail) edge_index = tid + shape.pieces * kE;
  if (r.zero) {
    for (int v = first + tid; v < last; v += kThreads) out[v] = make_uint4(0, 0, 0, 0);
    if (edge_index >= 0) store_elem<kType>(o, edge_index, 0.f);
    return;
  }
  const float mc = __fmul_rn(r.m, c);
  const bool fused = fused_ok<kType>(mc, c);
  auto grad = [&](float x) {
    const float u = fmaxf(fused ? fmaf(x, c, -mc) : (x - r.m) * c, kFloorU);
    return -exp2_fast(u) * fmaf(r.w1, u, r.w0);
  };
  const int full = (a.vocab - shape.head) / kE;   // pieces that lie in the vocabulary as a whole (may be negative: none)
  for (int v0 = first + tid; v0 < last; v0 += kUnroll * kThreads) {
    uint4 q[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = v0 + k * kThreads;
      q[k] = make_uint4(0, 0, 0, 0);
      if (v < last && shape.head + v * kE < a.vocab) q[k] = load16_once(pieces + v);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = v0 + k * kThreads;
      if (v >= last) break;
      float f[kE];
      if (fused) {
        unpack16<kType>(raised<kType>(q[k]), f);
#pragma unroll
        for (int i = 0; i < kE; i += 2) {
          const f32x2 u = fma2(pk2(f[i], f[i + 1]), bc2(c), bc2(-mc));
          float u0, u1;
          upk2(u, u0, u1);
          upk2(mul2(pk2(exp2_fast(u0), exp2_fast(u1)), fma2(bc2(-r.w1), u, bc2(-r.w0))), f[i], f[i + 1]);
        }
      } else {
        unpack16<kType>(q[k], f);
#pragma unroll
        for (int i = 0; i < kE; ++i) f[i] = grad(f[i]);
      }
      if (v >= full) {
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (shape.head + v * kE + i >= a.vocab) f[i] = 0.f;
      }
      out[v] = pack16<kType>(f);
    }
  }
  if (edge_index >= 0) store_elem<kType>(o, edge_index, edge_index < a.vocab ? grad(load_elem<kType>(p, edge_index)) : 0.f);
  // the target's and the alternatives' own terms, by rewriting those elements
  row_sync<kThreads>();
  const int begin = rank == 0 ? 0 : shape.head + first * kE, end = rank == split - 1 ? a.width : shape.head + last * kE;
  const int tops = a.d_top != nullptr ? a.top_k : 0;
  for (int i = tid; i <= tops; i += kThreads) {
    const long long j = i == 0 ? target : a.top_ids[row * a.top_k + i - 1];
    if (j < begin || j >= end || j >= a.vocab) continue;
    float g = i == 0 ? r.g : a.d_top[row * a.top_k + i - 1];
    bool twice = false;   // the target is an alternative as well: that one writes for both
    if (i == 0)
      for (int k = 0; k < tops; ++k) twice = twice || a.top_ids[row * a.top_k + k] == target;
    else if (j == target)
      g += r.g;
    if (!twice) store_elem<kType>(o, j, fmaf(a.inv_t, g, grad(load_elem<kType>(p, j))));
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
static bool valid(const CcfLogprobs* a) {
  return a != nullptr && a->x != nullptr && a->targets != nullptr && a->rows >= 1 && a->rows <= 0x0fffffffll && a->vocab >= 1 && a->vocab <= (1 << 30) &&
         a->width >= a->vocab && a->width <= (1 << 30) && (a->ld >= a->width || a->rows == 1) && a->top_k >= 0 && a->top_k <= CCF_LOGPROBS_MAX_TOP &&
         a->top_k <= a->vocab && a->type >= 0 && a->type <= 2 && (reinterpret_cast<uintptr_t>(a->x) & 15) == 0 && a->inv_t > 0.f;
}

template <int kType, int kThreads, bool kTop>
static int launch_fwd(const CcfLogprobs& a, int log_split, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  const int split = 1 << log_split;
  cfg.gridDim = dim3(kThreads == 32 ? static_cast<unsigned>((a.rows + 7) / 8) : static_cast<unsigned>(a.rows * split));
  cfg.blockDim = dim3(kThreads == 32 ? 256 : kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<kType, kThreads, kTop>, a, log_split);
  return e == cudaSuccess ? 0 : -static_cast<int>(e);
}

template <int kType, bool kTop>
static int choose_fwd(const CcfLogprobs& a, cudaStream_t st) {
  // us, 0 and 5 alternatives. A warp a row against more threads: 8192 x 1000 12 and 16 / 18 and 35, 4096 x 4000 14 and 18 / 14 and 21, 300 x 4000
  // 12 / 7. 128 threads against 256: 8192 x 50257 131 / 144, 2000 x 2000 8 / 12, 300 x 20000 10 / 8, 1000 x 20000 equal. Four blocks a row against one:
  // 64 x 50257 8 and 10 / 12 and 14; eight: 4 x 50257 with 20 alternatives 10 / 12.
  const bool many = a.rows >= 4 * sm_count();
  if (a.vocab <= 1024 || (many && a.vocab <= 4096)) return launch_fwd<kType, 32, kTop>(a, 0, st);
  if (many) return launch_fwd<kType, 128, kTop>(a, 0, st);
  int log_split = 0;
  while (log_split < 2 && a.rows << log_split < 2 * sm_count() && a.vocab >> log_split > 8192) ++log_split;
  return launch_fwd<kType, 256, kTop>(a, log_split, st);
}

template <int kType>
static int choose_bwd(const CcfLogprobs& a, cudaStream_t st) {
  const unsigned rows = static_cast<unsigned>(a.rows);
  // us, a warp a row against 256 threads: 8192 x 1000 10 / 29, 2000 x 2000 7.6 / 10.3, 300 x 1000 5.4 / 4.4, 16 x 4000 8 / 4
  if (a.width <= 1024 || (a.width <= 2048 && a.rows >= 4 * sm_count())) {
    logprobs_bwd_kernel<kType, 32><<<(rows + 7) / 8, 256, 0, st>>>(a);
  } else {
    int split = 1;   // of a row's columns. 64 x 50257 6 us, unsplit 12; with half or twice the blocks 1025 x 30522 takes 28.7 instead of 26.7
    const int pieces = a.width / kElemsPer16<kType>;
    while (split < 64 && a.rows * split < 8 * sm_count() && pieces / split > 256 * kUnroll) split *= 2;
    logprobs_bwd_kernel<kType, 256><<<dim3(rows, split), 256, 0, st>>>(a);
  }
  return launch_result();
}

}  // namespace ccf

extern "C" {

int ccf_sizeof_logprobs() { return static_cast<int>(sizeof(CcfLogprobs)); }

// logprobs, entropy [rows] and, for top_k > 0, top_logprobs and top_ids [rows, top_k]. A row without a finite logit: log probability -inf, entropy 0.
// A row with NaN or +inf: NaN. An ignored target: 0. A target outside the vocabulary: NaN, and recorded in `status` (code 5, the row).
// Alternatives: by value, equal ones by index; where no logit above -inf is left: id -1, -inf. x on a 16-byte boundary; its rows may begin anywhere.
int ccf_logprobs_fwd(const CcfLogprobs* a, void* stream) {
  using namespace ccf;
  if (!valid(a) || a->logprobs == nullptr || a->entropy == nullptr || (a->top_k > 0 && (a->top_ids == nullptr || a->top_logprobs == nullptr))) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool top = a->top_k > 0;
  if (a->type == kBf16) return top ? choose_fwd<kBf16, true>(*a, st) : choose_fwd<kBf16, false>(*a, st);
  if (a->type == kFp16) return top ? choose_fwd<kFp16, true>(*a, st) : choose_fwd<kFp16, false>(*a, st);
  return top ? choose_fwd<kFp32, true>(*a, st) : choose_fwd<kFp32, false>(*a, st);
}

// dx [rows, width], `dx_ld` elements between rows, from the gradients of the outputs that are given: zeros behind the vocabulary and in rows without a gradient.
int ccf_logprobs_bwd(const CcfLogprobs* a, void* stream) {
  using namespace ccf;
  if (!valid(a) || a->dx == nullptr || (reinterpret_cast<uintptr_t>(a->dx) & 15) != 0 || a->stats == nullptr ||
      (a->d_top != nullptr && (a->top_k == 0 || a->top_ids == nullptr)))
    return -2;
  if (a->rows > 1 && (a->dx_ld < a->width || (a->dx_ld - a->ld) % (a->type == kFp32 ? 4 : 8) != 0)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->type == kBf16) return choose_bwd<kBf16>(*a, st);
  if (a->type == kFp16) return choose_bwd<kFp16>(*a, st);
  return choose_bwd<kFp32>(*a, st);
}

}  // extern "C"
