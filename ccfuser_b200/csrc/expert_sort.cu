// Tokens sorted by expert and back: rows[row(t, j)] = x[t], and y[t] = sum_j w[t, j] rows[row(t, j)], with the gradients of both. The layer's own
// kernels (dispatch.cuh, combine.cu) do this inside their GEMMs; these are for experts that are not the layer's.
//
// The order is routing.py's: a slot's position is the number of earlier slots of the same expert, slots from `capacity` on are dropped, an expert
// outside [0, experts) is none. Every expert's rows begin at a multiple of `align`. Nothing depends on the order in which blocks run: no atomics
// on positions or sums.
#include "elements.cuh"
#include "expert_sort.h"

namespace ccf {

// ---- order -----------------------------------------------------------------------------------------------------------
// Bound by latency: a few bytes a slot. Up to kOrderTile slots one block does it all. Above, each block counts its slots' experts in a first kernel, and in
// the second adds up the counts of the blocks in front of it; both keep a slot's place in registers.
constexpr int kOrderThreads = 1024;
constexpr int kOrderBlocks = 32;                  // as many as a block reads the counts of
constexpr int kOrderMost = 8;                     // slots of a thread at a time

struct OrderShape {
  int threads, per, tiles, blocks;   // slots of a block: threads * per * tiles
};

inline OrderShape order_shape(long long slots, int experts) {
  OrderShape s;
  const int least = (experts + 31) / 32 * 32;      // one thread per expert
  const long long want = (slots + 31) / 32 * 32;
  s.threads = want > kOrderThreads ? kOrderThreads : static_cast<int>(want);
  if (s.threads < least) s.threads = least;
  s.per = 1;
  while (s.per < kOrderMost && static_cast<long long>(s.threads) * s.per * kOrderBlocks < slots) s.per *= 2;
  const long long tile = static_cast<long long>(s.threads) * s.per;
  const long long all = (slots + tile - 1) / tile;
  s.tiles = static_cast<int>((all + kOrderBlocks - 1) / kOrderBlocks);
  s.blocks = static_cast<int>((all + s.tiles - 1) / s.tiles);
  return s;
}

// slots of each expert in front of this one: of the same lane's earlier slots and of lower lanes, by warp; counts per warp are left in `mine`
template <int kPer>
__device__ __forceinline__ void rank_slots(const CcfOrder& o, long long first, int* mine, int (&e)[kPer], int (&r)[kPer]) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < o.experts; i += 32) mine[i] = 0;
#pragma unroll
  for (int l = 0; l < kPer; ++l) {
    const long long s = first + 32 * l + lane;
    const long long v = s < o.slots ? load_index(o.idx, s, o.wide) : -1;
    e[l] = v >= 0 && v < o.experts ? static_cast<int>(v) : -1;
  }
  __syncwarp();
#pragma unroll
  for (int l = 0; l < kPer; ++l) {
    const unsigned same = __match_any_sync(0xffffffffu, e[l]);
    const int below = __popc(same & ((1u << lane) - 1u));
    const int before = e[l] >= 0 ? mine[e[l]] : 0;
    __syncwarp();
    if (e[l] >= 0 && below == 0) mine[e[l]] = before + __popc(same);
    __syncwarp();
    r[l] = before + below;
  }
}

// counts[block][expert]
__global__ void __launch_bounds__(kOrderThreads) order_count_kernel(const __grid_constant__ CcfOrder o, long long chunk) {
  extern __shared__ int sum[];
  for (int e = threadIdx.x; e < o.experts; e += blockDim.x) sum[e] = 0;
  __syncthreads();
  const long long begin = blockIdx.x * chunk;
  for (long long at = 0; at < chunk; at += blockDim.x) {
    const long long s = begin + at + threadIdx.x;
    const long long v = s < o.slots ? load_index(o.idx, s, o.wide) : -1;
    const int e = v >= 0 && v < o.experts ? static_cast<int>(v) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && (same & ((1u << (threadIdx.x & 31)) - 1u)) == 0) atomicAdd(&sum[e], __popc(same));
  }
  __syncthreads();
  let_next_in();
  int* out = static_cast<int*>(o.scratch) + static_cast<long long>(blockIdx.x) * o.experts;
  for (int e = threadIdx.x; e < o.experts; e += blockDim.x) out[e] = sum[e];
}

// shared memory: [warps][experts] counts of the warps, then total, before, base and kept of each expert
template <int kPer>
__global__ void __launch_bounds__(kOrderThreads) order_place_kernel(const __grid_constant__ CcfOrder o, int tiles) {
  extern __shared__ int shared[];
  __shared__ int part[32];
  const int E = o.experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  int* const by_warp = shared;
  int* const total = shared + warps * E;
  int* const before = total + E;
  int* const base = before + E;        // E + 1
  int* const kept = base + E + 1;
  const long long chunk = static_cast<long long>(blockDim.x) * kPer * tiles, begin = blockIdx.x * chunk;
  int e[kPer], r[kPer];
  rank_slots<kPer>(o, begin + static_cast<long long>(warp) * 32 * kPer, by_warp + warp * E, e, r);
  if (tid < E) total[tid] = before[tid] = 0;
  __syncthreads();
  if (gridDim.x > 1) {
    wait_for_previous();
    const int* const counts = behind(static_cast<const int*>(o.scratch));
    const int blocks = static_cast<int>(gridDim.x);
    for (int i = tid; i < blocks * E; i += blockDim.x) {
      const int v = counts[i];
      if (v == 0) continue;
      const int x = i % E;
      atomicAdd(&total[x], v);
      if (i < static_cast<int>(blockIdx.x) * E) atomicAdd(&before[x], v);
    }
  } else if (tid < E) {
    int run = 0;
    for (int w = 0; w < warps; ++w) run += by_warp[w * E + tid];
    total[tid] = run;
  }
  __syncthreads();
  let_next_in();
  // rows of each expert and where they begin: one thread per expert, sums by warps
  int rows = 0, sum = 0;
  if (tid < E) {
    rows = static_cast<int>(min(static_cast<long long>(total[tid]), o.capacity));
    sum = (rows + o.align - 1) / o.align * o.align;
  }
  int run = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += v;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  if (warp == 0) {
    int v = lane < warps ? part[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    part[lane] = v;
  }
  __syncthreads();
  if (tid < E) {
    base[tid] = run - sum + (warp > 0 ? part[warp - 1] : 0);
    kept[tid] = rows;
    if (tid == E - 1) base[E] = base[tid] + sum;
    if (blockIdx.x == 0) {
      o.counts[tid] = rows;
      o.base[tid] = base[tid];
      if (tid == E - 1) o.base[E] = base[E];
    }
  }
  for (int tile = 0; tile < tiles; ++tile) {
    const long long first = begin + (static_cast<long long>(tile) * blockDim.x + warp * 32) * kPer;
    if (tile > 0) {
      __syncthreads();
      rank_slots<kPer>(o, first, by_warp + warp * E, e, r);
    }
    __syncthreads();
    if (tid < E) {      // rows in front of each warp's
      int at = before[tid];
      for (int w = 0; w < warps; ++w) {
        const int c = by_warp[w * E + tid];
        by_warp[w * E + tid] = at;
        at += c;
      }
      before[tid] = at;
    }
    __syncthreads();
#pragma unroll
    for (int l = 0; l < kPer; ++l) {
      const long long s = first + 32 * l + lane;
      if (s >= o.slots) continue;
      int row = -1;
      if (e[l] >= 0) {
        const int pos = by_warp[warp * E + e[l]] + r[l];
        if (pos < kept[e[l]]) row = base[e[l]] + pos;
      }
      o.slot_row[s] = row;
      if (row >= 0) o.row_slot[row] = static_cast<int>(s);
    }
  }
  // rows without a slot: between experts, one warp each, and behind the last
  for (int x = blockIdx.x * warps + warp; x < E; x += gridDim.x * warps)
    for (int row = base[x] + kept[x] + lane; row < base[x + 1]; row += 32) o.row_slot[row] = -1;
  for (long long row = base[E] + static_cast<long long>(blockIdx.x) * blockDim.x + tid; row < o.rows; row += static_cast<long long>(gridDim.x) * blockDim.x)
    o.row_slot[row] = -1;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// Bound by memory: each token's row is read once and written to its slots' rows (or read from them). A warp is shared by as many tokens as fit
// (lanes of a token: a power of two); a token's row is cut into pieces of kUnits units per lane.
constexpr int kRowThreads = 256;

struct RowShape {
  long long items;      // pieces of all tokens
  int lanes_log, pieces, units;   // lanes of a token, pieces and units of a row
};

inline RowShape row_shape(long long tokens, int units, int per_lane) {
  RowShape s;
  s.units = units;
  s.lanes_log = 0;
  while (s.lanes_log < 5 && (1 << s.lanes_log) < (units + per_lane - 1) / per_lane) ++s.lanes_log;
  s.pieces = (units + per_lane * (1 << s.lanes_log) - 1) / (per_lane * (1 << s.lanes_log));
  s.items = tokens * s.pieces;
  return s;
}
inline unsigned row_blocks(const RowShape& s) {
  const long long warps = (s.items + (32 >> s.lanes_log) - 1) / (32 >> s.lanes_log);
  return static_cast<unsigned>((warps * 32 + kRowThreads - 1) / kRowThreads);
}

// Rows that no slot goes to are zeroed by all warps of the grid, each its share of them.
template <typename Unit>
__device__ __forceinline__ void zero_rows(const CcfRows& a, Unit* out, int units) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32), warp = static_cast<long long>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  const long long share = (a.rows + warps - 1) / warps, begin = warp * share, end = min(begin + share, a.rows);
  for (long long r0 = begin; r0 < end; r0 += 32) {
    unsigned none = __ballot_sync(0xffffffffu, r0 + lane < end && a.row_slot[r0 + lane] < 0);
    while (none != 0) {
      Unit* const row = out + (r0 + __ffs(none) - 1) * units;
      none &= none - 1;
      for (int c = lane; c < units; c += 32) row[c] = Unit{};
    }
  }
}

template <typename Unit>
__global__ void __launch_bounds__(kRowThreads) sort_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s, long long ld) {
  constexpr int kU = 4;
  const int lanes = 1 << s.lanes_log, lane = threadIdx.x & (lanes - 1);
  const long long item = (static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x) >> s.lanes_log;
  Unit* const out = static_cast<Unit*>(a.rows_out);
  Unit v[kU];
  const long long t = item / s.pieces;
  const int c0 = static_cast<int>(item - t * s.pieces) * kU * lanes + lane;
  const bool mine = item < s.items;
  if (mine) {
    const Unit* const x = static_cast<const Unit*>(a.tokens_in) + t * ld;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (c0 + u * lanes < s.units) v[u] = x[c0 + u * lanes];
  }
  wait_for_previous();
  const int* const slot_row = behind(a.slot_row);
  if (mine) {
    for (int j = 0; j < a.top_k; ++j) {
      const int row = slot_row[t * a.top_k + j];
      if (row < 0 || row >= a.rows) continue;
      Unit* const y = out + static_cast<long long>(row) * s.units;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (c0 + u * lanes < s.units) y[c0 + u * lanes] = v[u];
    }
  }
  zero_rows(a, out, s.units);
}

// kVec: 16-byte units, else single elements
template <int kType, bool kVec>
struct RowUnit {
  static constexpr int kElems = kVec ? kElemsPer16<kType> : 1;
  float f[kElems];
  __device__ __forceinline__ void load(const void* base, long long unit) {
    if constexpr (kVec) unpack16<kType>(__ldg(static_cast<const uint4*>(base) + unit), f);
    else f[0] = load_elem<kType>(base, unit);
  }
  __device__ __forceinline__ void store(void* base, long long unit) const {
    if constexpr (kVec) static_cast<uint4*>(base)[unit] = pack16<kType>(f);
    else store_elem<kType>(base, unit, f[0]);
  }
};

__device__ __forceinline__ float load_weight(const CcfRows& a, long long slot) {
  return a.weight_type == kFp32 ? load_elem<kFp32>(a.weights, slot) : a.weight_type == kFp16 ? load_elem<kFp16>(a.weights, slot) : load_elem<kBf16>(a.weights, slot);
}

template <int kType, bool kVec>
__global__ void __launch_bounds__(kRowThreads) return_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s) {
  constexpr int kU = 2, kJ = 2;
  using Row = RowUnit<kType, kVec>;
  const int lanes = 1 << s.lanes_log, lane = threadIdx.x & (lanes - 1);
  const long long item = (static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x) >> s.lanes_log;
  if (item >= s.items) return;
  const long long t = item / s.pieces;
  const int c0 = static_cast<int>(item - t * s.pieces) * kU * lanes + lane;
  Row sum[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u)
#pragma unroll
    for (int i = 0; i < Row::kElems; ++i) sum[u].f[i] = 0.f;
  for (int j0 = 0; j0 < a.top_k; j0 += kJ) {
    Row v[kJ][kU];
    float w[kJ];
    bool on[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const long long slot = t * a.top_k + j0 + j;
      const int row = j0 + j < a.top_k ? __ldg(a.slot_row + slot) : -1;
      on[j] = row >= 0 && row < a.rows;
      w[j] = on[j] && a.weights != nullptr ? load_weight(a, slot) : 1.f;
      if (!on[j]) continue;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (c0 + u * lanes < s.units) v[j][u].load(a.rows_in, static_cast<long long>(row) * s.units + c0 + u * lanes);
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      if (!on[j]) continue;
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int i = 0; i < Row::kElems; ++i) sum[u].f[i] = fmaf(w[j], v[j][u].f[i], sum[u].f[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (c0 + u * lanes < s.units) sum[u].store(a.tokens_out, t * s.units + c0 + u * lanes);
}

// `warps` of a block share a token; up to kK slots at a time
template <int kType, bool kVec, int kK>
__global__ void __launch_bounds__(kRowThreads) return_rows_bwd_kernel(const __grid_constant__ CcfRows a, int units, int warps, long long ld) {
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float part[kWarps][kK];
  using Row = RowUnit<kType, kVec>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % warps;
  const long long t = static_cast<long long>(blockIdx.x) * (kWarps / warps) + warp / warps;
  const bool mine = t < a.tokens;
  for (int j0 = 0; j0 < a.top_k; j0 += kK) {
    float dot[kK], w[kK];
    int row[kK];
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      const long long slot = t * a.top_k + j0 + j;
      row[j] = mine && j0 + j < a.top_k ? __ldg(a.slot_row + slot) : -1;
      if (row[j] >= a.rows) row[j] = -1;
      w[j] = row[j] >= 0 && a.weights != nullptr ? load_weight(a, slot) : 1.f;
      dot[j] = 0.f;
    }
    if (mine) {
      for (int c = sub * 32 + lane; c < units; c += 32 * warps) {
        Row dy, y[kK];
        dy.load(a.tokens_in, t * ld + c);
        if (a.d_weights != nullptr) {
#pragma unroll
          for (int j = 0; j < kK; ++j)
            if (row[j] >= 0) y[j].load(a.rows_in, static_cast<long long>(row[j]) * units + c);
        }
#pragma unroll
        for (int j = 0; j < kK; ++j) {
          if (row[j] < 0) continue;
          if (a.d_weights != nullptr) {
#pragma unroll
            for (int i = 0; i < Row::kElems; ++i) dot[j] = fmaf(dy.f[i], y[j].f[i], dot[j]);
          }
          if (a.rows_out != nullptr) {
            Row d;
#pragma unroll
            for (int i = 0; i < Row::kElems; ++i) d.f[i] = w[j] * dy.f[i];
            d.store(a.rows_out, static_cast<long long>(row[j]) * units + c);
          }
        }
      }
    }
    if (a.d_weights == nullptr) continue;
#pragma unroll
    for (int j = 0; j < kK; ++j) {
#pragma unroll
      for (int m = 16; m > 0; m /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
      if (lane == 0) part[warp][j] = dot[j];
    }
    __syncthreads();
    if (mine && sub == 0 && lane < kK && j0 + lane < a.top_k) {
      float sum = 0.f;
      for (int i = 0; i < warps; ++i) sum += part[warp + i][lane];
      const long long slot = t * a.top_k + j0 + lane;
      if (a.weight_type == kFp32) store_elem<kFp32>(a.d_weights, slot, sum);
      else if (a.weight_type == kFp16) store_elem<kFp16>(a.d_weights, slot, sum);
      else store_elem<kBf16>(a.d_weights, slot, sum);
    }
    __syncthreads();
  }
  if (a.rows_out != nullptr) {
    if constexpr (kVec) zero_rows(a, static_cast<uint4*>(a.rows_out), units);
    else if constexpr (kType == kFp32) zero_rows(a, static_cast<uint32_t*>(a.rows_out), units);
    else zero_rows(a, static_cast<uint16_t*>(a.rows_out), units);
  }
}

inline int elem_bytes(int type) { return type == kFp32 ? 4 : 2; }

inline bool rows_ok(const CcfRows& r) {
  return r.tokens >= 1 && r.rows >= 0 && r.rows <= 0x7fffffffLL && r.top_k >= 1 && r.tokens <= CCF_SORT_MAX_SLOTS && r.tokens * r.top_k <= CCF_SORT_MAX_SLOTS &&
         r.d >= 1 && r.d <= CCF_SORT_MAX_D && r.type >= 0 && r.type <= 2 && r.weight_type >= 0 && r.weight_type <= 2 && r.slot_row != nullptr;
}

// bytes of the largest unit (16 at most) that rows of d elements, `ld` apart, can be read in
inline int unit_bytes(const CcfRows& r, long long ld, const void* a, const void* b) {
  const unsigned long long size = elem_bytes(r.type);
  const unsigned long long bits = r.d * size | ld * size | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

template <typename Unit>
static int launch_sort(const CcfRows& r, int early, cudaStream_t st) {
  const int size = elem_bytes(r.type);
  const RowShape s = row_shape(r.tokens, static_cast<int>(static_cast<long long>(r.d) * size / sizeof(Unit)), 4);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_blocks(s));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr = early_attribute();
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, sort_rows_kernel<Unit>, r, s, static_cast<long long>(r.ld * size / sizeof(Unit)));
  return err == cudaSuccess ? 0 : -static_cast<int>(err);
}

template <int kType, bool kVec>
static int launch_return(const CcfRows& r, cudaStream_t st) {
  const RowShape s = row_shape(r.tokens, kVec ? r.d / kElemsPer16<kType> : r.d, 2);
  return_rows_kernel<kType, kVec><<<row_blocks(s), kRowThreads, 0, st>>>(r, s);
  return launch_result();
}

template <int kType, bool kVec>
static int launch_return_bwd(const CcfRows& r, cudaStream_t st) {
  const int units = kVec ? r.d / kElemsPer16<kType> : r.d;
  const long long ld = kVec ? r.ld / kElemsPer16<kType> : r.ld;
  int warps = 1;      // few tokens: several warps each
  while (warps < kRowThreads / 32 && warps * 32 < units && r.tokens * warps < 16LL * sm_count()) warps *= 2;
  const int tokens = kRowThreads / 32 / warps;
  const unsigned blocks = static_cast<unsigned>((r.tokens + tokens - 1) / tokens);
  const auto kern = r.top_k == 1   ? return_rows_bwd_kernel<kType, kVec, 1>
                    : r.top_k == 2 ? return_rows_bwd_kernel<kType, kVec, 2>
                    : r.top_k <= 4 ? return_rows_bwd_kernel<kType, kVec, 4>
                                   : return_rows_bwd_kernel<kType, kVec, 8>;
  kern<<<blocks, kRowThreads, 0, st>>>(r, units, warps, ld);
  return launch_result();
}

static size_t order_shared(const OrderShape& s, int experts) { return (static_cast<size_t>(s.threads / 32) * experts + 4 * experts + 1) * sizeof(int); }

template <int kPer>
static cudaError_t launch_place(const CcfOrder& o, const OrderShape& s, int early, cudaStream_t st) {
  const size_t shared = order_shared(s, o.experts);
  if (shared > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(order_place_kernel<kPer>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
    if (err != cudaSuccess) return err;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute attr = early_attribute();
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, order_place_kernel<kPer>, o, s.tiles);
}

inline int not_capturing(cudaStream_t st) { return early_launches(0, st); }

}  // namespace ccf

extern "C" {

int ccf_sizeof_order() { return static_cast<int>(sizeof(CcfOrder)); }
int ccf_sizeof_rows() { return static_cast<int>(sizeof(CcfRows)); }

long long ccf_order_rows(long long slots, int experts, long long capacity, int align) {
  if (slots < 0 || slots > CCF_SORT_MAX_SLOTS || experts < 1 || experts > CCF_SORT_MAX_EXPERTS || capacity < 1 || align < 1 || align > CCF_SORT_MAX_ALIGN) return -1;
  const long long kept = capacity < slots ? (experts * capacity < slots ? experts * capacity : slots) : slots;
  const long long rows = (kept + (experts < kept ? experts : kept) * (align - 1)) / align * align;
  return rows <= 0x7fffffffLL ? rows : -1;
}

long long ccf_order_scratch(long long slots, int experts) {
  if (slots < 1 || slots > CCF_SORT_MAX_SLOTS || experts < 1 || experts > CCF_SORT_MAX_EXPERTS) return -1;
  const ccf::OrderShape s = ccf::order_shape(slots, experts);
  return s.blocks == 1 ? 0 : static_cast<long long>(s.blocks) * experts * 4;
}

int ccf_order(const CcfOrder* o, void* stream) {
  using namespace ccf;
  const long long rows = ccf_order_rows(o->slots, o->experts, o->capacity, o->align);
  if (o->slots < 1 || rows < 0 || rows != o->rows) return -2;
  const OrderShape s = order_shape(o->slots, o->experts);
  if (o->idx == nullptr || o->slot_row == nullptr || o->row_slot == nullptr || o->counts == nullptr || o->base == nullptr ||
      (s.blocks > 1 && o->scratch == nullptr))
    return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int early = 0;
  if (s.blocks > 1) {
    early = not_capturing(st);
    order_count_kernel<<<s.blocks, kOrderThreads, o->experts * sizeof(int), st>>>(*o, static_cast<long long>(s.threads) * s.per * s.tiles);
    const int rc = launch_result();
    if (rc != 0) return rc;
  }
  const cudaError_t err = s.per == 1   ? launch_place<1>(*o, s, early, st)
                          : s.per == 2 ? launch_place<2>(*o, s, early, st)
                          : s.per == 4 ? launch_place<4>(*o, s, early, st)
                                       : launch_place<8>(*o, s, early, st);
  return err != cudaSuccess ? -static_cast<int>(err) : s.blocks > 1 ? 2 : 1;
}

int ccf_sort_rows(const CcfRows* r, int behind_order, void* stream) {
  using namespace ccf;
  if (!rows_ok(*r) || r->tokens_in == nullptr || r->ld < r->d || (r->rows > 0 && (r->rows_out == nullptr || r->row_slot == nullptr))) return -2;
  if (r->rows == 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int early = behind_order ? not_capturing(st) : 0;
  switch (unit_bytes(*r, r->ld, r->tokens_in, r->rows_out)) {
    case 16: return launch_sort<uint4>(*r, early, st);
    case 8: return launch_sort<uint2>(*r, early, st);
    case 4: return launch_sort<uint32_t>(*r, early, st);
    default: return launch_sort<uint16_t>(*r, early, st);
  }
}

int ccf_return_rows(const CcfRows* r, void* stream) {
  using namespace ccf;
  if (!rows_ok(*r) || r->tokens_out == nullptr || (r->rows > 0 && r->rows_in == nullptr)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = unit_bytes(*r, r->d, r->rows_in, r->tokens_out) == 16;
  if (r->type == kBf16) return vec ? launch_return<kBf16, true>(*r, st) : launch_return<kBf16, false>(*r, st);
  if (r->type == kFp16) return vec ? launch_return<kFp16, true>(*r, st) : launch_return<kFp16, false>(*r, st);
  return vec ? launch_return<kFp32, true>(*r, st) : launch_return<kFp32, false>(*r, st);
}

int ccf_return_rows_bwd(const CcfRows* r, void* stream) {
  using namespace ccf;
  if (!rows_ok(*r) || r->tokens_in == nullptr || r->ld < r->d || (r->d_weights != nullptr && r->rows > 0 && r->rows_in == nullptr) ||
      (r->rows_out != nullptr && r->row_slot == nullptr))
    return -2;
  if (r->rows_out == nullptr && r->d_weights == nullptr) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const void* const in = r->d_weights != nullptr ? r->rows_in : nullptr;
  const bool vec = unit_bytes(*r, r->ld, r->tokens_in, r->rows_out) == 16 && reinterpret_cast<uintptr_t>(in) % 16 == 0;
  if (r->type == kBf16) return vec ? launch_return_bwd<kBf16, true>(*r, st) : launch_return_bwd<kBf16, false>(*r, st);
  if (r->type == kFp16) return vec ? launch_return_bwd<kFp16, true>(*r, st) : launch_return_bwd<kFp16, false>(*r, st);
  return vec ? launch_return_bwd<kFp32, true>(*r, st) : launch_return_bwd<kFp32, false>(*r, st);
}

}  // extern "C"
