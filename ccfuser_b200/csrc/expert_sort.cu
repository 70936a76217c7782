// Tokens sorted by expert and back: rows[row(t, j)] = x[t], and y[t] = sum_j w[t, j] rows[row(t, j)], with the gradients of both. The layer's own
// kernels (dispatch.cuh, combine.cu) do this inside their GEMMs; these are for experts that are not the layer's.
//
// The order is routing.py's: a slot's position is the number of earlier slots of the same expert, slots from `capacity` on are dropped, an expert
// outside [0, experts) is none. Every expert's rows begin at a multiple of `align`. Nothing depends on the order in which blocks run: no atomics
// on positions or sums.
#include <algorithm>

#include "elements.cuh"
#include "expert_sort.h"

namespace ccf {

// ---- order -----------------------------------------------------------------------------------------------------------
// Bound by latency: a few bytes a slot. Up to a block's threads in slots one block does it all. Above, each block counts its slots' experts in a first kernel, and in
// the second adds up the counts of the blocks in front of it. Both kernels, of a captured graph, with blocks of 512 and of 1024 threads: 16384 slots of 64 experts 7.0 and 8.5 us, of
// 128 6.7 and 8.7, 65536 of 128 8.6 and 9.0, of 256 11.0 and 9.9, 131072 of 256 12.5 and 11.5, 524288 25.2 and 22.3 (with at most 16, 32 and 64 blocks instead of 128, these two:
// 31, 19, 13 and 108, 57, 33).
constexpr int kOrderThreads = 1024;
constexpr int kOrderBlocks = 128;                 // a block reads the counts of as many
constexpr long long kOrderMany = 1 << 24;         // slots x experts from which on blocks have kOrderThreads, else half of them
constexpr int kOrderMost = 8;                     // slots of a thread at a time

struct OrderShape {
  int threads, per, tiles, blocks;   // slots of a block: threads * per * tiles
};

inline OrderShape order_shape(long long slots, int experts) {
  OrderShape s;
  const int least = (experts + 31) / 32 * 32;      // one thread per expert
  const long long want = (slots + 31) / 32 * 32;
  const int most = slots * experts < kOrderMany ? kOrderThreads / 2 : kOrderThreads;
  s.threads = want > most ? most : static_cast<int>(want);
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

// rows of each expert and where they begin, from the totals of a block's threads: one thread per expert, sums by warps. `write`: also for the caller.
__device__ __forceinline__ void place_experts(const CcfOrder& o, const int* total, int* base, int* kept, int* part, bool write) {
  const int E = o.experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
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
    const int first = run - sum + (warp > 0 ? part[warp - 1] : 0);
    base[tid] = first;
    kept[tid] = rows;
    if (tid == E - 1) base[E] = first + sum;
    if (write) {
      o.counts[tid] = rows;
      o.base[tid] = first;
      if (tid == E - 1) o.base[E] = first + sum;
    }
  }
}

// counts[block][expert]; `chunk`, the slots of a block: a multiple of its threads
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
    // a thread adds up every `groups`-th block's count of one expert
    const int blocks = static_cast<int>(gridDim.x), mine = static_cast<int>(blockIdx.x), width = E < 32 ? E : (E + 31) / 32 * 32, groups = blockDim.x / width;
    const int group = tid / width, x = tid - group * width;
    if (x < E && group < groups) {
      int all = 0, front = 0;
#pragma unroll 8
      for (int b = group; b < blocks; b += groups) {
        const int v = counts[b * E + x];
        all += v;
        if (b < mine) front += v;
      }
      atomicAdd(&total[x], all);
      atomicAdd(&before[x], front);
    }
  } else if (tid < E) {
    int run = 0;
    for (int w = 0; w < warps; ++w) run += by_warp[w * E + tid];
    total[tid] = run;
  }
  __syncthreads();
  let_next_in();
  place_experts(o, total, base, kept, part, blockIdx.x == 0);
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

__host__ __device__ inline int elem_bytes(int type) { return type == kFp32 ? 4 : 2; }

// ---- rows ------------------------------------------------------------------------------------------------------------
// Bound by memory: each token's row is read once and written to its slots' rows (or read from them). A token has a part of a warp (a power of two of
// lanes, for short rows), a warp, or several warps of a block; each lane walks the row with some units in flight.
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;

struct RowShape {
  int units, lanes_log, warps;   // units of a row; lanes of a token up to a warp, then warps of a token (a power of two)
};

inline RowShape row_shape(long long tokens, int units, int per_lane, long long want_warps) {
  RowShape s = {units, 0, 1};
  while (s.lanes_log < 5 && (1 << s.lanes_log) < (units + per_lane - 1) / per_lane) ++s.lanes_log;
  while (s.lanes_log == 5 && s.warps < kRowWarps && s.warps * 32 * per_lane < units && tokens * s.warps < want_warps) s.warps *= 2;
  return s;
}
inline unsigned row_blocks(const RowShape& s, long long tokens) {
  const long long of_block = (kRowThreads >> s.lanes_log) / s.warps;
  return static_cast<unsigned>((tokens + of_block - 1) / of_block);
}
// With rows that no slot goes to: a warp for every four of them, up to a wave (16 tokens of 2048 in tiles of 128 rows: 75 us without, 12 with).
inline unsigned row_blocks(const RowShape& s, const CcfRows& r) {
  const long long tokens = row_blocks(s, r.tokens), none = (r.rows - r.tokens * r.top_k) / (4 * kRowWarps), wave = 8ll * sm_count();
  return static_cast<unsigned>(std::max(tokens, std::min(none, wave)));
}
// this thread's token, its first unit and the distance to the next
struct RowPlace {
  long long token;
  int unit, step;
  __device__ __forceinline__ RowPlace(const RowShape& s) {
    const int lanes = s.warps << s.lanes_log;      // lanes of a token
    token = static_cast<long long>(blockIdx.x) * (kRowThreads / lanes) + threadIdx.x / lanes;
    unit = threadIdx.x % lanes;
    step = lanes;
  }
};

// Rows that no slot goes to are zeroed by all warps of the grid, each its share of them.
template <typename Unit>
__device__ __forceinline__ void zero_rows(const CcfRows& a, Unit* out, int units) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * kRowWarps, warp = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
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

// 16-byte units that a lane has in flight, and slots whose units: 16384 tokens of 4096 bf16, two slots, back: two units of two slots 65 us (floor 62), one of two 86, one or two of
// four 85, four of two 76; its gradient: one unit 110, two 107, four 108 (eight slots of 1024 fp16 111, 101 and 135); sorted: two, four and eight 67, 66 and 64 (8192 of 2048
// in tiles of 128 rows: 24.2, 23.7 and 24.5).
constexpr int kSortUnits = 4, kReturnUnits = 2, kReturnSlots = 2, kReturnBwdUnits = 2;
// Warps per SM up to which tokens are shared by several. 8192 tokens of 2048 bf16, two slots, with 16 and 64: back 19.0 and 19.6 us, its gradient 36.9 and 36.7 (six slots of 4096
// tokens 43 and 62), sorted 26.2 and 23.7.
constexpr int kSortWarps = 64, kReturnWarps = 16;

__global__ void __launch_bounds__(kRowThreads) sort_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s, long long ld) {
  constexpr int kU = kSortUnits;
  const RowPlace at(s);
  const bool mine = at.token < a.tokens;
  const uint4* const x = static_cast<const uint4*>(a.tokens_in) + at.token * ld;
  uint4* const out = static_cast<uint4*>(a.rows_out);
  uint4 v[kU];
  const auto load = [&](int c) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (mine && c + u * at.step < s.units) v[u] = x[c + u * at.step];
  };
  load(at.unit);      // the tokens are there before the order is
  wait_for_previous();
  const int* const slot_row = behind(a.slot_row) + at.token * a.top_k;
  if (mine) {
    for (int c = at.unit; c < s.units; c += kU * at.step) {
      if (c != at.unit) load(c);
      for (int j = 0; j < a.top_k; ++j) {
        const int row = slot_row[j];
        if (row < 0 || row >= a.rows) continue;
        uint4* const y = out + static_cast<long long>(row) * s.units;
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (c + u * at.step < s.units) y[c + u * at.step] = v[u];
      }
    }
  }
  zero_rows(a, out, s.units);
}

template <int kType>
using Values = float[kElemsPer16<kType>];

__device__ __forceinline__ float load_weight(const CcfRows& a, long long slot) {
  return a.weight_type == kFp32 ? load_elem<kFp32>(a.weights, slot) : a.weight_type == kFp16 ? load_elem<kFp16>(a.weights, slot) : load_elem<kBf16>(a.weights, slot);
}

template <int kType>
__global__ void __launch_bounds__(kRowThreads) return_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s) {
  constexpr int kU = kReturnUnits, kJ = kReturnSlots, kE = kElemsPer16<kType>;
  const uint4* const rows = static_cast<const uint4*>(a.rows_in);
  const RowPlace at(s);
  if (at.token >= a.tokens) return;
  for (int c = at.unit; c < s.units; c += kU * at.step) {
    float sum[kU][kE] = {};
    for (int j0 = 0; j0 < a.top_k; j0 += kJ) {
      uint4 v[kJ][kU];
      float w[kJ];
      bool on[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const long long slot = at.token * a.top_k + j0 + j;
        const int row = j0 + j < a.top_k ? __ldg(a.slot_row + slot) : -1;
        on[j] = row >= 0 && row < a.rows;
        w[j] = on[j] && a.weights != nullptr ? load_weight(a, slot) : 1.f;
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (on[j] && c + u * at.step < s.units) v[j][u] = __ldg(rows + static_cast<long long>(row) * s.units + c + u * at.step);
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        if (!on[j]) continue;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          Values<kType> f;
          unpack16<kType>(v[j][u], f);
#pragma unroll
          for (int i = 0; i < kE; ++i) sum[u][i] = fmaf(w[j], f[i], sum[u][i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (c + u * at.step < s.units) static_cast<uint4*>(a.tokens_out)[at.token * s.units + c + u * at.step] = pack16<kType>(sum[u]);
  }
}

// The weights' gradients of kK slots from j0 on: sums over a token's lanes, and over its warps, in a fixed order.
template <int kK>
__device__ __forceinline__ void store_dots(const CcfRows& a, const RowShape& s, const RowPlace& at, bool mine, int j0, float (&dot)[kK], float (*part)[kK]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < kK; ++j)
    for (int m = (1 << s.lanes_log) / 2; m > 0; m /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
  if (s.warps > 1) {
#pragma unroll
    for (int j = 0; j < kK; ++j)
      if (lane == 0) part[warp][j] = dot[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      dot[j] = 0.f;
      if (at.unit == 0)
        for (int i = 0; i < s.warps; ++i) dot[j] += part[warp + i][j];
    }
    __syncthreads();
  }
  if (!mine || at.unit != 0) return;
#pragma unroll
  for (int j = 0; j < kK; ++j) {
    if (j0 + j >= a.top_k) break;
    const long long slot = at.token * a.top_k + j0 + j;
    if (a.weight_type == kFp32) store_elem<kFp32>(a.d_weights, slot, dot[j]);
    else if (a.weight_type == kFp16) store_elem<kFp16>(a.d_weights, slot, dot[j]);
    else store_elem<kBf16>(a.d_weights, slot, dot[j]);
  }
}
// the row of a token's slot, -1: none, and its weight
__device__ __forceinline__ int slot_of(const CcfRows& a, const RowPlace& at, bool mine, int j, float& w) {
  const long long slot = at.token * a.top_k + j;
  int row = mine && j < a.top_k ? __ldg(a.slot_row + slot) : -1;
  if (row >= a.rows) row = -1;
  w = row >= 0 && a.weights != nullptr ? load_weight(a, slot) : 1.f;
  return row;
}

// up to kK slots at a time
template <int kType, int kK>
__global__ void __launch_bounds__(kRowThreads) return_rows_bwd_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s, long long ld) {
  constexpr int kU = kReturnBwdUnits, kE = kElemsPer16<kType>;
  __shared__ float part[kRowWarps][kK];
  const RowPlace at(s);
  const bool mine = at.token < a.tokens;
  const uint4* const x = static_cast<const uint4*>(a.tokens_in) + at.token * ld;
  const uint4* const rows = static_cast<const uint4*>(a.rows_in);
  for (int j0 = 0; j0 < a.top_k; j0 += kK) {
    float dot[kK], w[kK];
    int row[kK];
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      row[j] = slot_of(a, at, mine, j0 + j, w[j]);
      dot[j] = 0.f;
    }
    for (int c = at.unit; mine && c < s.units; c += kU * at.step) {
      uint4 xv[kU], yv[kK][kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (c + u * at.step >= s.units) break;
        xv[u] = __ldg(x + c + u * at.step);
        if (a.d_weights == nullptr) continue;
#pragma unroll
        for (int j = 0; j < kK; ++j)
          if (row[j] >= 0) yv[j][u] = __ldg(rows + static_cast<long long>(row[j]) * s.units + c + u * at.step);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (c + u * at.step >= s.units) break;
        Values<kType> dy;
        unpack16<kType>(xv[u], dy);
#pragma unroll
        for (int j = 0; j < kK; ++j) {
          if (row[j] < 0) continue;
          if (a.d_weights != nullptr) {
            Values<kType> f;
            unpack16<kType>(yv[j][u], f);
#pragma unroll
            for (int i = 0; i < kE; ++i) dot[j] = fmaf(dy[i], f[i], dot[j]);
          }
          if (a.rows_out != nullptr) {
            Values<kType> d;
#pragma unroll
            for (int i = 0; i < kE; ++i) d[i] = w[j] * dy[i];
            static_cast<uint4*>(a.rows_out)[static_cast<long long>(row[j]) * s.units + c + u * at.step] = pack16<kType>(d);
          }
        }
      }
    }
    if (a.d_weights != nullptr) store_dots<kK>(a, s, at, mine, j0, dot, part);
  }
  if (a.rows_out != nullptr) zero_rows(a, static_cast<uint4*>(a.rows_out), s.units);
}

// ---- rows that do not all begin on 16 bytes ---------------------------------------------------------------------------------
// The same over the aligned 16-byte pieces of what is written: each is put together from the two aligned pieces of a source that it lies across. Single
// elements took 266, 221 and 80 us where these take 82, 134 and 74 (16384 tokens of 3001 bf16, two slots; back, its gradient, sorted; floors 45, 75 and 45). Two pieces of the
// way back in flight 106, of its gradient 144.
constexpr int kReturnPieces = 1;     // that a lane has in flight on the way back
// pieces of a row of `bytes` at `row`
__device__ __forceinline__ int piece_count(const char* row, int bytes) {
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
  return (off + bytes + 15) >> 4;
}
__device__ __forceinline__ int piece_begin(const char* row, int piece) { return 16 * piece - static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); }

// Bytes [rel, rel + 16) of a row; what lies outside the row is anything. Only aligned pieces that hold a byte of the row are read.
__device__ __forceinline__ uint4 load_across(const char* row, int bytes, int rel) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(row) + rel;
  const int off = static_cast<int>(p & 15), lo_rel = rel - off;
  const uint4* const q = reinterpret_cast<const uint4*>(p - off);
  uint4 lo = {}, hi = {};
  if (lo_rel + 16 > 0 && lo_rel < bytes) lo = __ldg(q);
  if (off != 0 && lo_rel + 32 > 0 && lo_rel + 16 < bytes) hi = __ldg(q + 1);
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (off & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int shift = (off & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift), __funnelshift_r(w[2], w[3], shift), __funnelshift_r(w[3], w[4], shift));
}
// those of its bytes that belong to the row
template <int kBytes>
__device__ __forceinline__ void store_piece(char* row, int bytes, int rel, const uint4& v) {
  if (rel >= 0 && rel + 16 <= bytes) {
    *reinterpret_cast<uint4*>(row + rel) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 16; i += kBytes) {
    if (rel + i < 0 || rel + i >= bytes) continue;
    if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(row + rel + i) = w[i / 4];
    else *reinterpret_cast<uint16_t*>(row + rel + i) = static_cast<uint16_t>(w[i / 4] >> (8 * (i & 3)));
  }
}

template <int kBytes>
__device__ __forceinline__ void zero_odd_rows(const CcfRows& a) {
  if constexpr (kBytes == 4) zero_rows(a, static_cast<uint32_t*>(a.rows_out), a.d);
  else zero_rows(a, static_cast<uint16_t*>(a.rows_out), a.d);
}

template <int kBytes>
__global__ void __launch_bounds__(kRowThreads) sort_odd_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s) {
  const RowPlace at(s);
  const bool mine = at.token < a.tokens;
  const int bytes = a.d * kBytes;
  const char* const x = static_cast<const char*>(a.tokens_in) + at.token * a.ld * kBytes;
  wait_for_previous();
  const int* const slot_row = behind(a.slot_row) + at.token * a.top_k;
  for (int j = 0; mine && j < a.top_k; ++j) {
    const int row = slot_row[j];
    if (row < 0 || row >= a.rows) continue;
    char* const y = static_cast<char*>(a.rows_out) + static_cast<long long>(row) * bytes;
    const int pieces = piece_count(y, bytes);
#pragma unroll 2
    for (int c = at.unit; c < pieces; c += at.step) {
      const int rel = piece_begin(y, c);
      store_piece<kBytes>(y, bytes, rel, load_across(x, bytes, rel));
    }
  }
  zero_odd_rows<kBytes>(a);
}

template <int kType>
__global__ void __launch_bounds__(kRowThreads) return_odd_rows_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s) {
  constexpr int kU = kReturnPieces, kJ = kReturnSlots, kE = kElemsPer16<kType>, kBytes = kElemBytes<kType>;
  const RowPlace at(s);
  if (at.token >= a.tokens) return;
  const int bytes = a.d * kBytes;
  char* const y = static_cast<char*>(a.tokens_out) + at.token * bytes;
  const int pieces = piece_count(y, bytes);
  for (int c = at.unit; c < pieces; c += kU * at.step) {
    Values<kType> sum[kU] = {};
    for (int j0 = 0; j0 < a.top_k; j0 += kJ) {
      uint4 v[kU][kJ];
      float w[kJ];
      int row[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        row[j] = slot_of(a, at, true, j0 + j, w[j]);
        const char* const from = static_cast<const char*>(a.rows_in) + static_cast<long long>(row[j]) * bytes;
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (row[j] >= 0 && c + u * at.step < pieces) v[u][j] = load_across(from, bytes, piece_begin(y, c + u * at.step));
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        if (row[j] < 0) continue;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          Values<kType> f;
          unpack16<kType>(v[u][j], f);
#pragma unroll
          for (int i = 0; i < kE; ++i) sum[u][i] = fmaf(w[j], f[i], sum[u][i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (c + u * at.step < pieces) store_piece<kBytes>(y, bytes, piece_begin(y, c + u * at.step), pack16<kType>(sum[u]));
  }
}

template <int kType, int kK>
__global__ void __launch_bounds__(kRowThreads) return_odd_rows_bwd_kernel(const __grid_constant__ CcfRows a, const __grid_constant__ RowShape s) {
  constexpr int kE = kElemsPer16<kType>, kBytes = kElemBytes<kType>;
  __shared__ float part[kRowWarps][kK];
  const RowPlace at(s);
  const bool mine = at.token < a.tokens;
  const int bytes = a.d * kBytes;
  const char* const x = static_cast<const char*>(a.tokens_in) + at.token * a.ld * kBytes;
  for (int j0 = 0; j0 < a.top_k; j0 += kK) {
    float dot[kK];
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      dot[j] = 0.f;
      float w;
      const int row = slot_of(a, at, mine, j0 + j, w);
      if (row < 0) continue;
      char* const out = static_cast<char*>(a.rows_out) + static_cast<long long>(row) * bytes;      // the grid of pieces is the output's, or its rows' alone
      const char* const y = static_cast<const char*>(a.rows_in) + static_cast<long long>(row) * bytes;
      const char* const grid = a.rows_out != nullptr ? out : y;
      const int pieces = piece_count(grid, bytes);
#pragma unroll 1
      for (int c = at.unit; c < pieces; c += at.step) {
        const int rel = piece_begin(grid, c);
        Values<kType> dy;
        unpack16<kType>(load_across(x, bytes, rel), dy);
        if (a.d_weights != nullptr) {
          Values<kType> f;
          unpack16<kType>(load_across(y, bytes, rel), f);
          if (rel >= 0 && rel + 16 <= bytes) {
#pragma unroll
            for (int i = 0; i < kE; ++i) dot[j] = fmaf(dy[i], f[i], dot[j]);
          } else {
#pragma unroll
            for (int i = 0; i < kE; ++i)
              if (rel + i * kBytes >= 0 && rel + i * kBytes < bytes) dot[j] = fmaf(dy[i], f[i], dot[j]);
          }
        }
        if (a.rows_out != nullptr) {
#pragma unroll
          for (int i = 0; i < kE; ++i) dy[i] *= w;
          store_piece<kBytes>(out, bytes, rel, pack16<kType>(dy));
        }
      }
    }
    if (a.d_weights != nullptr) store_dots<kK>(a, s, at, mine, j0, dot, part);
  }
  if (a.rows_out != nullptr) zero_odd_rows<kBytes>(a);
}

// ---- a few tokens: order and rows in one launch ----------------------------------------------------------------------------
// Every block orders all slots for itself and copies the rows of its tokens. Of a captured graph, with the two or three kernels above: 16 tokens of 2048, two of 64
// experts, 2.7 us (6.5), 128 tokens 3.0 (5.9), 256 4.5 (6.2), 512 5.5 (8.8), 1024 8.7 (9.2); 512 in tiles of 128 rows 10.4 (15.0), 128 tokens with eight of 256 experts 7.9 (14.7).
constexpr int kFewThreads = 256, kFewPer = 8, kFewSlots = kFewThreads * kFewPer, kFewExperts = kFewThreads;

// kBytes: of an element where rows do not all begin on 16 bytes, else 0
template <int kPer, int kBytes>
__global__ void __launch_bounds__(kFewThreads) sort_few_kernel(const __grid_constant__ CcfOrder o, const __grid_constant__ CcfRows a) {
  constexpr int kWarps = kFewThreads / 32;
  __shared__ int by_warp[kWarps * kFewExperts], total[kFewExperts], base[kFewExperts + 1], kept[kFewExperts], part[32], row_of[kFewSlots];
  const int E = o.experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int e[kPer], r[kPer];
  rank_slots<kPer>(o, warp * 32 * kPer, by_warp + warp * E, e, r);
  __syncthreads();
  if (tid < E) {
    int run = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = by_warp[w * E + tid];
      by_warp[w * E + tid] = run;
      run += c;
    }
    total[tid] = run;
  }
  __syncthreads();
  place_experts(o, total, base, kept, part, blockIdx.x == 0);
  __syncthreads();
  const int slots = static_cast<int>(o.slots), blocks = static_cast<int>(gridDim.x), block = static_cast<int>(blockIdx.x);
#pragma unroll
  for (int l = 0; l < kPer; ++l) {
    const int s = warp * 32 * kPer + 32 * l + lane;
    if (s >= slots) continue;
    int row = -1;
    if (e[l] >= 0) {
      const int pos = by_warp[warp * E + e[l]] + r[l];
      if (pos < kept[e[l]]) row = base[e[l]] + pos;
    }
    row_of[s] = row;
    if (block == 0) {
      o.slot_row[s] = row;
      if (row >= 0) o.row_slot[row] = s;
    }
  }
  __syncthreads();
  const int bytes = a.d * (kBytes == 0 ? elem_bytes(a.type) : kBytes);
  char* const out = static_cast<char*>(a.rows_out);
  for (int t = block; t < a.tokens; t += blocks) {
    const char* const x = static_cast<const char*>(a.tokens_in) + t * a.ld * elem_bytes(a.type);
    if constexpr (kBytes == 0) {
      for (int c = tid; c < bytes / 16; c += kFewThreads) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(x) + c);
        for (int j = 0; j < a.top_k; ++j) {
          const int row = row_of[t * a.top_k + j];
          if (row >= 0) *reinterpret_cast<uint4*>(out + static_cast<long long>(row) * bytes + 16 * c) = v;
        }
      }
    } else {
      for (int j = 0; j < a.top_k; ++j) {
        const int row = row_of[t * a.top_k + j];
        if (row < 0) continue;
        char* const y = out + static_cast<long long>(row) * bytes;
        for (int c = tid; c < piece_count(y, bytes); c += kFewThreads) {
          const int rel = piece_begin(y, c);
          store_piece<kBytes>(y, bytes, rel, load_across(x, bytes, rel));
        }
      }
    }
  }
  // rows without a slot: a warp each
  const int warps = blocks * kWarps, mine = block * kWarps + warp;
  const auto none = [&](int row) {
    if (lane == 0) o.row_slot[row] = -1;
    char* const y = out + static_cast<long long>(row) * bytes;
    if constexpr (kBytes == 0) {
      for (int c = lane; c < bytes / 16; c += 32) reinterpret_cast<uint4*>(y)[c] = uint4{};
    } else if constexpr (kBytes == 4) {
      for (int c = lane; c < a.d; c += 32) reinterpret_cast<uint32_t*>(y)[c] = 0;
    } else {
      for (int c = lane; c < a.d; c += 32) reinterpret_cast<uint16_t*>(y)[c] = 0;
    }
  };
  if (o.align > 1) {      // an expert's are shared by every E-th warp
    const int shares = warps >= E ? warps / E : 1;
    for (int i = mine; i < E * shares; i += warps) {
      const int x = i % E;
      for (int row = base[x] + kept[x] + i / E; row < base[x + 1]; row += shares) none(row);
    }
  }
  for (long long row = base[E] + mine; row < o.rows; row += warps) none(static_cast<int>(row));
}

// ---- launches ------------------------------------------------------------------------------------------------------------
inline bool rows_ok(const CcfRows& r) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(r.tokens_in) | reinterpret_cast<uintptr_t>(r.rows_in) | reinterpret_cast<uintptr_t>(r.tokens_out) |
                       reinterpret_cast<uintptr_t>(r.rows_out);
  return r.type >= 0 && r.type <= 2 && at % elem_bytes(r.type) == 0 && r.tokens >= 1 && r.rows >= 0 && r.rows <= 0x7fffffffLL && r.top_k >= 1 &&
         r.tokens <= CCF_SORT_MAX_SLOTS && r.tokens * r.top_k <= CCF_SORT_MAX_SLOTS && r.d >= 1 && r.d <= CCF_SORT_MAX_D && r.weight_type >= 0 && r.weight_type <= 2 &&
         r.slot_row != nullptr;
}
// whether all rows begin on 16 bytes
inline bool rows_aligned(const CcfRows& r, long long ld, const void* a, const void* b, const void* c) {
  const unsigned long long size = elem_bytes(r.type);
  return ((r.d * size | ld * size | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 15) == 0;
}
// 16-byte units of a row, or pieces at most
inline int units_of(const CcfRows& r, bool aligned) { return static_cast<int>((static_cast<long long>(r.d) * elem_bytes(r.type) + 15) / 16) + (aligned ? 0 : 1); }

static int launch_sort(const CcfRows& r, int early, cudaStream_t st) {
  const bool aligned = rows_aligned(r, r.ld, r.tokens_in, r.rows_out, nullptr);
  const RowShape s = row_shape(r.tokens, units_of(r, aligned), aligned ? kSortUnits : 2, kSortWarps * sm_count());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_blocks(s, r));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr = early_attribute();
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  const cudaError_t err = aligned               ? cudaLaunchKernelEx(&cfg, sort_rows_kernel, r, s, r.ld * elem_bytes(r.type) / 16)
                          : r.type == kFp32 ? cudaLaunchKernelEx(&cfg, sort_odd_rows_kernel<4>, r, s)
                                                : cudaLaunchKernelEx(&cfg, sort_odd_rows_kernel<2>, r, s);
  return err == cudaSuccess ? 0 : -static_cast<int>(err);
}

template <int kType>
static int launch_return(const CcfRows& r, cudaStream_t st) {
  const bool aligned = rows_aligned(r, r.d, r.rows_in, r.tokens_out, nullptr);
  const RowShape s = row_shape(r.tokens, units_of(r, aligned), aligned ? kReturnUnits : 1, (aligned ? kReturnWarps : kSortWarps) * sm_count());
  if (aligned) return_rows_kernel<kType><<<row_blocks(s, r.tokens), kRowThreads, 0, st>>>(r, s);
  else return_odd_rows_kernel<kType><<<row_blocks(s, r.tokens), kRowThreads, 0, st>>>(r, s);
  return launch_result();
}

template <int kType>
static int launch_return_bwd(const CcfRows& r, cudaStream_t st) {
  const bool aligned = rows_aligned(r, r.ld, r.tokens_in, r.rows_out, r.d_weights != nullptr ? r.rows_in : nullptr);
  const RowShape s = row_shape(r.tokens, units_of(r, aligned), kReturnBwdUnits, kReturnWarps * sm_count());
  const unsigned blocks = r.rows_out != nullptr ? row_blocks(s, r) : row_blocks(s, r.tokens);
  if (aligned) {
    const auto kern = r.top_k == 1   ? return_rows_bwd_kernel<kType, 1>
                      : r.top_k == 2 ? return_rows_bwd_kernel<kType, 2>
                      : r.top_k <= 4 ? return_rows_bwd_kernel<kType, 4>
                                     : return_rows_bwd_kernel<kType, 8>;
    kern<<<blocks, kRowThreads, 0, st>>>(r, s, r.ld * elem_bytes(r.type) / 16);
  } else {
    const auto kern = r.top_k <= 2 ? return_odd_rows_bwd_kernel<kType, 2> : return_odd_rows_bwd_kernel<kType, 4>;
    kern<<<blocks, kRowThreads, 0, st>>>(r, s);
  }
  return launch_result();
}

constexpr size_t order_shared(int threads, int experts) { return (static_cast<size_t>(threads / 32) * experts + 4 * experts + 1) * sizeof(int); }

template <int kPer>
static cudaError_t launch_place(const CcfOrder& o, const OrderShape& s, int early, cudaStream_t st) {
  const size_t shared = order_shared(s.threads, o.experts);
  if (shared > 48 * 1024) {      // the most of any call: another thread's call may come between this and the launch
    constexpr int most = static_cast<int>(order_shared(kOrderThreads, CCF_SORT_MAX_EXPERTS));
    const cudaError_t err = cudaFuncSetAttribute(order_place_kernel<kPer>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
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

static bool order_ok(const CcfOrder& o) {
  const long long rows = ccf_order_rows(o.slots, o.experts, o.capacity, o.align);
  return o.slots >= 1 && rows >= 0 && rows == o.rows && o.idx != nullptr && o.slot_row != nullptr && o.row_slot != nullptr && o.counts != nullptr && o.base != nullptr;
}

int ccf_order(const CcfOrder* o, void* stream) {
  using namespace ccf;
  if (!order_ok(*o)) return -2;
  const OrderShape s = order_shape(o->slots, o->experts);
  if (s.blocks > 1 && o->scratch == nullptr) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int early = 0;
  if (s.blocks > 1) {
    early = not_capturing(st);
    order_count_kernel<<<s.blocks, s.threads, o->experts * sizeof(int), st>>>(*o, static_cast<long long>(s.threads) * s.per * s.tiles);
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
  return launch_sort(*r, early, st);
}

int ccf_sort_by_expert(const CcfOrder* o, const CcfRows* r, void* stream) {
  using namespace ccf;
  if (!order_ok(*o) || !rows_ok(*r) || r->tokens_in == nullptr || r->ld < r->d || r->rows_out == nullptr || r->tokens * r->top_k != o->slots || r->rows != o->rows ||
      r->slot_row != o->slot_row || r->row_slot != o->row_slot)
    return -2;
  if (o->slots > kFewSlots || o->experts > kFewExperts) {
    const int launches = ccf_order(o, stream);
    if (launches < 0) return launches;
    const int rc = ccf_sort_rows(r, 1, stream);
    return rc < 0 ? rc : launches + 1;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool aligned = rows_aligned(*r, r->ld, r->tokens_in, r->rows_out, nullptr);
  // a block for each token and for every eight rows without a slot, up to one per SM
  const long long want = r->tokens + (r->rows - o->slots > 0 ? (r->rows - o->slots) / 8 : 0);
  const unsigned blocks = static_cast<unsigned>(want < sm_count() ? want : sm_count());
  const int bytes = aligned ? 0 : elem_bytes(r->type);
  const auto pick = [bytes](auto aligned_rows, auto halves, auto floats) { return bytes == 0 ? aligned_rows : bytes == 2 ? halves : floats; };
  const auto kern = o->slots <= kFewThreads       ? pick(sort_few_kernel<1, 0>, sort_few_kernel<1, 2>, sort_few_kernel<1, 4>)
                    : o->slots <= 4 * kFewThreads ? pick(sort_few_kernel<4, 0>, sort_few_kernel<4, 2>, sort_few_kernel<4, 4>)
                                                  : pick(sort_few_kernel<kFewPer, 0>, sort_few_kernel<kFewPer, 2>, sort_few_kernel<kFewPer, 4>);
  kern<<<blocks, kFewThreads, 0, st>>>(*o, *r);
  const int rc = launch_result();
  return rc < 0 ? rc : 1;
}

int ccf_return_rows(const CcfRows* r, void* stream) {
  using namespace ccf;
  if (!rows_ok(*r) || r->tokens_out == nullptr || (r->rows > 0 && r->rows_in == nullptr)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return r->type == kBf16 ? launch_return<kBf16>(*r, st) : r->type == kFp16 ? launch_return<kFp16>(*r, st) : launch_return<kFp32>(*r, st);
}

int ccf_return_rows_bwd(const CcfRows* r, void* stream) {
  using namespace ccf;
  if (!rows_ok(*r) || r->tokens_in == nullptr || r->ld < r->d || (r->d_weights != nullptr && r->rows > 0 && r->rows_in == nullptr) ||
      (r->rows_out != nullptr && r->row_slot == nullptr))
    return -2;
  if (r->rows_out == nullptr && r->d_weights == nullptr) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return r->type == kBf16 ? launch_return_bwd<kBf16>(*r, st) : r->type == kFp16 ? launch_return_bwd<kFp16>(*r, st) : launch_return_bwd<kFp32>(*r, st);
}

}  // extern "C"
