// Sums of embedding lookups and their dense gradients: y_t = scale * W[id_t] + P[pos_t] + T[type_t], the input of the example models
// (stock GPT-2 / BERT / Transformer-XL: mix_moe/mix_moe/examples/models/moe_gpt.py, moe_bert.py,
// transformer-xl/mem_transformer_mix_moe.py).
//
// Both directions are bound by bytes. Forward: the used rows in, y out. Backward: dW[v] = scale * sum of dy_t over the tokens with id v, in
// fp32, rounded once; dy is read once and every row of the gradient written once. The tokens are sorted by (id, place) first, and a row's
// sum runs over its tokens in an order that the ids determine: no atomics on values, the same bits every time. GPT's step (8192 tokens of 2048
// bf16, 50304 and 1024 rows) 57 us, 4.7 TB/s of its 270 MB: the sort in front (10.7 us) and the latency of the sums leave the memory idle for part of it.
#include <cooperative_groups.h>

#include "elements.cuh"
#include "embedding.h"

namespace ccf {

constexpr int kSortChunk = 1024;     // keys that one block sorts in shared memory
constexpr int kEmbWarps = 8;
constexpr int kJoinWarps = 16;
constexpr uint32_t kShort = 4;       // further pieces of a run that a warp adds up by itself
constexpr uint32_t kNoRow = 0xffffffffu;   // id of a token without a gradient: skipped row, index out of range

// a product that may pass 32 bits, in one instruction
__device__ __forceinline__ uint64_t wide(uint32_t a, uint32_t b) { return static_cast<uint64_t>(a) * b; }

// What a warp, or kLanes of its lanes, hold of a row: kLanes * kE consecutive elements from a column on. kVec: 16 bytes per lane; otherwise (rows off
// 16-byte boundaries) one element per lane and access.
template <int kType, bool kVec, int kLanes = 32>
struct Slice {
  static constexpr int kE = kElemsPer16<kType>;
  static constexpr int kCols = kLanes * kE;
  uint4 q;
  float s[kVec ? 1 : kE];

  static __device__ __forceinline__ int lane() { return lane_id() & (kLanes - 1); }
  static __device__ __forceinline__ int col(int i) { return kVec ? lane() * kE + i : lane() + kLanes * i; }
  __device__ __forceinline__ void load(const void* p, size_t at, int left, bool on) {
    if constexpr (kVec) {
      q = make_uint4(0, 0, 0, 0);
      if (on && lane() * kE < left)
        q = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + at * kElemBytes<kType>) + lane());
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) s[i] = on && col(i) < left ? load_elem<kType>(p, static_cast<long long>(at) + col(i)) : 0.f;
    }
  }
  // f += scale * this, or with kFirst f = scale * this, in pairs
  template <bool kFirst>
  __device__ __forceinline__ void add_to(f32x2 (&f)[kE / 2], f32x2 scale) const {
    float v[kE];
    get(v);
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) {
      const f32x2 x = pk2(v[2 * i], v[2 * i + 1]);
      f[i] = kFirst ? mul2(x, scale) : fma2(x, scale, f[i]);
    }
  }
  __device__ __forceinline__ void get(float (&f)[kE]) const {
    if constexpr (kVec) {
      unpack16<kType>(q, f);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) f[i] = s[i];
    }
  }
  static __device__ __forceinline__ void store(void* p, size_t at, int left, const float (&f)[kE]) {
    if constexpr (kVec) {
      if (lane() * kE < left)
        reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p) + at * kElemBytes<kType>)[lane()] = pack16<kType>(f);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (col(i) < left) store_elem<kType>(p, static_cast<long long>(at) + col(i), f[i]);
    }
  }
  static __device__ __forceinline__ void store_f32(float* p, int left, const float (&f)[kE]) {
    if constexpr (kVec) {
      if (lane() * kE >= left) return;
#pragma unroll
      for (int i = 0; i < kE; i += 4) reinterpret_cast<float4*>(p + col(i))[0] = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (col(i) < left) p[col(i)] = f[i];
    }
  }
  static __device__ __forceinline__ void load_f32(const float* p, int left, float (&f)[kE]) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kE; i += 4) {
        const float4 v = lane() * kE < left ? reinterpret_cast<const float4*>(p + col(i))[0] : make_float4(0.f, 0.f, 0.f, 0.f);
        f[i] = v.x;
        f[i + 1] = v.y;
        f[i + 2] = v.z;
        f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) f[i] = col(i) < left ? p[col(i)] : 0.f;
    }
  }
  static __device__ __forceinline__ void store_zero(void* p, size_t at, int left) {   // past the L2 where it may: nobody reads it soon
    if constexpr (kVec) {
      if (lane() * kE < left) __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p) + at * kElemBytes<kType>) + lane(), make_uint4(0, 0, 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (col(i) < left) store_elem<kType>(p, static_cast<long long>(at) + col(i), 0.f);
    }
  }
};

// ---- forward -----------------------------------------------------------------------------------------------------------
// A warp takes one slice of the columns for up to 16 consecutive tokens: their ids in one load, then kFwdRows tokens' rows of every table in flight (64
// registers, four blocks an SM). With a token at a time the chain from an id to its row was walked for every kilobyte. Few tokens: fewer for each warp, so that
// they spread over the card. 8192 tokens of 2048 bf16 with positions 14.8 us (52 MB from and to memory: 3.5 TB/s); tokens at one place of
// several sequences, whose position then comes from L1, 16.4.
constexpr int kFwdTokens = 16;
template <int kTables>
constexpr int kFwdRows = kTables <= 2 ? 4 : 2;

template <int kType, bool kVec, int kTables>
__global__ void __launch_bounds__(32 * kEmbWarps, 4) embedding_fwd_kernel(const __grid_constant__ CcfEmbed e, void* __restrict__ y, int* status, uint32_t each,
                                                                          uint32_t slices) {
  using S = Slice<kType, kVec>;
  constexpr int kRows = kFwdRows<kTables>;
  const uint32_t unit = blockIdx.x * kEmbWarps + (threadIdx.x >> 5), part = unit / slices, c = (unit - part * slices) * S::kCols;
  const uint32_t tokens = static_cast<uint32_t>(e.tokens), begin = part * each;
  if (begin >= tokens) return;
  const uint32_t n = min(each, tokens - begin);
  const int left = e.d - static_cast<int>(c);
  uint64_t at[kTables];   // where lane t finds token t's row
  bool in = true;
#pragma unroll
  for (int k = 0; k < kTables; ++k) {
    const CcfEmbedTable& w = e.table[k];
    const uint32_t t = begin + min(static_cast<uint32_t>(lane_id()), n - 1);
    const long long id = w.ids != nullptr ? load_index(w.ids, t, w.wide) : static_cast<long long>(t % static_cast<uint32_t>(e.seq));
    const bool here = id >= 0 && id < w.rows;
    in = in && here;
    at[k] = here ? static_cast<uint64_t>(id) * w.ld + c : c;
  }
  const uint32_t good = __ballot_sync(0xffffffffu, in);
  if (c == 0 && !in && lane_id() < n) report_index(status, begin + lane_id());
  for (uint32_t t0 = 0; t0 < n; t0 += kRows) {
    S row[kTables][kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
#pragma unroll
      for (int k = 0; k < kTables; ++k) row[k][u].load(e.table[k].weight, __shfl_sync(0xffffffffu, at[k], t0 + u), left, t0 + u < n);
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (t0 + u >= n) break;
      f32x2 pairs[S::kE / 2];
      row[0][u].template add_to<true>(pairs, bc2(e.table[0].scale));
#pragma unroll
      for (int k = 1; k < kTables; ++k) row[k][u].template add_to<false>(pairs, bc2(e.table[k].scale));
      float sum[S::kE];
#pragma unroll
      for (int i = 0; i < S::kE / 2; ++i) upk2(pairs[i], sum[2 * i], sum[2 * i + 1]);
      if (!(good >> (t0 + u) & 1)) {
#pragma unroll
        for (int i = 0; i < S::kE; ++i) sum[i] = __int_as_float(0x7fc00000);
      }
      S::store(y, wide(begin + t0 + u, e.d) + c, left, sum);
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// Scratch of one table. `keys`: (id << 32 | token), sorted. `slot`: for a row that some token has, one of its tokens. A run of equal ids is cut where
// a piece of the sorted tokens ends: a piece leaves the sum of a run that came from the piece before in `head`, of one that began in it and goes on in
// `tail`; `list` holds the pieces that left a tail, with the run's id: from the front
// those of runs with at most kShort further pieces, from the back the others; `count` says how many of each.
struct GradTable {
  const void* ids;
  void* grad;
  uint64_t* sorted_chunks;
  uint32_t* chunk_ids;   // the ids of sorted_chunks
  uint64_t* keys;
  uint32_t* slot;
  float* head;
  float* tail;
  uint2* list;
  int* count;
  long long rows;
  long long skip;
  float scale;
  int wide;
  uint32_t piece, pieces, blocks;   // tokens of a piece, pieces, blocks that sum them
};
struct GradArgs {
  GradTable table[CCF_EMBED_TABLES];
  const void* dy;
  int* status;
  uint32_t tokens, seq, batch;
  uint32_t chunks, slices;
  uint32_t sums;   // blocks that sum, those of all tables
  int tables, d;
};

__device__ __forceinline__ uint32_t id_of(uint64_t key) { return static_cast<uint32_t>(key >> 32); }

// The i-th token in the order of the ids. Positions need no sort: place s of every sequence, in the order of the sequences.
__device__ __forceinline__ uint64_t key_at(const GradArgs& g, const GradTable& t, uint32_t i) {
  if (t.ids != nullptr) return t.keys[i];   // not through the read-only path: an earlier launch of this call wrote it
  const uint32_t s = i / g.batch;
  return static_cast<uint64_t>(s) << 32 | ((i - s * g.batch) * g.seq + s);
}

// The place of a key among all: its place in its own chunk and, for every other chunk, the keys there that are smaller: those of smaller ids and, in
// earlier chunks, of the same. `ids`: those of kSide chunks from chunk c on, in order, kNoRow where there is none; searched side by side, three instructions a
// step (with bounds and both comparisons in it eight, and 7.7 us for 8192 tokens in eight blocks instead of 4).
constexpr int kSide = 8;
__device__ __forceinline__ uint32_t smaller_elsewhere(const GradArgs& g, const uint32_t* ids, uint32_t c, uint32_t own, uint32_t id) {
  uint32_t lo[kSide], below[kSide], n = 0;
#pragma unroll
  for (int u = 0; u < kSide; ++u) {
    lo[u] = 0;
    below[u] = c + u < own ? id + 1 : id;
  }
#pragma unroll
  for (uint32_t step = kSortChunk / 2; step > 0; step /= 2) {
#pragma unroll
    for (int u = 0; u < kSide; ++u)
      if (ids[u * kSortChunk + lo[u] + step - 1] < below[u]) lo[u] += step;
  }
#pragma unroll
  for (int u = 0; u < kSide; ++u) {
    lo[u] += ids[u * kSortChunk + lo[u]] < below[u];
    // a token without a row stands behind all of an earlier chunk (its id + 1 is 0)
    if (id == kNoRow && c + u < own) lo[u] = kSortChunk;
    if (c + u != own) n += lo[u];
  }
  return n;
}

// Key of the sort: (id, place in the chunk) in 32 bits for tables of less than kShortRows rows, in 64 for larger ones.
constexpr uint32_t kShortRows = (1u << 22) - 1;
template <typename Key>
constexpr int kPlaceBits = sizeof(Key) == 4 ? 10 : 32;
template <typename Key>
constexpr uint32_t kLast = sizeof(Key) == 4 ? kShortRows : kNoRow;   // the id of a token without a row
template <typename Key>
__device__ __forceinline__ uint32_t key_id(Key key) {
  const uint32_t id = static_cast<uint32_t>(key >> kPlaceBits<Key>);
  return id == kLast<Key> ? kNoRow : id;
}

// n keys of a block of kSortChunk threads, one each, in order: bitonic, with exchanges inside a warp by shuffles and the others through shared memory.
template <typename Key>
__device__ __forceinline__ Key sort_keys(Key key, Key (&other)[2][kSortChunk], uint32_t n) {
  const uint32_t tid = threadIdx.x;
  int half = 0;
#pragma unroll 1
  for (uint32_t size = 2; size < 2 * n; size *= 2) {
    const bool up = (tid & size) == 0;
#pragma unroll 1
    for (uint32_t j = size / 2; j >= 32; j /= 2, half ^= 1) {
      other[half][tid] = key;
      __syncthreads();
      const Key o = other[half][tid ^ j];
      key = (((tid & j) == 0) == up) == (o < key) ? o : key;
    }
#pragma unroll
    for (uint32_t j = 16; j > 0; j /= 2) {
      if (j >= size) continue;
      const Key o = __shfl_xor_sync(0xffffffffu, key, j);
      key = (((tid & j) == 0) == up) == (o < key) ? o : key;
    }
  }
  return key;
}

// Each block sorts one chunk of keys, one for each thread.
// Up to kSide chunks are one cluster, whose blocks then read each other's ids and put every key in its place among all: 8192 tokens in one launch.
// Every token also leaves its place in `slot` at its id, whichever of equal ids comes last: a row is used if the token named there has its id. So
// `slot` needs no zeros beforehand, and what it says is the same whoever won. 8192 tokens 10.7 us; a chunk of 2048 64-bit keys sorted in shared
// memory alone took 17, and the merge as a launch of its own 9 more.
template <typename Key>
__global__ void __launch_bounds__(kSortChunk) embedding_sort_kernel(const __grid_constant__ GradArgs g) {
  namespace cg = cooperative_groups;
  __shared__ Key other[2][kSortChunk];
  __shared__ uint32_t ids[kSide * kSortChunk];
  const GradTable& t = g.table[blockIdx.y];
  let_next_in();
  if (blockIdx.x == 0 && threadIdx.x < 2) t.count[threadIdx.x] = 0;
  if (t.ids == nullptr) return;
  const uint32_t tid = threadIdx.x, own = blockIdx.x, base = own * kSortChunk;
  const uint32_t n = own < g.chunks ? min(g.tokens - base, static_cast<uint32_t>(kSortChunk)) : 0;
  Key key = ~static_cast<Key>(0);
  if (tid < n) {
    const long long id = load_index(t.ids, base + tid, t.wide);
    const bool in = id >= 0 && id < t.rows;
    if (!in) report_index(g.status, base + tid);
    else t.slot[id] = base + tid;
    key = static_cast<Key>(in && id != t.skip ? static_cast<uint32_t>(id) : kLast<Key>) << kPlaceBits<Key> | tid;
  }
  key = sort_keys(key, other, n);
  const uint32_t id = tid < n ? key_id(key) : kNoRow;
  const uint64_t full = static_cast<uint64_t>(id) << 32 | (base + (static_cast<uint32_t>(key) & (kSortChunk - 1)));
  if (g.chunks > kSide) {   // the merging kernel goes on
    if (tid < n) t.sorted_chunks[base + tid] = full;
    t.chunk_ids[base + tid] = id;
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (own < g.chunks) ids[own * kSortChunk + tid] = id;
  cluster.sync();
#pragma unroll
  for (uint32_t u = 0; u < kSide; ++u)
    if (u != own) ids[u * kSortChunk + tid] = u < g.chunks ? cluster.map_shared_rank(ids, u)[u * kSortChunk + tid] : kNoRow;
  cluster.sync();   // nobody leaves while its shared memory is read
  if (tid < n) t.keys[tid + smaller_elsewhere(g, ids, 0, own, id)] = full;
}

// More chunks than a cluster has blocks: kMergeThreads keys of one chunk a block, the ids of kSide chunks at a time in shared memory.
constexpr int kMergeThreads = 256;
__global__ void __launch_bounds__(kMergeThreads) embedding_merge_kernel(const __grid_constant__ GradArgs g) {
  constexpr int kEach = kSide * kSortChunk / 4 / kMergeThreads;   // 16-byte pieces of ids for each thread
  __shared__ uint4 staged[kSide * kSortChunk / 4];
  after_previous();
  const GradTable& t = g.table[blockIdx.y];
  if (t.ids == nullptr) return;
  const uint32_t i = blockIdx.x * kMergeThreads + threadIdx.x, own = i / kSortChunk;
  const uint64_t key = i < g.tokens ? t.sorted_chunks[i] : ~0ull;
  uint32_t place = i % kSortChunk;
  for (uint32_t c = 0; c < g.chunks; c += kSide) {
    const uint32_t most = min(static_cast<uint32_t>(kSide), g.chunks - c) * (kSortChunk / 4);   // the rest: no chunks
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const uint32_t at = u * kMergeThreads + threadIdx.x;
      staged[at] = at < most ? reinterpret_cast<const uint4*>(t.chunk_ids + c * kSortChunk)[at] : make_uint4(kNoRow, kNoRow, kNoRow, kNoRow);
    }
    __syncthreads();
    place += smaller_elsewhere(g, reinterpret_cast<const uint32_t*>(staged), c, own, id_of(key));
    __syncthreads();
  }
  if (i < g.tokens) t.keys[place] = key;
}

// Up to kSortChunk tokens: one launch. A block for each table and narrow slice of the columns sorts the tokens by itself (every block the same ones: cheaper than
// waiting for one that did). kFewLanes lanes sum a piece of as many tokens, and what runs leave at the pieces' ends meets in shared memory. The other blocks look
// through the ids for those of their kFewRows rows and write zeros into the rest. 1000 tokens of 512, 10000 rows: 12.3 us (with whole warps, so a quarter of
// the blocks, 20.5), in three launches 17.8 and 6 us more of the host's time; 1024 of 4096 with one word in half of the places 13.7 and 16.4.
constexpr uint32_t kFewRows = 128, kFewLanes = 8;
template <int kType, bool kVec, typename Key>
__global__ void __launch_bounds__(kSortChunk) embedding_few_kernel(const __grid_constant__ GradArgs g) {
  using S = Slice<kType, kVec, kFewLanes>;
  using Row = Slice<kType, kVec>;
  constexpr int kUnroll = kVec ? 4 : 2;
  extern __shared__ __align__(16) float ends[];   // [pieces][head, tail][kCols]
  __shared__ Key other[2][kSortChunk];
  __shared__ uint32_t sid[kSortChunk + 1], token[kSortChunk], tail_run[kSortChunk / kFewLanes];
  const uint32_t tid = threadIdx.x, piece = tid / kFewLanes, n = g.tokens;
  auto id_at = [&](const GradTable& t, uint32_t i) { return t.ids != nullptr ? load_index(t.ids, i, t.wide) : static_cast<long long>(i % g.seq); };
  if (blockIdx.x >= g.sums) {
    uint32_t w = blockIdx.x - g.sums;
    int k = 0;
    while (w >= (g.table[k].rows + kFewRows - 1) / kFewRows) w -= static_cast<uint32_t>((g.table[k++].rows + kFewRows - 1) / kFewRows);
    const GradTable& t = g.table[k];
    const long long first = static_cast<long long>(w) * kFewRows;
    if (tid < kFewRows) sid[tid] = 0;
    __syncthreads();
    if (tid < n) {
      const long long id = id_at(t, tid);
      if (id >= first && id < first + kFewRows && id != t.skip) sid[id - first] = 1;
    }
    __syncthreads();
    for (uint32_t r = tid >> 5; r < kFewRows && first + r < t.rows; r += kSortChunk / 32) {
      if (sid[r]) continue;
      const size_t at = wide(static_cast<uint32_t>(first) + r, g.d);
      for (int c = 0; c < g.d; c += Row::kCols) Row::store_zero(t.grad, at + c, g.d - c);
    }
    return;
  }
  const GradTable& t = g.table[blockIdx.x / g.slices];
  const uint32_t c = blockIdx.x % g.slices * S::kCols;
  const int left = g.d - static_cast<int>(c);
  Key key = ~static_cast<Key>(0);
  if (tid < n) {
    const long long id = id_at(t, tid);
    const bool in = id >= 0 && id < t.rows;
    if (!in && c == 0) report_index(g.status, tid);
    key = static_cast<Key>(in && id != t.skip ? static_cast<uint32_t>(id) : kLast<Key>) << kPlaceBits<Key> | tid;
  }
  key = sort_keys(key, other, n);
  sid[tid] = tid < n ? key_id(key) : kNoRow;
  token[tid] = static_cast<uint32_t>(key) & (kSortChunk - 1);
  if (tid == 0) sid[kSortChunk] = kNoRow;
  if (S::lane() == 0) tail_run[piece] = kNoRow;
  __syncthreads();
  const uint32_t begin = piece * kFewLanes;
  float* const head = ends + piece * 2 * S::kCols;
  if (begin < n) {
    uint32_t run = sid[begin];
    bool from_before = begin > 0 && run == sid[begin - 1];
    f32x2 acc[S::kE / 2] = {};
    auto finish = [&](bool goes_on) {
      float f[S::kE];
#pragma unroll
      for (int i = 0; i < S::kE / 2; ++i) {
        upk2(acc[i], f[2 * i], f[2 * i + 1]);
        acc[i] = 0;
      }
      if (run != kNoRow) {
        if (from_before || goes_on) {
          S::store_f32(from_before ? head : head + S::kCols, S::kCols, f);
          if (!from_before && S::lane() == 0) tail_run[piece] = run;
        } else {
#pragma unroll
          for (int i = 0; i < S::kE; ++i) f[i] *= t.scale;
          S::store(t.grad, wide(run, g.d) + c, left, f);
        }
      }
      from_before = false;
    };
    const uint32_t m = min(kFewLanes, n - begin);
    for (uint32_t j0 = 0; j0 < m; j0 += kUnroll) {
      S part[kUnroll];
      uint32_t id[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        id[u] = j0 + u < m ? sid[begin + j0 + u] : kNoRow;
        part[u].load(g.dy, id[u] != kNoRow ? wide(token[begin + j0 + u], g.d) + c : c, left, id[u] != kNoRow);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (j0 + u >= m) break;
        if (id[u] != run) {
          finish(false);
          run = id[u];
        }
        float f[S::kE];
        part[u].get(f);
#pragma unroll
        for (int i = 0; i < S::kE / 2; ++i) acc[i] = add2(acc[i], pk2(f[2 * i], f[2 * i + 1]));
      }
    }
    finish(sid[begin + m] == run);
  }
  __syncthreads();
  const uint32_t run = tail_run[piece];
  if (run == kNoRow) return;
  float acc[S::kE], part[S::kE];
  S::load_f32(head + S::kCols, S::kCols, acc);
  for (uint32_t q = piece + 1; q * kFewLanes < n && sid[q * kFewLanes] == run; ++q) {
    S::load_f32(ends + q * 2 * S::kCols, S::kCols, part);
#pragma unroll
    for (int i = 0; i < S::kE; ++i) acc[i] += part[i];
  }
#pragma unroll
  for (int i = 0; i < S::kE; ++i) acc[i] *= t.scale;
  S::store(t.grad, wide(run, g.d) + c, left, acc);
}

// Sums, then the zeros of the rows that no token has, 32 rows a block. A summing warp takes one piece of the sorted tokens and one slice of the columns.
// Positions come first: their order is known, so these blocks do not wait for the sort, and they leave dy in L2 for the sums by id. Zeros in front of
// the sums, or between them, were no faster (16384 tokens of 1024, 50304 rows: 46 us against 45): blocks that wait hold the places of blocks that could write.
template <int kType, bool kVec>
__global__ void __launch_bounds__(32 * kEmbWarps, 5) embedding_sum_kernel(const __grid_constant__ GradArgs g) {
  using S = Slice<kType, kVec>;
  constexpr int kUnroll = kVec ? 4 : 2;   // 40 warps an SM with four rows in flight: 72 us a pass, 24 with eight 76
  const uint32_t warp = threadIdx.x >> 5;
  if (blockIdx.x >= g.sums) {
    uint32_t w = blockIdx.x - g.sums;
    int k = 0;
    while (w >= (g.table[k].rows + 31) / 32) w -= static_cast<uint32_t>((g.table[k++].rows + 31) / 32);
    const GradTable& t = g.table[k];
    if (t.ids != nullptr) wait_for_previous();
    let_next_in();
    const long long row = static_cast<long long>(w) * 32 + warp * 4 + lane_id();
    bool used = true;
    if (lane_id() < 4 && row < t.rows) {
      if (t.ids == nullptr) {
        used = row < g.seq;
      } else {
        const uint32_t token = __ldcg(t.slot + row);
        used = row != t.skip && token < g.tokens &&
               (t.wide ? __ldcg(reinterpret_cast<const long long*>(t.ids) + token) : __ldcg(reinterpret_cast<const int*>(t.ids) + token)) == row;
      }
    }
    const uint32_t unused = __ballot_sync(0xffffffffu, !used);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (!(unused >> r & 1)) continue;
      const size_t first = wide(w * 32 + warp * 4 + r, g.d);
      for (int c = 0; c < g.d; c += S::kCols) S::store_zero(t.grad, first + c, g.d - c);
    }
    wait_for_previous();   // every block waits before it ends, so that the end of this kernel is the end of those in front of it
    return;
  }
  uint32_t at = blockIdx.x;
  int k = 0;
  while (at >= g.table[k].blocks) at -= g.table[k++].blocks;
  const GradTable& t = g.table[k];
  if (t.ids != nullptr) wait_for_previous();
  let_next_in();
  const uint32_t unit = at * kEmbWarps + warp, piece = unit / g.slices, c = (unit - piece * g.slices) * S::kCols;
  if (piece >= t.pieces) {
    wait_for_previous();
    return;
  }
  const int left = g.d - static_cast<int>(c);
  const uint32_t begin = piece * t.piece, n = min(t.piece, g.tokens - begin);
  const uint64_t mine = lane_id() < n ? key_at(g, t, begin + lane_id()) : ~0ull;
  const uint32_t before = begin > 0 ? id_of(key_at(g, t, begin - 1)) : kNoRow;
  const uint32_t after = begin + n < g.tokens ? id_of(key_at(g, t, begin + n)) : kNoRow;
  f32x2 acc[S::kE / 2] = {};
  uint32_t run = __shfl_sync(0xffffffffu, id_of(mine), 0);
  bool from_before = begin > 0 && run == before;
  auto finish = [&](bool goes_on) {
    float f[S::kE];
#pragma unroll
    for (int i = 0; i < S::kE / 2; ++i) {
      upk2(acc[i], f[2 * i], f[2 * i + 1]);
      acc[i] = 0;
    }
    if (run != kNoRow) {
      if (from_before) {
        S::store_f32(t.head + wide(piece, g.d) + c, left, f);
      } else if (goes_on) {
        S::store_f32(t.tail + wide(piece, g.d) + c, left, f);
        if (c == 0 && lane_id() == 0) {
          wait_for_previous();   // the sorting kernel zeroed the counts
          const uint32_t far = piece + kShort + 1;
          const bool is_long = far < t.pieces && id_of(key_at(g, t, far * t.piece)) == run;
          const int at = atomicAdd(t.count + is_long, 1);
          t.list[is_long ? t.pieces - 1 - at : at] = make_uint2(piece, run);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kE; ++i) f[i] *= t.scale;
        S::store(t.grad, wide(run, g.d) + c, left, f);
      }
    }
    from_before = false;
  };
  for (uint32_t j0 = 0; j0 < n; j0 += kUnroll) {
    S part[kUnroll];
    uint32_t id[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t k = __shfl_sync(0xffffffffu, mine, (j0 + u) & 31);
      id[u] = j0 + u < n ? id_of(k) : kNoRow;
      part[u].load(g.dy, wide(static_cast<uint32_t>(k), g.d) + c, left, id[u] != kNoRow);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (j0 + u >= n) break;
      if (id[u] != run) {
        finish(false);
        run = id[u];
      }
      float f[S::kE];
      part[u].get(f);
#pragma unroll
      for (int i = 0; i < S::kE / 2; ++i) acc[i] = add2(acc[i], pk2(f[2 * i], f[2 * i + 1]));
    }
  }
  finish(after == run);
  wait_for_previous();
}

// Runs that cross pieces: the tail of the piece where the run began, then the heads of those behind it, in their order. Most runs go on for a few pieces:
// a warp adds one up, all of its heads in flight, each read together with the key that says whether it counts. Runs of more than kShort further pieces are for
// a whole block, whose warps take every kJoinWarps-th piece each; their sums are added in the warps' order. Those come first: they take longest.
template <int kType, bool kVec>
__global__ void __launch_bounds__(32 * kJoinWarps) embedding_join_kernel(const __grid_constant__ GradArgs g) {
  using S = Slice<kType, kVec>;
  __shared__ __align__(16) float red[kJoinWarps][S::kCols];
  after_previous();
  const GradTable& t = g.table[blockIdx.y];
  const uint32_t warp = threadIdx.x >> 5, shorts = static_cast<uint32_t>(t.count[0]) * g.slices, longs = static_cast<uint32_t>(t.count[1]) * g.slices;
  auto add_heads = [&](uint32_t q, uint32_t step, uint32_t c, int left, uint32_t run, float (&acc)[S::kE]) {   // of kShort pieces; whether all counted
    float part[kShort][S::kE];
    uint32_t id[kShort];
#pragma unroll
    for (uint32_t u = 0; u < kShort; ++u) {
      const uint32_t p = min(q + u * step, t.pieces - 1);
      id[u] = q + u * step < t.pieces ? id_of(key_at(g, t, p * t.piece)) : kNoRow;
      S::load_f32(t.head + wide(p, g.d) + c, left, part[u]);
    }
    bool on = true;
#pragma unroll
    for (uint32_t u = 0; u < kShort; ++u) {
      on = on && id[u] == run;   // the same id, so the run goes on: what the head's memory holds otherwise is not added
#pragma unroll
      for (int i = 0; i < S::kE; ++i) acc[i] = on ? acc[i] + part[u][i] : acc[i];
    }
    return on;
  };
  for (uint32_t it = blockIdx.x; it < longs; it += gridDim.x) {
    const uint2 what = t.list[t.pieces - 1 - it / g.slices];
    const uint32_t c = it % g.slices * S::kCols;
    const int left = g.d - static_cast<int>(c);
    float acc[S::kE] = {};
    for (uint32_t q = what.x + 1 + warp; q < t.pieces && add_heads(q, kJoinWarps, c, left, what.y, acc); q += kShort * kJoinWarps) {}
    S::store_f32(red[warp], S::kCols, acc);
    __syncthreads();
    for (int j = threadIdx.x; j < S::kCols && j < left; j += 32 * kJoinWarps) {
      float s = t.tail[wide(what.x, g.d) + c + j];
#pragma unroll
      for (int k = 0; k < kJoinWarps; ++k) s += red[k][j];
      store_elem<kType>(t.grad, static_cast<long long>(wide(what.y, g.d) + c + j), s * t.scale);
    }
    __syncthreads();
  }
  // from the other end of the grid
  for (uint32_t it = (gridDim.x - 1 - blockIdx.x) * kJoinWarps + warp; it < shorts; it += gridDim.x * kJoinWarps) {
    const uint2 what = t.list[it / g.slices];
    const uint32_t c = it % g.slices * S::kCols;
    const int left = g.d - static_cast<int>(c);
    float acc[S::kE];
    S::load_f32(t.tail + wide(what.x, g.d) + c, left, acc);
    add_heads(what.x + 1, 1, c, left, what.y, acc);
#pragma unroll
    for (int i = 0; i < S::kE; ++i) acc[i] *= t.scale;
    S::store(t.grad, wide(what.y, g.d) + c, left, acc);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
// Tokens of a piece of the sorted order: 16 (with 32 the pass of the GPT step takes 4 us more, with 8 10). Runs by position are all as long as there are
// sequences: whole ones where they fit.
static uint32_t piece_of(bool sorted, long long batch) {
  return static_cast<uint32_t>(sorted || batch > 32 ? 16 : batch <= 16 ? 16 / batch * batch : batch);
}

static size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// Lays the scratch out; returns its size.
static size_t lay_out(GradTable* t, void* base, long long tokens, long long rows, int d, bool sorted, long long batch) {
  const size_t n = static_cast<size_t>(tokens), piece = piece_of(sorted, batch), pieces = (n + piece - 1) / piece;
  uint8_t* p = static_cast<uint8_t*>(base);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* r = p + at;
    at += up16(bytes);
    return r;
  };
  GradTable x{};
  x.count = reinterpret_cast<int*>(take(8));
  x.list = reinterpret_cast<uint2*>(take(8 * pieces));
  x.head = reinterpret_cast<float*>(take(4 * pieces * d));
  x.tail = reinterpret_cast<float*>(take(4 * pieces * d));
  if (sorted) {
    const size_t chunks = (n + kSortChunk - 1) / kSortChunk;
    x.slot = reinterpret_cast<uint32_t*>(take(4 * static_cast<size_t>(rows)));
    x.keys = reinterpret_cast<uint64_t*>(take(8 * n));
    x.sorted_chunks = reinterpret_cast<uint64_t*>(take(chunks > kSide ? 8 * n : 0));
    x.chunk_ids = reinterpret_cast<uint32_t*>(take(chunks > kSide ? 4 * chunks * kSortChunk : 0));
  }
  if (t != nullptr) {
    t->piece = static_cast<uint32_t>(piece);
    t->pieces = static_cast<uint32_t>(pieces);
    t->count = x.count;
    t->list = x.list;
    t->head = x.head;
    t->tail = x.tail;
    t->slot = x.slot;
    t->sorted_chunks = x.sorted_chunks;
    t->keys = x.keys;
    t->chunk_ids = x.chunk_ids;
  }
  return at;
}

static bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool valid(const CcfEmbed* e) {
  if (e == nullptr || e->tables < 1 || e->tables > CCF_EMBED_TABLES || e->type < 0 || e->type > 2 || e->d < 1 || e->d > CCF_EMBED_MAX_D || e->tokens < 1 ||
      e->tokens > CCF_EMBED_MAX_TOKENS || e->seq < 1 || e->tokens % e->seq != 0)
    return false;
  for (int k = 0; k < e->tables; ++k) {
    const CcfEmbedTable& t = e->table[k];
    if (t.rows < 1 || t.rows > 0x7fffffffll || (t.ids == nullptr && t.rows < e->seq)) return false;
  }
  return true;
}

static cudaError_t launch_behind(void (*kern)(GradArgs), dim3 grid, int threads, cudaStream_t st, int early, const GradArgs& g) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr = early_attribute();
  cfg.attrs = &attr;
  cfg.numAttrs = early;
  return cudaLaunchKernelEx(&cfg, kern, g);
}

template <int kType, bool kVec>
static int launch_fwd(const CcfEmbed& e, void* y, int* status, cudaStream_t st) {
  const uint32_t slices = (e.d + Slice<kType, kVec>::kCols - 1) / Slice<kType, kVec>::kCols;
  uint32_t each = kFwdTokens;
  const int least = 16 * sm_count();
  while (each > 1 && (e.tokens + each - 1) / each * slices < least) each /= 2;   // 16 warps an SM at least, while there are that many
  const long long units = (e.tokens + each - 1) / each * slices, blocks = (units + kEmbWarps - 1) / kEmbWarps;
  if (units > 0xffffff00ll || blocks > 0x7fffffffll) return -2;
  const auto kern = e.tables == 1 ? embedding_fwd_kernel<kType, kVec, 1> : e.tables == 2 ? embedding_fwd_kernel<kType, kVec, 2>
                                                                                        : embedding_fwd_kernel<kType, kVec, 3>;
  kern<<<static_cast<unsigned>(blocks), 32 * kEmbWarps, 0, st>>>(e, y, status, each, slices);
  return launch_result();
}

template <int kType, bool kVec>
static int launch_few(GradArgs& g, cudaStream_t st) {
  using S = Slice<kType, kVec, kFewLanes>;
  long long zeros = 0, largest = 0;
  for (int k = 0; k < g.tables; ++k) {
    zeros += (g.table[k].rows + kFewRows - 1) / kFewRows;
    largest = g.table[k].rows > largest ? g.table[k].rows : largest;
  }
  g.slices = (g.d + S::kCols - 1) / S::kCols;
  g.sums = g.slices * g.tables;
  constexpr int kSmem = kSortChunk / kFewLanes * 2 * S::kCols * 4;
  const bool narrow = largest < kShortRows;
  const auto kern = narrow ? embedding_few_kernel<kType, kVec, uint32_t> : embedding_few_kernel<kType, kVec, uint64_t>;
  static bool configured[64][2] = {};   // per device: the attribute belongs to the (function, device) pair
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63][narrow]) {
    const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return -static_cast<int>(err);
    configured[dev & 63][narrow] = true;
  }
  kern<<<static_cast<unsigned>(g.sums + zeros), kSortChunk, kSmem, st>>>(g);
  const int rc = launch_result();
  return rc == 0 ? 1 : rc;
}

template <int kType, bool kVec>
static int launch_bwd(GradArgs& g, cudaStream_t st) {
  using S = Slice<kType, kVec>;
  g.slices = (g.d + S::kCols - 1) / S::kCols;
  if (g.chunks == 1) return launch_few<kType, kVec>(g, st);
  long long sums = 0, zeros = 0, largest = 0;
  uint32_t most = 0;
  bool sorted = false;
  for (int k = 0; k < g.tables; ++k) {
    GradTable& t = g.table[k];
    const long long units = static_cast<long long>(t.pieces) * g.slices, blocks = (units + kEmbWarps - 1) / kEmbWarps;
    if (units > 0x7fffffffll) return -2;
    t.blocks = static_cast<uint32_t>(blocks);
    sums += blocks;
    zeros += (t.rows + 31) / 32;
    sorted = sorted || t.ids != nullptr;
    largest = t.rows > largest ? t.rows : largest;
    most = t.pieces > most ? t.pieces : most;
  }
  if (sums + zeros > 0x7fffffffll) return -2;
  g.sums = static_cast<uint32_t>(sums);
  const dim3 blocks(static_cast<unsigned>(sums + zeros));
  // kernels set up while the one in front runs: 8192 tokens 57 us, without 68; 16384 46 / 49; at 65536, where a merging kernel runs long beside blocks
  // that wait for it, 77 / 68
  const int may_overlap = g.tokens <= 32768 && early_launches(0, st);
  int launches = 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  while (g.chunks <= kSide && attr.val.clusterDim.x < g.chunks) attr.val.clusterDim.x *= 2;
  cfg.gridDim = dim3(!sorted ? 1 : g.chunks <= kSide ? attr.val.clusterDim.x : g.chunks, g.tables);
  cfg.blockDim = dim3(kSortChunk);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = sorted && attr.val.clusterDim.x > 1 ? 1 : 0;
  cudaError_t err = cudaLaunchKernelEx(&cfg, largest < kShortRows ? embedding_sort_kernel<uint32_t> : embedding_sort_kernel<uint64_t>, g);
  if (err == cudaSuccess && sorted && g.chunks > kSide) {
    err = launch_behind(embedding_merge_kernel, dim3((g.tokens + kMergeThreads - 1) / kMergeThreads, g.tables), kMergeThreads, st, may_overlap, g);
    ++launches;
  }
  if (err == cudaSuccess) err = launch_behind(embedding_sum_kernel<kType, kVec>, blocks, 32 * kEmbWarps, st, may_overlap, g);
  if (err == cudaSuccess && most > 1) {
    const unsigned items = most * g.slices, wave = 2 * sm_count();
    err = launch_behind(embedding_join_kernel<kType, kVec>, dim3(items < wave ? items : wave, g.tables), 32 * kJoinWarps, st, may_overlap, g);
    ++launches;
  }
  return err == cudaSuccess ? launches : -static_cast<int>(err);
}

}  // namespace ccf

extern "C" {

int ccf_sizeof_embed() { return static_cast<int>(sizeof(CcfEmbed)); }

// y [tokens, d] = the sum over the tables of scale * weight[id]. An index out of range is recorded in `status` (code 5, the token) and gives a row
// of NaN. At most 2^26 tokens, 2^31 - 1 rows and 2^24 columns; tokens is a multiple of seq.
int ccf_embedding_fwd(const CcfEmbed* e, void* y, int* status, void* stream) {
  using namespace ccf;
  if (!valid(e) || y == nullptr) return -2;
  const int size = e->type == kFp32 ? 4 : 2;
  bool vec = e->d * size % 16 == 0 && on16(y);
  for (int k = 0; k < e->tables; ++k) {
    if (e->table[k].weight == nullptr || e->table[k].ld < e->d) return -2;
    vec = vec && on16(e->table[k].weight) && e->table[k].ld * size % 16 == 0;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (e->type * 2 + vec) {
    case 0: return launch_fwd<kBf16, false>(*e, y, status, st);
    case 1: return launch_fwd<kBf16, true>(*e, y, status, st);
    case 2: return launch_fwd<kFp16, false>(*e, y, status, st);
    case 3: return launch_fwd<kFp16, true>(*e, y, status, st);
    case 4: return launch_fwd<kFp32, false>(*e, y, status, st);
    default: return launch_fwd<kFp32, true>(*e, y, status, st);
  }
}

// Bytes of scratch that a table needs in ccf_embedding_bwd; sorted: it has ids. None (0) for up to 1024 tokens. -1: a size out of range.
long long ccf_embedding_scratch(long long tokens, long long seq, long long rows, int d, int sorted) {
  if (tokens < 1 || tokens > CCF_EMBED_MAX_TOKENS || seq < 1 || tokens % seq != 0 || rows < 1 || rows > 0x7fffffffll || d < 1 || d > CCF_EMBED_MAX_D) return -1;
  if (tokens <= ccf::kSortChunk) return 0;
  return static_cast<long long>(ccf::lay_out(nullptr, nullptr, tokens, rows, d, sorted != 0, tokens / seq));
}

// grad [rows, d] of every table from dy [tokens, d]: all rows are written, those that no token has with zeros. `scratch` of each table on a
// 16-byte boundary. A token whose index is out of range adds nothing and is recorded in `status`. Returns the number of its launches, or a negative
// code.
int ccf_embedding_bwd(const CcfEmbed* e, const void* dy, int* status, void* stream) {
  using namespace ccf;
  if (!valid(e) || dy == nullptr) return -2;
  const int size = e->type == kFp32 ? 4 : 2;
  GradArgs g{};
  bool vec = e->d * size % 16 == 0 && on16(dy);
  g.dy = dy;
  g.status = status;
  g.tokens = static_cast<uint32_t>(e->tokens);
  g.seq = static_cast<uint32_t>(e->seq);
  g.batch = g.tokens / g.seq;
  g.chunks = (g.tokens + kSortChunk - 1) / kSortChunk;
  g.tables = e->tables;
  g.d = e->d;
  int order[CCF_EMBED_TABLES], n = 0;   // tables without ids first (embedding_sum_kernel)
  for (int sorted = 0; sorted < 2; ++sorted)
    for (int k = 0; k < e->tables; ++k)
      if ((e->table[k].ids != nullptr) == (sorted != 0)) order[n++] = k;
  for (int k = 0; k < e->tables; ++k) {
    const CcfEmbedTable& t = e->table[order[k]];
    if (t.grad == nullptr || (g.chunks > 1 && (t.scratch == nullptr || !on16(t.scratch)))) return -2;
    vec = vec && on16(t.grad);
    GradTable& o = g.table[k];
    if (g.chunks > 1) lay_out(&o, t.scratch, e->tokens, t.rows, e->d, t.ids != nullptr, g.batch);
    o.ids = t.ids;
    o.grad = t.grad;
    o.rows = t.rows;
    o.skip = t.skip;
    o.scale = t.scale;
    o.wide = t.wide;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (e->type * 2 + vec) {
    case 0: return launch_bwd<kBf16, false>(g, st);
    case 1: return launch_bwd<kBf16, true>(g, st);
    case 2: return launch_bwd<kFp16, false>(g, st);
    case 3: return launch_bwd<kFp16, true>(g, st);
    case 4: return launch_bwd<kFp32, false>(g, st);
    default: return launch_bwd<kFp32, true>(g, st);
  }
}

}  // extern "C"
