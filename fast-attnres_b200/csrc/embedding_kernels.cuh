// Embedding lookup with scaling and position rows, and its gradients.
//
//   out[n] = scale * table[id_n] + positions[n mod T]
//   dtable[v] = scale * sum over {n : id_n = v} of g_n        (zero for the padding id)
//   dpositions[t] = sum over {n : n mod T = t} of g_n
//
// Sums are FP32 and are rounded once.  The table's gradient is dense, so its cost is the write of
// [V, D] plus the read of [N, D].  It is formed in a fixed order without atomics on values:
//
//  1. embedding_sort_kernel: one cluster sorts the pairs (id, position) by id, stable.  Beside it
//     runs embedding_early_kernel with what needs nothing of the sort: the zero rows of ids that do
//     not occur (its CTAs read the ids themselves and mark those of their own range) and the
//     position gradient.
//  2. embedding_sum_kernel: tiles of consecutive sorted pairs; a run of equal ids that lies inside
//     a tile is summed and stored, the pieces of a run that crosses tiles go to a workspace.  The
//     load does not depend on how skewed the ids are.
//  3. embedding_join_kernel: adds those pieces in tile order.
//
// Up to kFewTokens tokens take one launch instead, without a sort.
//
// Measured, 16 384 ids of 32 000: lookup 47 us at 4096 BF16 columns with positions (6.4 TB/s);
// gradients 57 us at 1024 FP32 columns and 124 us at 4096 BF16 ones, positions included, where the
// writing alone (139 and 295 MB at 3.8 TB/s, what memory takes without reads) is 37 and 78 us.  The
// sort takes 20 us (13 us for up to a thousand ids, 158 us for 262 144), hidden behind the zeros.
#pragma once

#include <cooperative_groups.h>

#include "typed_access.cuh"

namespace attnres_b200 {

struct EmbedParams {
  const void* tokens;
  int32_t tokens_64;  // 8-byte ids, else 4-byte
  int32_t V;
  int64_t N;
  int64_t T;        // positions repeat with this period
  int64_t padding;  // id without gradient, or -1
  int32_t D;
  float scale;
  const void* table;  // forward
  int64_t table_row_stride;
  int32_t table_type;
  const void* positions;  // forward, may be NULL
  int64_t position_row_stride;
  int32_t position_type;
  void* out;  // forward [N,D] contiguous
  int32_t out_type;
  // backward
  const void* grad;  // [N,D], type out_type
  int64_t grad_row_stride;
  void* dtable;      // [V,D] contiguous, type table_type; may be NULL
  void* dpositions;  // [T,D] contiguous, type position_type; may be NULL
  uint2* pairs[2];   // (id or V, position), ping-pong
  int32_t passes, digit_bits;
  int32_t tile;      // sorted pairs of a tile
  float* pieces;     // [tiles][2][D]: leading and trailing run of a tile
  int32_t* runs;     // how many runs cross tiles, then the tiles they begin in
};

__device__ __forceinline__ int64_t load_id(const EmbedParams& p, int64_t n) {
  return p.tokens_64 ? __ldg(static_cast<const long long*>(p.tokens) + n)
                     : (int64_t)__ldg(static_cast<const int*>(p.tokens) + n);
}

// The id under which a token's gradient is collected; V collects what has no gradient.
__device__ __forceinline__ uint32_t gradient_key(const EmbedParams& p, int64_t n) {
  const int64_t id = load_id(p, n);
  return (id < 0 || id >= p.V || id == p.padding) ? (uint32_t)p.V : (uint32_t)id;
}

// What a lane owns of a block of columns: eight neighbours where rows allow 16-byte accesses, else
// `elements` of them `lanes` apart.
struct Columns {
  int lanes;   // that share one row (a power of two); a warp serves 32 / lanes narrow rows at once
  int blocks;  // of lanes * elements columns
};

inline Columns columns_of(int D, int elements) {
  Columns c{1, 0};
  while (c.lanes < 32 && c.lanes * elements < D) c.lanes *= 2;
  c.blocks = (D + c.lanes * elements - 1) / (c.lanes * elements);
  return c;
}

template <bool VECTOR, int E>
__device__ __forceinline__ int first_column(int block, int lanes, int lane) {
  return VECTOR ? (block * lanes + lane) * 8 : block * lanes * E + lane;
}
template <bool VECTOR, int E>
__device__ __forceinline__ int owned_columns(int column, int lanes, int D) {
  if (column >= D) return 0;
  if constexpr (VECTOR) return 8;
  int count = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) count += column + e * lanes < D;
  return count;
}

constexpr int kEmbedThreads = 256;
constexpr int kEmbedBlocks = 4;  // column blocks of one forward unit

// Columns a lane of the gradient's kernels owns.  A warp sums a tile of 32 pairs in one block of
// columns, one row after the other; element by element eight columns would leave too few warps and
// too many instructions to each (6185 ids of 1001 columns: 38 us with eight, 16 us with two).
template <bool VECTOR>
__host__ __device__ constexpr int gradient_columns() {
  return VECTOR ? 8 : 2;
}

enum EmbedPositions { kNoPositions, kNarrowPositions, kWidePositions };

template <bool VECTOR, bool WIDE, int POSITIONS>
__global__ void __launch_bounds__(kEmbedThreads)
embedding_fwd_kernel(const EmbedParams p, int lanes) {
  constexpr bool kAdd = POSITIONS != kNoPositions, kAddWide = POSITIONS == kWidePositions;
  const int lane = threadIdx.x % lanes;
  const int64_t n = (int64_t)blockIdx.x * (kEmbedThreads / lanes) + threadIdx.x / lanes;
  if (n >= p.N) return;
  const int64_t id = load_id(p, n);
  const bool known = id >= 0 && id < p.V;
  const int64_t row = known ? id * p.table_row_stride : 0;
  const int64_t position = kAdd ? (n % p.T) * p.position_row_stride : 0;
  Share<VECTOR, WIDE> raw[kEmbedBlocks];
  Share<VECTOR, kAddWide> add[kAdd ? kEmbedBlocks : 1];
#pragma unroll
  for (int b = 0; b < kEmbedBlocks; ++b) {
    const int column = first_column<VECTOR, 8>(blockIdx.y * kEmbedBlocks + b, lanes, lane);
    const int count = owned_columns<VECTOR, 8>(column, lanes, p.D);
    if (count > 0) {
      raw[b].load(p.table, row + column, lanes, count);
      if constexpr (kAdd) add[b].load(p.positions, position + column, lanes, count);
    }
  }
#pragma unroll
  for (int b = 0; b < kEmbedBlocks; ++b) {
    const int column = first_column<VECTOR, 8>(blockIdx.y * kEmbedBlocks + b, lanes, lane);
    const int count = owned_columns<VECTOR, 8>(column, lanes, p.D);
    if (count > 0) {
      float f[8], q[8];
      raw[b].unpack(p.table_type, f);
      // No such row (row 0 was read in its place): not a number, so that a wrong id cannot pass
      // unseen.
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = known ? f[e] * p.scale : __int_as_float(0x7fc00000);
      if constexpr (kAdd) {
        add[b].unpack(p.position_type, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += q[e];
      }
      store_share<VECTOR>(p.out, p.out_type, n * p.D + column, lanes, count, f);
    }
  }
}

// ------------------------------------------------------------------------------ gradient, step 1

constexpr int kSortCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxDigitBits = 9;
constexpr int kSortDigits = 1 << kSortMaxDigitBits;
// Per-warp digit counts, the CTA's totals and the digits' first places.
constexpr uint32_t kSortSmem = (kSortWarps + 2) * kSortDigits * 4 + 64;

// Stable radix sort of (id, position) by one cluster.  Every warp owns a contiguous share of the
// sequence; a digit's places are ordered by warp, and inside a warp by sequence order.
__global__ void __cluster_dims__(kSortCluster, 1, 1) __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const EmbedParams p) {
  // The kernel beside this one may start at once; it waits for this one before it ends.
  start_next_kernel();
  extern __shared__ uint32_t smem[];
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t* counts = smem;                                // [warps][digits]
  uint32_t* totals = smem + kSortWarps * kSortDigits;     // [digits], read by the peers
  uint32_t* places = totals + kSortDigits;                // [digits]
  uint32_t* warp_sums = places + kSortDigits;             // [16]
  const int64_t share = ((p.N + kSortCluster * kSortWarps * 32 - 1) /
                         (kSortCluster * kSortWarps * 32)) * 32;
  const int64_t begin = min(p.N, (int64_t)(rank * kSortWarps + warp) * share);
  const int64_t end = min(p.N, begin + share);
  uint32_t* my_counts = counts + warp * kSortDigits;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit_bits;
    const uint32_t mask = (1u << p.digit_bits) - 1u;
    const uint2* src = p.pairs[(pass + 1) & 1];  // pass 0 reads the ids themselves
    uint2* dst = p.pairs[pass & 1];
    for (int i = tid; i < kSortWarps * kSortDigits; i += kSortThreads) counts[i] = 0u;
    __syncthreads();
    for (int64_t i = begin + lane; i < end; i += 32) {
      const uint32_t key = pass == 0 ? gradient_key(p, i) : __ldcg(src + i).x;
      atomicAdd(&my_counts[(key >> shift) & mask], 1u);
    }
    __syncthreads();
    if (tid < kSortDigits) {  // exclusive over the CTA's warps
      uint32_t run = 0u;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = counts[w * kSortDigits + tid];
        counts[w * kSortDigits + tid] = run;
        run += c;
      }
      totals[tid] = run;
    }
    cluster.sync();
    uint32_t below = 0u, all = 0u, inclusive = 0u;
    if (tid < kSortDigits) {
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        const uint32_t v = cluster.map_shared_rank(totals, c)[tid];
        if (c < rank) below += v;
        all += v;
      }
      inclusive = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += v;
      }
      if (lane == 31) warp_sums[warp] = inclusive;
    }
    __syncthreads();
    if (tid < kSortDigits) {
      uint32_t before = 0u;
      for (int w = 0; w < warp; ++w) before += warp_sums[w];
      places[tid] = before + inclusive - all + below;
    }
    __syncthreads();
    for (int64_t first = begin; first < end; first += 32) {
      const int64_t i = first + lane;
      const uint32_t live = __ballot_sync(0xffffffffu, i < end);
      if (i < end) {
        uint2 pair;
        if (pass == 0) pair = make_uint2(gradient_key(p, i), (uint32_t)i);
        else pair = __ldcg(src + i);
        const uint32_t digit = (pair.x >> shift) & mask;
        const uint32_t peers = __match_any_sync(live, digit);
        const int leader = __ffs(peers) - 1;
        uint32_t place = 0u;
        if (lane == leader) {
          place = my_counts[digit];
          my_counts[digit] = place + __popc(peers);
        }
        place = __shfl_sync(peers, place, leader) + __popc(peers & ((1u << lane) - 1u));
        __stcg(dst + places[digit] + place, pair);
      }
      __syncwarp();
    }
    // Orders this pass's stores before the next one's loads (and the peers' reads of `totals`
    // before they are overwritten), cluster-wide.
    cluster.sync();
  }
}

// Zeroes [0, bytes) of a row with one warp, whatever its alignment.
__device__ __forceinline__ void zero_row(char* row, int64_t bytes, int lane) {
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15));
  const int64_t body = (bytes - head) / 16, tail = head + body * 16;
  for (int64_t i = lane * 2; i < head; i += 64) *reinterpret_cast<unsigned short*>(row + i) = 0;
  uint4* aligned = reinterpret_cast<uint4*>(row + head);
  for (int64_t i = lane; i < body; i += 32) aligned[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = tail + lane * 2; i < bytes; i += 64) *reinterpret_cast<unsigned short*>(row + i) = 0;
}

constexpr int kFillWords = 1024;  // bitmap of the ids a CTA fills
constexpr int kFillRange = kFillWords * 32;

constexpr int kPositionBatch = 4;  // sequences whose rows a thread has in flight
constexpr int kEarlyThreads = 256;

// Up to this many tokens are not sorted: a warp finds those of its id by comparing all of them, and
// one launch does everything.  128 tokens of 300 ids, 4096 BF16 columns: 3.5 us against 13.9 with the
// sort; 8 of 1988 ids, 264 columns: 3.2 against 11.1.  The longest sum is a single id's, by one warp
// for its columns: 15.0 against 14.0 us with 128 tokens, 32 against 14 with 256.
constexpr int64_t kFewTokens = 128;

// The gradient row of token n's id in one block of columns, by the warp of the id's first token.
template <bool VECTOR, bool WIDE>
__device__ __forceinline__ void sum_few(const EmbedParams& p, int n, int block) {
  constexpr int E = gradient_columns<VECTOR>(), kWords = (int)kFewTokens / 32;
  constexpr int kBatch = !VECTOR ? 16 : WIDE ? 4 : 8;  // rows in flight
  const int lane = threadIdx.x & 31;
  const uint32_t nothing = (uint32_t)p.V, id = gradient_key(p, n);
  if (id == nothing) return;
  uint32_t keys[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j)
    keys[j] = j * 32 + lane < p.N ? gradient_key(p, j * 32 + lane) : nothing;
  const int column = first_column<VECTOR, E>(block, 32, lane);
  const int count = owned_columns<VECTOR, E>(column, 32, p.D);
  float sum[E] = {};
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    uint32_t same = __ballot_sync(0xffffffffu, keys[j] == id);
    if (same != 0u && j * 32 + __ffs(same) - 1 < n) return;  // the whole warp: not the first
    while (same != 0u) {
      Share<VECTOR, WIDE, E> raw[kBatch];
      uint32_t left = same;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (left != 0u && count > 0)
          raw[k].load(p.grad, (int64_t)(j * 32 + __ffs(left) - 1) * p.grad_row_stride + column, 32, count);
        left &= left - 1u;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (same != 0u) {
          float f[E];
          raw[k].unpack(p.out_type, f);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += f[e];
        }
        same &= same - 1u;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] *= p.scale;
  if (count > 0)
    store_share<VECTOR, E>(p.dtable, p.table_type, (int64_t)id * p.D + column, 32, count, sum);
}

// CTAs [0, fill_ctas) write the zero rows of a range of ids each, the others the position gradient.
// FEW: `sum_ctas` before them write the rows of the ids that occur, which makes it the whole backward.
template <bool VECTOR, bool WIDE, bool FEW>
__global__ void __launch_bounds__(kEarlyThreads, VECTOR && !FEW ? 5 : 3)
embedding_early_kernel(const EmbedParams p, int element_bytes, int fill_ctas, int sum_ctas) {
  __shared__ uint32_t used[kFillWords];
  const int tid = threadIdx.x;
  const int cta = (int)blockIdx.x - sum_ctas;
  if (FEW && cta < 0) {
    constexpr int kColumns = 32 * gradient_columns<VECTOR>();
    const int warp = blockIdx.x * (kEarlyThreads / 32) + tid / 32, blocks = (p.D + kColumns - 1) / kColumns;
    if (warp < p.N * blocks) sum_few<VECTOR, WIDE>(p, warp / blocks, warp % blocks);
  } else if (cta < fill_ctas) {
    // Ids [low, low + range) are this CTA's; a bit is set for those that have a gradient.
    const int64_t low = (int64_t)p.V * cta / fill_ctas;
    const int range = (int)((int64_t)p.V * (cta + 1) / fill_ctas - low);
    for (int i = tid; i < (range + 31) / 32; i += kEarlyThreads) used[i] = 0u;
    __syncthreads();
#pragma unroll 8
    for (int64_t n = tid; n < p.N; n += kEarlyThreads) {
      const int64_t key = (int64_t)gradient_key(p, n) - low;
      if (key >= 0 && key < range) atomicOr(&used[key >> 5], 1u << (key & 31));
    }
    __syncthreads();
    const int64_t row_bytes = (int64_t)p.D * element_bytes;
    for (int v = tid >> 5; v < range; v += kEarlyThreads / 32) {
      if (!((used[v >> 5] >> (v & 31)) & 1u))
        zero_row(static_cast<char*>(p.dtable) + (low + v) * row_bytes, row_bytes, tid & 31);
    }
  } else {
    const int chunks = (p.D + 7) / 8;
    const int64_t items = p.T * chunks, batch = p.N / p.T;
    const int64_t i = (int64_t)(cta - fill_ctas) * kEarlyThreads + tid;
    if (i < items) {
      const int64_t t = i / chunks;
      const int column = (int)(i - t * chunks) * 8, count = min(8, p.D - column);
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int64_t b = 0; b < batch; b += kPositionBatch) {
        Share<VECTOR, WIDE> raw[kPositionBatch];
#pragma unroll
        for (int k = 0; k < kPositionBatch; ++k)
          if (b + k < batch)
            raw[k].load(p.grad, ((b + k) * p.T + t) * p.grad_row_stride + column, 1, count);
#pragma unroll
        for (int k = 0; k < kPositionBatch; ++k) {
          if (b + k < batch) {
            float f[8];
            raw[k].unpack(p.out_type, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
          }
        }
      }
      store_share<VECTOR>(p.dpositions, p.position_type, t * p.D + column, 1, count, sum);
    }
  }
  // What follows in the stream waits for this kernel, and through this also for the sort.
  if constexpr (!FEW) wait_for_previous_kernel();
}

// ------------------------------------------------------------------------------ gradient, step 2

constexpr int kJoinBatch = 8;  // pieces in flight per lane

// Small CTAs: registers (102) allow five to an SM, 640 threads against 512 in CTAs of 256, and the
// last ones end closer together.
constexpr int kSumThreads = 128;

template <bool VECTOR, bool WIDE>
__global__ void __launch_bounds__(kSumThreads)
embedding_sum_kernel(const EmbedParams p, int lanes, int blocks, int64_t tiles) {
  start_next_kernel();  // the joining waits for the end
  constexpr int E = gradient_columns<VECTOR>();
  constexpr int kSumBatch = VECTOR ? 8 : 16;  // rows in flight per lane
  const int lane = threadIdx.x % lanes;
  const int64_t unit = (int64_t)blockIdx.x * (kSumThreads / lanes) + threadIdx.x / lanes;
  const int64_t tile = unit / blocks;
  const int column = first_column<VECTOR, E>((int)(unit % blocks), lanes, lane);
  const int count = owned_columns<VECTOR, E>(column, lanes, p.D);
  if (tile >= tiles || count == 0) return;
  const uint2* pairs = p.pairs[(p.passes - 1) & 1];
  const uint32_t nothing = (uint32_t)p.V;
  const int64_t begin = tile * p.tile, end = min(p.N, begin + p.tile);
  const uint32_t before = begin > 0 ? __ldg(&pairs[begin - 1].x) : nothing;
  const uint32_t after = end < p.N ? __ldg(&pairs[end].x) : nothing;
  float sum[E] = {};
  uint32_t current = __ldg(&pairs[begin].x);
  bool leading = current == before;  // the run began in an earlier tile
  auto finish = [&](bool continues) {
    if (current == nothing) return;
    if (!leading && !continues) {
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] *= p.scale;
      store_share<VECTOR, E>(p.dtable, p.table_type, (int64_t)current * p.D + column, lanes, count, sum);
    } else {
      store_share<VECTOR, E>(p.pieces, ATTNRES_B200_FP32, (2 * tile + (leading ? 0 : 1)) * p.D + column,
                     lanes, count, sum);
    }
  };
  uint2 next[kSumBatch];
  auto fetch = [&](int64_t i) {
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k)
      next[k] = i + k < end ? __ldg(pairs + i + k) : make_uint2(nothing, 0u);
  };
  fetch(begin);
  for (int64_t i = begin; i < end; i += kSumBatch) {
    uint2 pair[kSumBatch];
    Share<VECTOR, WIDE, E> raw[kSumBatch];
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k) pair[k] = next[k];
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k)
      if (pair[k].x != nothing)
        raw[k].load(p.grad, (int64_t)pair[k].y * p.grad_row_stride + column, lanes, count);
    fetch(i + kSumBatch);
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k) {
      if (i + k < end) {
        if (pair[k].x != current) {
          finish(false);
          current = pair[k].x;
          leading = false;
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] = 0.f;
        }
        if (current != nothing) {
          float f[E];
          raw[k].unpack(p.out_type, f);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += f[e];
        }
      }
    }
  }
  const bool continues = current == after && current != nothing;
  finish(continues);
  // A run that begins here and goes on: one of the kernel's units puts it on the list to join.
  if (continues && !leading && column == 0) p.runs[1 + atomicAdd(p.runs, 1)] = (int32_t)tile;
}

// ------------------------------------------------------------------------------ gradient, step 3

// A warp joins the pieces of one run in one block of columns.  (The order of the list is not fixed,
// but each run is joined on its own, in tile order.)
template <bool VECTOR>
__global__ void __launch_bounds__(kEmbedThreads)
embedding_join_kernel(const EmbedParams p, int lanes, int blocks, int64_t tiles) {
  wait_for_previous_kernel();
  constexpr int E = gradient_columns<VECTOR>();
  const int lane = threadIdx.x & 31;
  const uint2* pairs = p.pairs[(p.passes - 1) & 1];
  const int64_t units = (int64_t)__ldcg(p.runs) * blocks;
  for (int64_t unit = (int64_t)blockIdx.x * (kEmbedThreads / 32) + threadIdx.x / 32; unit < units;
       unit += (int64_t)gridDim.x * (kEmbedThreads / 32)) {
    const int64_t tile = __ldcg(p.runs + 1 + unit / blocks);
    const uint32_t id = __ldg(&pairs[(tile + 1) * p.tile].x);
    int64_t last = tile;  // the last tile that holds a piece
    while (true) {
      const int64_t other = last + 1 + lane;
      const bool in_run = other < tiles && __ldg(&pairs[min(other, tiles - 1) * p.tile].x) == id;
      const uint32_t votes = __ballot_sync(0xffffffffu, in_run);
      last += __popc(votes);
      if (votes != 0xffffffffu) break;
    }
    const int column = first_column<VECTOR, E>((int)(unit % blocks), lanes, lane);
    const int count = lane < lanes ? owned_columns<VECTOR, E>(column, lanes, p.D) : 0;
    if (count == 0) continue;
    float sum[E], f[E];
    Share<VECTOR, true, E> start;
    start.load(p.pieces, (2 * tile + 1) * p.D + column, lanes, count);
    start.unpack(ATTNRES_B200_FP32, sum);
    for (int64_t next = tile + 1; next <= last; next += kJoinBatch) {
      Share<VECTOR, true, E> raw[kJoinBatch];
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k)
        if (next + k <= last) raw[k].load(p.pieces, 2 * (next + k) * p.D + column, lanes, count);
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        if (next + k <= last) {
          raw[k].unpack(ATTNRES_B200_FP32, f);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += f[e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] *= p.scale;
    store_share<VECTOR, E>(p.dtable, p.table_type, (int64_t)id * p.D + column, lanes, count, sum);
  }
}

}  // namespace attnres_b200
