// Embedding lookup with scaling and position rows, and its gradients.
//
//   out[n] = scale * table[id_n] + positions[n mod T]
//   dtable[v] = scale * sum over {n : id_n = v} of g_n        (zero for the padding id)
//   dpositions[t] = sum over {n : n mod T = t} of g_n
//
// Sums are FP32 and are rounded once.  The table's gradient is dense, so its cost is the write of
// [V, D] plus the read of [N, D].  It is formed in a fixed order without atomics on values:
//
//  1. embedding_sort_kernel: one cluster sorts the pairs (id, position) by id, stable, while all
//     other clusters write the zero rows of ids that do not occur (each reads the ids itself and
//     marks those of its own range, so nobody waits for the sort) and sum the position gradient.
//  2. embedding_sum_kernel: tiles of consecutive sorted pairs; a run of equal ids that lies inside
//     a tile is summed and stored, the pieces of a run that crosses tiles go to a workspace.  The
//     load does not depend on how skewed the ids are.
//  3. embedding_join_kernel: adds those pieces in tile order.
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

// Lanes that share one row (a power of two): a warp serves 32 / lanes narrow rows at once.
inline int embed_lanes(int D) {
  int lanes = 1;
  while (lanes < 32 && lanes * 8 < D) lanes *= 2;
  return lanes;
}

// What a lane owns of a block of 8 * lanes columns.
template <bool VECTOR>
__device__ __forceinline__ int first_column(int block, int lanes, int lane) {
  return VECTOR ? (block * lanes + lane) * 8 : block * lanes * 8 + lane;
}
template <bool VECTOR>
__device__ __forceinline__ int owned_columns(int column, int lanes, int D) {
  if (column >= D) return 0;
  if constexpr (VECTOR) return 8;
  return min(8, (D - column + lanes - 1) / lanes);
}

constexpr int kEmbedThreads = 256;
constexpr int kEmbedBlocks = 4;  // column blocks of one forward unit

template <bool VECTOR>
__global__ void __launch_bounds__(kEmbedThreads)
embedding_fwd_kernel(const EmbedParams p, int lanes) {
  const int lane = threadIdx.x % lanes;
  const int64_t n = (int64_t)blockIdx.x * (kEmbedThreads / lanes) + threadIdx.x / lanes;
  if (n >= p.N) return;
  const int64_t id = load_id(p, n);
  const bool known = id >= 0 && id < p.V;
  const int64_t row = known ? id * p.table_row_stride : 0;
  const int64_t position = p.positions != nullptr ? (n % p.T) * p.position_row_stride : 0;
  Raw8 raw[kEmbedBlocks], add[kEmbedBlocks];
#pragma unroll
  for (int b = 0; b < kEmbedBlocks; ++b) {
    const int column = first_column<VECTOR>(blockIdx.y * kEmbedBlocks + b, lanes, lane);
    const int count = owned_columns<VECTOR>(column, lanes, p.D);
    if (count > 0) {
      if (known) raw[b] = load_raw8<VECTOR>(p.table, p.table_type, row + column, lanes, count);
      if (p.positions != nullptr)
        add[b] = load_raw8<VECTOR>(p.positions, p.position_type, position + column, lanes, count);
    }
  }
#pragma unroll
  for (int b = 0; b < kEmbedBlocks; ++b) {
    const int column = first_column<VECTOR>(blockIdx.y * kEmbedBlocks + b, lanes, lane);
    const int count = owned_columns<VECTOR>(column, lanes, p.D);
    if (count > 0) {
      float f[8], q[8];
      if (known) {
        unpack_raw8(raw[b], p.table_type, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= p.scale;
      } else {
        // No such row: not a number, so that a wrong id cannot pass unseen.
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __int_as_float(0x7fc00000);
      }
      if (p.positions != nullptr) {
        unpack_raw8(add[b], p.position_type, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += q[e];
      }
      store8<VECTOR>(p.out, p.out_type, n * p.D + column, lanes, count, f);
    }
  }
}

// ------------------------------------------------------------------------------ gradient, step 1

constexpr int kSortCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxDigitBits = 9;
constexpr int kSortDigits = 1 << kSortMaxDigitBits;
// Per-warp digit counts, the CTA's totals and the digits' first places; the other clusters use
// the same bytes as the bitmap of their range of ids.
constexpr uint32_t kSortSmem = (kSortWarps + 2) * kSortDigits * 4 + 64;
constexpr int kSortMaxRange = (int)(kSortSmem - 64) * 8;  // ids a bitmap holds

// Stable radix sort of (id, position) by one cluster.  Every warp owns a contiguous share of the
// sequence; a digit's places are ordered by warp, and inside a warp by sequence order.
__device__ inline void sort_pairs(const EmbedParams& p, uint32_t* smem) {
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

template <bool VECTOR>
__global__ void __cluster_dims__(kSortCluster, 1, 1) __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const EmbedParams p, int element_bytes) {
  extern __shared__ uint32_t sort_smem[];
  const int tid = threadIdx.x;
  if (blockIdx.x < kSortCluster) {
    if (p.dtable != nullptr) sort_pairs(p, sort_smem);
    return;
  }
  const int helper = blockIdx.x - kSortCluster, helpers = gridDim.x - kSortCluster;
  if (p.dpositions != nullptr) {
    const int chunks = (p.D + 7) / 8;
    const int64_t items = p.T * chunks, batch = p.N / p.T;
    for (int64_t i = (int64_t)helper * kSortThreads + tid; i < items;
         i += (int64_t)helpers * kSortThreads) {
      const int64_t t = i / chunks;
      const int column = (int)(i % chunks) * 8, count = min(8, p.D - column);
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int64_t b = 0; b < batch; ++b) {
        float f[8];
        unpack_raw8(load_raw8<VECTOR>(p.grad, p.out_type,
                                      (b * p.T + t) * p.grad_row_stride + column, 1, count),
                    p.out_type, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += f[e];
      }
      store8<VECTOR>(p.dpositions, p.position_type, t * p.D + column, 1, count, sum);
    }
  }
  if (p.dtable == nullptr) return;
  // Ids [low, high) are this CTA's; a bit is set for those that have a gradient.
  const int64_t low = (int64_t)p.V * helper / helpers, high = (int64_t)p.V * (helper + 1) / helpers;
  const int range = (int)(high - low), words = (range + 31) / 32;
  for (int i = tid; i < words; i += kSortThreads) sort_smem[i] = 0u;
  __syncthreads();
#pragma unroll 4
  for (int64_t n = tid; n < p.N; n += kSortThreads) {
    const int64_t key = (int64_t)gradient_key(p, n) - low;
    if (key >= 0 && key < range) atomicOr(&sort_smem[key >> 5], 1u << (key & 31));
  }
  __syncthreads();
  const int64_t row_bytes = (int64_t)p.D * element_bytes;
  for (int v = tid >> 5; v < range; v += kSortWarps) {
    if (!((sort_smem[v >> 5] >> (v & 31)) & 1u))
      zero_row(static_cast<char*>(p.dtable) + (low + v) * row_bytes, row_bytes, tid & 31);
  }
}

// ------------------------------------------------------------------------------ gradient, step 2

constexpr int kSumBatch = 8;  // rows in flight per lane

template <bool VECTOR>
__global__ void __launch_bounds__(kEmbedThreads)
embedding_sum_kernel(const EmbedParams p, int lanes, int blocks, int64_t tiles) {
  const int lane = threadIdx.x % lanes;
  const int64_t unit = (int64_t)blockIdx.x * (kEmbedThreads / lanes) + threadIdx.x / lanes;
  const int64_t tile = unit / blocks;
  const int column = first_column<VECTOR>((int)(unit % blocks), lanes, lane);
  const int count = owned_columns<VECTOR>(column, lanes, p.D);
  if (tile >= tiles || count == 0) return;
  const uint2* pairs = p.pairs[(p.passes - 1) & 1];
  const uint32_t nothing = (uint32_t)p.V;
  const int64_t begin = tile * p.tile, end = min(p.N, begin + p.tile);
  const uint32_t before = begin > 0 ? __ldg(&pairs[begin - 1].x) : nothing;
  const uint32_t after = end < p.N ? __ldg(&pairs[end].x) : nothing;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  uint32_t current = __ldg(&pairs[begin].x);
  bool leading = current == before;  // the run began in an earlier tile
  auto finish = [&](bool continues) {
    if (current == nothing) return;
    if (!leading && !continues) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] *= p.scale;
      store8<VECTOR>(p.dtable, p.table_type, (int64_t)current * p.D + column, lanes, count, sum);
    } else {
      store8<VECTOR>(p.pieces, ATTNRES_B200_FP32, (2 * tile + (leading ? 0 : 1)) * p.D + column,
                     lanes, count, sum);
    }
  };
  for (int64_t i = begin; i < end; i += kSumBatch) {
    uint2 pair[kSumBatch];
    Raw8 raw[kSumBatch];
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k)
      pair[k] = i + k < end ? __ldg(pairs + i + k) : make_uint2(nothing, 0u);
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k)
      if (pair[k].x != nothing)
        raw[k] = load_raw8<VECTOR>(p.grad, p.out_type,
                                   (int64_t)pair[k].y * p.grad_row_stride + column, lanes, count);
#pragma unroll
    for (int k = 0; k < kSumBatch; ++k) {
      if (i + k < end) {
        if (pair[k].x != current) {
          finish(false);
          current = pair[k].x;
          leading = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] = 0.f;
        }
        if (current != nothing) {
          float f[8];
          unpack_raw8(raw[k], p.out_type, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
      }
    }
  }
  finish(current == after);
}

// ------------------------------------------------------------------------------ gradient, step 3

template <bool VECTOR>
__global__ void __launch_bounds__(kEmbedThreads)
embedding_join_kernel(const EmbedParams p, int lanes, int blocks, int64_t tiles) {
  const int lane = threadIdx.x % lanes;
  const int64_t unit = (int64_t)blockIdx.x * (kEmbedThreads / lanes) + threadIdx.x / lanes;
  const int64_t tile = unit / blocks;
  const int column = first_column<VECTOR>((int)(unit % blocks), lanes, lane);
  const int count = owned_columns<VECTOR>(column, lanes, p.D);
  if (tile >= tiles - 1 || count == 0) return;
  const uint2* pairs = p.pairs[(p.passes - 1) & 1];
  const int64_t begin = tile * p.tile, end = begin + p.tile;  // a tile follows, so this one is full
  const uint32_t id = __ldg(&pairs[end - 1].x);
  if (id == (uint32_t)p.V || __ldg(&pairs[end].x) != id) return;
  // Only the tile in which the run begins joins it.
  if (begin > 0 && __ldg(&pairs[begin].x) == id && __ldg(&pairs[begin - 1].x) == id) return;
  float sum[8], f[8];
  unpack_raw8(load_raw8<VECTOR>(p.pieces, ATTNRES_B200_FP32, (2 * tile + 1) * p.D + column, lanes,
                                count),
              ATTNRES_B200_FP32, sum);
  int64_t next = tile + 1;
  while (next < tiles) {
    bool in_run[4];
    Raw8 raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      in_run[k] = next + k < tiles && __ldg(&pairs[(next + k) * p.tile].x) == id;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (in_run[k])
        raw[k] = load_raw8<VECTOR>(p.pieces, ATTNRES_B200_FP32, 2 * (next + k) * p.D + column, lanes,
                                   count);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (in_run[k]) {
        unpack_raw8(raw[k], ATTNRES_B200_FP32, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += f[e];
      }
    }
    if (!in_run[3]) break;
    next += 4;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] *= p.scale;
  store8<VECTOR>(p.dtable, p.table_type, (int64_t)id * p.D + column, lanes, count, sum);
}

}  // namespace attnres_b200
