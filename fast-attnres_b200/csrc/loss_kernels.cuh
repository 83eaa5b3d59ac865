// Softmax cross entropy of z = scale * H W^T against target ids, without keeping z.
//
//   lse_n = log sum_v exp(z_nv)          loss_n = lse_n - z_n,target
//   P_nv  = c_n (exp(z_nv - lse_n) - [v = target_n])     c_n: what the loss of row n weighs
//   dH    = scale P W                    dW = scale P^T H
//
// Every product runs on the tensor cores with FP32 accumulators:
//   kStats      tiles of z in tensor memory, reduced at once to a (max, sum) pair per row and half
//               tile; a second kernel joins the pairs.  z never leaves the SM.
//   kProbs      the same tiles again, turned into P (16-bit, the inputs' type) for one piece of
//               the vocabulary;
//   kGradients  dH from the piece and the piece's rows of dW, in one launch.
// The backward forms z a second time: that costs a quarter of the training pass's products and no
// memory.  Where the loss is one number, its gradients are known up to that number's upstream
// gradient, and the forward can form them at once, from one z (kCodes instead of kStats):
//   kCodes      a piece of the rows: (max, sum) pairs as above, and z as 16-bit codes, the distance
//               from the half tile's maximum in steps of 2^-11 powers of two (a probability is off
//               by 2^-12.5 at most, an eighth of what P's own rounding to BF16 allows);
//   loss_probs_kernel turns the codes into P in place once the rows' sums are known.
//
// Rows whose target is the ignored id take no part: the kept rows are first gathered into
// consecutive ones (their number stays on the device), so padding costs no products and whatever
// an ignored row holds, infinities included, reaches no result.
#pragma once

#include "tcgen05.cuh"
#include "typed_access.cuh"

namespace attnres_b200 {

// ------------------------------------------------------------------------------ gathering rows

struct GatherParams {
  const void* hidden;       // 16-bit [N, D], feature stride 1
  int64_t hidden_row_stride;
  const void* targets;
  int32_t targets_64;
  int64_t N;
  int32_t D, Dp;            // Dp: D rounded up to eight
  int32_t V;
  int64_t ignored;
  int32_t block_rows;
  unsigned short* kept;     // [N, Dp]: the kept rows, zeros up to the next multiple of 128 rows
  int32_t* kept_index;      // [N]: their rows in the input
  int32_t* kept_target;     // [N]: their targets, -1 when outside the vocabulary
  int32_t* count;
  float* target_logit;      // [N], to be filled in by the products
  float* losses;            // [N]: zero for ignored rows
  // The gradients' common scale for an upstream gradient of one, and dH, whose ignored rows are
  // zeroed; NULL where the forward forms no gradients.
  float* gradient_scale;
  int32_t mean;
  unsigned short* dhidden;
};

__device__ __forceinline__ int64_t load_target(const void* targets, int wide, int64_t n) {
  return wide ? __ldg(static_cast<const long long*>(targets) + n)
              : (int64_t)__ldg(static_cast<const int*>(targets) + n);
}

// Eight 16-bit elements from any even address, `count` of them in the row: words where the address
// allows, so that nothing beyond the elements is read.  The rest are zeros.
__device__ __forceinline__ uint4 load_eight(const unsigned short* src, int count) {
  uint32_t w[4] = {};
  if (count < 8) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < count) w[i / 2] |= (uint32_t)__ldg(src + i) << (i % 2 * 16);
  } else if ((reinterpret_cast<uintptr_t>(src) & 2) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
  } else {
    uint32_t inner[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) inner[i] = __ldg(reinterpret_cast<const uint32_t*>(src + 1) + i);
    w[0] = __byte_perm(__ldg(src), inner[0], 0x5410);
    w[1] = __byte_perm(inner[0], inner[1], 0x5432);
    w[2] = __byte_perm(inner[1], inner[2], 0x5432);
    w[3] = __byte_perm(inner[2], __ldg(src + 7), 0x5432);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One 16-bit row of D elements into a 16-byte aligned one of Dp, by one warp; NULL: zeros.
template <bool VECTOR>
__device__ __forceinline__ void copy_row(unsigned short* dst, const unsigned short* src, int D,
                                         int Dp, int lane) {
  uint4* to = reinterpret_cast<uint4*>(dst);
  if (src == nullptr) {
    for (int c = lane; c < Dp / 8; c += 32) to[c] = make_uint4(0, 0, 0, 0);
  } else if constexpr (VECTOR) {
#pragma unroll 8
    for (int c = lane; c < Dp / 8; c += 32) to[c] = __ldg(reinterpret_cast<const uint4*>(src) + c);
  } else {
#pragma unroll 4
    for (int c = lane; c < Dp / 8; c += 32) to[c] = load_eight(src + c * 8, D - c * 8);
  }
}

constexpr int kGatherThreads = 1024;

template <bool VECTOR>
__global__ void __launch_bounds__(kGatherThreads) loss_gather_kernel(const GatherParams p) {
  // With more than a CTA to an SM the waiting kernel would take room that the gathering needs.
  if (gridDim.x <= 148) start_next_kernel();
  wait_for_previous_kernel();
  __shared__ int warp_counts[kGatherThreads / 32];
  __shared__ int places[kGatherThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t first = (int64_t)blockIdx.x * p.block_rows;
  const int64_t last = min(p.N, first + p.block_rows);
  // Kept rows before this CTA's: every CTA counts them for itself.
  int before = 0;
#pragma unroll 4
  for (int64_t n = tid; n < first; n += kGatherThreads)
    before += load_target(p.targets, p.targets_64, n) != p.ignored;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) warp_counts[warp] = before;
  __syncthreads();
  int place = 0;
  for (int w = 0; w < kGatherThreads / 32; ++w) place += warp_counts[w];
  __syncthreads();
  for (int64_t base = first; base < last; base += kGatherThreads) {
    const int64_t n = base + tid;
    const int64_t target = n < last ? load_target(p.targets, p.targets_64, n) : p.ignored;
    const bool keep = n < last && target != p.ignored;
    const uint32_t votes = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_counts[warp] = __popc(votes);
    __syncthreads();
    int mine = place, total = 0;
    for (int w = 0; w < kGatherThreads / 32; ++w) {
      if (w < warp) mine += warp_counts[w];
      total += warp_counts[w];
    }
    mine += __popc(votes & ((1u << lane) - 1u));
    places[tid] = keep ? mine : -1;
    if (keep) {
      p.kept_index[mine] = (int32_t)n;
      p.kept_target[mine] = (target >= 0 && target < p.V) ? (int32_t)target : -1;
      p.target_logit[mine] = __int_as_float(0x7fc00000);  // stays when there is no such logit
    } else if (n < last) {
      p.losses[n] = 0.f;
    }
    __syncthreads();
    const int rows = (int)min((int64_t)kGatherThreads, last - base);
    for (int r = warp; r < rows; r += kGatherThreads / 32) {
      if (places[r] >= 0)
        copy_row<VECTOR>(p.kept + (int64_t)places[r] * p.Dp,
                         static_cast<const unsigned short*>(p.hidden) +
                             (base + r) * p.hidden_row_stride,
                         p.D, p.Dp, lane);
      else if (p.dhidden != nullptr)
        for (int i = lane; i < p.D; i += 32) p.dhidden[(base + r) * p.D + i] = 0;
    }
    place += total;
    __syncthreads();
  }
  if (last == p.N) {  // the last CTA knows how many there are
    if (tid == 0) {
      *p.count = place;
      if (p.gradient_scale != nullptr)  // no kept row: the gradients are zeros
        *p.gradient_scale = place == 0 ? 0.f : p.mean ? 1.f / (float)place : 1.f;
    }
    const int64_t padded = min(p.N, ((int64_t)place + 127) / 128 * 128);
    for (int64_t r = place + warp; r < padded; r += kGatherThreads / 32)
      copy_row<VECTOR>(p.kept + r * p.Dp, nullptr, p.D, p.Dp, lane);
  }
}

// A weight whose rows the TMA cannot take (width or alignment) is laid out with rows of Dp.
__global__ void __launch_bounds__(256)
loss_pad_kernel(unsigned short* dst, const unsigned short* src, int64_t row_stride, int64_t rows,
                int D, int Dp) {
  start_next_kernel();
  wait_for_previous_kernel();
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8)
    copy_row<false>(dst + r * Dp, src + r * row_stride, D, Dp, threadIdx.x & 31);
}

// ------------------------------------------------------------------------------ the products

enum LossPass { kStats, kProbs, kGradients, kCodes };

// A CTA alone forms tiles of 128 x 256; a pair of CTAs (PAIR) one of 256 x 256 with cta_group::2,
// each holding 128 rows of A and of the result and half of B.  Alone, a CTA loads 48 KB for every
// 128 x 256 x 64 products, which at the tensor cores' rate is more than the 64 bytes a cycle that
// L2 gives an SM; in a pair it is 32 KB.
constexpr int kTileN = 256, kTileK = 64;
constexpr int kBoxBytes = 64 * 64 * 2;
constexpr int kCtaRows = 128;
constexpr int tile_rows(bool pair) { return pair ? 256 : 128; }
constexpr int stage_boxes_b(bool pair) { return pair ? 2 : 4; }
constexpr int stage_bytes(bool pair) { return (2 + stage_boxes_b(pair)) * kBoxBytes; }
constexpr int stage_count(bool pair) { return pair ? 6 : 4; }
constexpr int kEpilogueWarps = 8;
constexpr int kProductThreads = 64 + kEpilogueWarps * 32;
constexpr int kStoreBytes = 4096;  // a warp's block on its way out: 32 rows of 128 bytes
constexpr uint32_t product_smem(bool pair) {
  return stage_count(pair) * stage_bytes(pair) + kEpilogueWarps * kStoreBytes + 1024;
}
// FP16 keeps P times 2^15: probabilities of a large vocabulary would be subnormal.
constexpr float kHalfLift = 32768.f;
constexpr float kCodeSteps = 2048.f;  // of a code, to a power of two
// Steps of K (1024 features) after which a tile of logits goes to registers and is added there.  The
// tensor cores truncate as they add, which shrinks a logit by about D 10^-9 of itself: at 4096
// features the loss was off by 1.8e-6, in segments of 1024 by 4e-7.
constexpr int kSegmentSteps = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct ProductParams {
  const int32_t* count;  // kept rows
  int32_t N, V, D;
  int32_t first_row;     // kept rows [first_row, first_row + row_limit)
  int32_t row_limit;
  int32_t v0, vn;        // the piece: ids [v0, v0 + vn)
  float scale;
  const int32_t* kept_index;
  const int32_t* kept_target;
  float2* partials;        // kStats, kCodes: [row_limit][2 tiles_n] (max, sum) in powers of two
  float* target_logit;     // kStats, kCodes: scale * log2(e) * z of the target
  const float* lse2;       // kProbs: log2 of the sum of exponentials
  const float* weight_of;  // kProbs: c_n over gradient_scale[0]
  const float* gradient_scale;  // kGradients
  void* dhidden;           // kGradients: [N, D] or NULL
  void* dweight;           // kGradients: [V, D] or NULL
  float* slices_out;       // dH in several slices of the vocabulary: FP32 [slices][N, D], or NULL
  float* weight_out;       // dW in several slices or pieces of the rows: FP32 [slices][V, D], or NULL
  int32_t slices, weight_slices;  // that a piece's sums for dH and dW are cut into
  int32_t add_hidden, add_weight;  // not the first piece: slices_out, or weight_out, is added to
  int32_t vector_dhidden, vector_dweight;  // their rows allow 16-byte stores
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  return pack_half2(lo, hi);
}

__device__ __forceinline__ void store_shared16(uint32_t smem, uint32_t a, uint32_t b, uint32_t c,
                                               uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t smem) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(smem)
               : "memory");
  return v;
}

// A warp's block waits in shared memory as 32 rows of 128 bytes, 16-byte chunk c of row r at
// c ^ (r mod 8): the TMA's 128-byte swizzle, and free of bank conflicts both ways.
__device__ __forceinline__ uint32_t block_slot(uint32_t staging, int row, int chunk) {
  return staging + row * 128 + ((chunk ^ (row & 7)) << 4);
}

// Writes the block out row by row, so that a store covers whole lines: `mine` is the element offset
// in `out` of this lane's row, or negative when that row has no place; `columns` (of 128 bytes'
// worth) are valid.  `add` (FP32 only) adds to what is there.
template <typename T>
__device__ __forceinline__ void write_block(uint32_t staging, T* out, int64_t mine, int columns,
                                            bool vector, int lane, bool add = false) {
  constexpr int per_chunk = 16 / (int)sizeof(T), width = 8 * per_chunk;
  __syncwarp();
  if (vector) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = i * 4 + (lane >> 3), chunk = lane & 7;
      const int64_t offset = __shfl_sync(0xffffffffu, mine, row);
      if (offset >= 0 && chunk * per_chunk < columns) {
        uint4* place = reinterpret_cast<uint4*>(out + offset + chunk * per_chunk);
        uint4 v = load_shared16(block_slot(staging, row, chunk));
        if (sizeof(T) == 4 && add) {
          const uint4 there = *place;
          v.x = __float_as_uint(__uint_as_float(there.x) + __uint_as_float(v.x));
          v.y = __float_as_uint(__uint_as_float(there.y) + __uint_as_float(v.y));
          v.z = __float_as_uint(__uint_as_float(there.z) + __uint_as_float(v.z));
          v.w = __float_as_uint(__uint_as_float(there.w) + __uint_as_float(v.w));
        }
        *place = v;
      }
    }
  } else {
    // Element by element, eight rows' loads before their stores.
    constexpr int each = width / 32;
#pragma unroll 1
    for (int first = 0; first < 32; first += 8) {
      uint32_t v[8][each];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int e = 0; e < each; ++e) {
          const int column = e * 32 + lane;
          const uint32_t slot = block_slot(staging, first + i, column / per_chunk) +
                                column % per_chunk * (int)sizeof(T);
          if constexpr (sizeof(T) == 4)
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i][e]) : "r"(slot));
          else
            asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v[i][e]) : "r"(slot));
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t offset = __shfl_sync(0xffffffffu, mine, first + i);
#pragma unroll
        for (int e = 0; e < each; ++e) {
          const int column = e * 32 + lane;
          if (offset < 0 || column >= columns) continue;
          if constexpr (sizeof(T) == 4)
            out[offset + column] = __uint_as_float(v[i][e]) + (add ? (float)out[offset + column] : 0.f);
          else
            reinterpret_cast<unsigned short*>(out)[offset + column] = (unsigned short)v[i][e];
        }
      }
    }
  }
  __syncwarp();
}

// One tile's place in its product: which matrices, where it begins, which steps along K.
struct Tile {
  int m, n;           // first row and column of the result
  int k_first, k_steps;
  bool weight;        // kGradients: dW rather than dH
  int slice;          // of its sum
};

// The tiles of a launch in the order in which CTAs take them.  z: 2048 rows share each column tile
// while it is in L2.  Gradients: the few column tiles of a row tile run side by side, so P comes
// from memory once; dH first, its sums are the longer ones when there are few rows.
template <int PASS, bool PAIR>
struct TileOrder {
  static constexpr int kRows = tile_rows(PAIR);
  int tiles_m, tiles_n, steps;     // kGradients: of dH
  int width = kTileN;              // kGradients: columns of a tile, D spread evenly over the tiles
  int weight_m, weight_steps, slice_steps, weight_slice_steps;
  int hidden_tiles, total;

  __device__ TileOrder(const ProductParams& p, int rows) {
    if constexpr (PASS == kGradients) {
      tiles_n = (p.D + kTileN - 1) / kTileN;
      width = ((p.D + tiles_n - 1) / tiles_n + 31) / 32 * 32;
      tiles_m = p.dhidden != nullptr ? (rows + kRows - 1) / kRows : 0;
      steps = (p.vn + kTileK - 1) / kTileK;
      slice_steps = (steps + p.slices - 1) / p.slices;
      weight_m = p.dweight != nullptr ? (p.vn + kRows - 1) / kRows : 0;
      weight_steps = (rows + kTileK - 1) / kTileK;
      weight_slice_steps = (weight_steps + p.weight_slices - 1) / p.weight_slices;
      hidden_tiles = tiles_m * tiles_n * p.slices;
      total = hidden_tiles + weight_m * tiles_n * p.weight_slices;
    } else {
      tiles_m = (rows + kRows - 1) / kRows;
      tiles_n = (p.vn + kTileN - 1) / kTileN;
      steps = (p.D + kTileK - 1) / kTileK;
      total = tiles_m * tiles_n;
    }
  }

  __device__ Tile at(int index) const {
    Tile t;
    t.weight = false;
    t.slice = 0;
    t.k_first = 0;
    if constexpr (PASS == kGradients) {
      t.weight = index >= hidden_tiles;
      int rest = t.weight ? index - hidden_tiles : index;
      const int per_slice = (t.weight ? weight_m : tiles_m) * tiles_n;
      const int length = t.weight ? weight_slice_steps : slice_steps;
      t.slice = rest / per_slice;
      rest -= t.slice * per_slice;
      t.k_first = t.slice * length;
      t.k_steps = max(0, min(length, (t.weight ? weight_steps : steps) - t.k_first));
      const int row = rest / tiles_n;
      t.m = row * kRows;
      t.n = (rest - row * tiles_n) * width;
    } else {
      constexpr int kGroup = 2048 / kRows;
      const int group = index / (kGroup * tiles_n), rest = index - group * kGroup * tiles_n;
      const int height = min(kGroup, tiles_m - group * kGroup);
      const int column = rest / height;
      t.m = (group * kGroup + rest - column * height) * kRows;
      t.n = column * kTileN;
      t.k_steps = steps;
    }
    return t;
  }
};

// 16 384 rows, 32 000 ids, BF16: kStats 753 us at 1024 features (1.43 PFLOP/s), kCodes 828, kGradients
// 1570 (1.37 PFLOP/s); at 4096 features (14 750 rows) kCodes 2.72 ms (1.42), kGradients 5.45 ms (1.42).
// Power bounds them: clocks fall to 1.56 GHz within 200 us and to 1.35 in a long run, where cuBLAS
// keeps 1.38 PFLOP/s on this GPU.
//
// Warp 0 loads, warp 1 multiplies (in a pair: the first CTA's, for both), warps 2..9 take finished
// tiles out of tensor memory while the next one is formed in its other half.
// Maps: kGradients: P, head, kept rows; the others: kept rows, head, P or codes (to store).
template <int PASS, typename T, bool PAIR>
__global__ void __launch_bounds__(kProductThreads, 1)
loss_product_kernel(const __grid_constant__ CUtensorMap map_0,
                    const __grid_constant__ CUtensorMap map_1,
                    const __grid_constant__ CUtensorMap map_2, const ProductParams p) {
  constexpr bool kBf16 = !__is_same(T, __half);
  constexpr int kRows = tile_rows(PAIR), kStages = stage_count(PAIR);
  constexpr int kStageBytes = stage_bytes(PAIR), kBoxesB = stage_boxes_b(PAIR);
  extern __shared__ unsigned char product_memory[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], done[2], taken[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const uint32_t stages = (smem_addr(product_memory) + 1023u) & ~1023u;
  start_next_kernel();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&done[b], 1);
      mbar_init(&taken[b], kEpilogueWarps * (PAIR ? 2 : 1));
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tensor_map(&map_0);
    prefetch_tensor_map(&map_1);
  }
  if (warp == 1) tmem_alloc_512<PAIR>(&tmem_slot);
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // the other CTA's barriers exist
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  // All of this ran beside the end of the kernel in front; its results are used from here on.
  wait_for_previous_kernel();
  // Kept rows of this launch, counted from first_row on.
  const int kept = min(max(*p.count - p.first_row, 0), p.row_limit);
  const TileOrder<PASS, PAIR> order(p, kept);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (int i = worker; i < order.total && alive; i += workers) {
        const Tile t = order.at(i);
        // Where this CTA's operands begin along M and N, and which tensors they come from.
        const bool a_mn = PASS == kGradients && t.weight;
        const CUtensorMap* map_b = PASS == kGradients && t.weight ? &map_2 : &map_1;
        const int a0 = t.m + rank * kCtaRows + (PASS != kGradients ? p.first_row : 0);
        const int b0 = t.n + rank * (order.width / 2) + (PASS == kGradients ? 0 : p.v0);
        const int bk = PASS != kGradients ? 0 : t.weight ? p.first_row : p.v0;
        const int boxes = PASS != kGradients ? kBoxesB : (order.width / (PAIR ? 2 : 1) + 63) / 64;
        for (int k = t.k_first; k < t.k_first + t.k_steps; ++k) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, &abort_flag)) {
            alive = false;
            break;
          }
          uint32_t bar = smem_addr(&full[stage]);
          if constexpr (PAIR) bar = cluster_address(bar, 0);
          if (rank == 0) mbar_expect_tx(&full[stage], (2 + boxes) * kBoxBytes * (PAIR ? 2 : 1));
          const uint32_t a = stages + stage * kStageBytes, b = a + 2 * kBoxBytes;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            tensor_load_2d<PAIR>(a + j * kBoxBytes, &map_0, a_mn ? a0 + j * 64 : k * kTileK,
                                 a_mn ? k * kTileK : a0 + j * 64, bar);
#pragma unroll
          for (int j = 0; j < kBoxesB; ++j) {
            if (PASS != kGradients || j < boxes)
              tensor_load_2d<PAIR>(b + j * kBoxBytes, map_b,
                                   PASS == kGradients ? b0 + j * 64 : k * kTileK,
                                   PASS == kGradients ? bk + k * kTileK : b0 + j * 64, bar);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, buffer = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool alive = true;
      for (int i = worker; i < order.total && alive; i += workers) {
        const Tile t = order.at(i);
        // 16 elements of K: 32 bytes along a K-major row, two 1 KB groups of MN-major rows.
        const bool a_mn = PASS == kGradients && t.weight;
        const uint32_t instruction = mma_instruction(kBf16, a_mn, PASS == kGradients, kRows, order.width);
        const uint32_t step_a = (a_mn ? 2048 : 32) >> 4;
        constexpr uint32_t step_b = (PASS == kGradients ? 2048 : 32) >> 4;
        int k = 0;
        do {
          const int last = PASS == kGradients ? t.k_steps : min(t.k_steps, k + kSegmentSteps);
          if (!mbar_wait(&taken[buffer], buffer_phase ^ 1u, &abort_flag)) {
            alive = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t d = tmem + buffer * kTileN;
          for (int first = k; k < last; ++k) {
            if (!mbar_wait(&full[stage], phase, &abort_flag)) {
              alive = false;
              break;
            }
            tcgen05_fence_after();
            const uint32_t a = stages + stage * kStageBytes, b = a + 2 * kBoxBytes;
            const uint64_t da = operand_descriptor(a), db = operand_descriptor(b);
#pragma unroll
            for (int kk = 0; kk < kTileK / 16; ++kk)
              tcgen05_mma_f16<PAIR>(d, da + kk * step_a, db + kk * step_b, instruction,
                                    k > first || kk > 0);
            tcgen05_commit<PAIR>(&empty[stage]);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!alive) break;
          tcgen05_commit<PAIR>(&done[buffer]);
          buffer ^= 1;
          if (buffer == 0) buffer_phase ^= 1u;
        } while (k < t.k_steps);
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t staging = stages + kStages * kStageBytes + (warp - 2) * kStoreBytes;
    const float to_log2 = p.scale * kLog2e;
    float out_scale = 0.f;
    if constexpr (PASS == kGradients)
      out_scale = p.scale * *p.gradient_scale * (kBf16 ? 1.f : 1.f / kHalfLift);
    uint32_t taken_bar[2] = {smem_addr(&taken[0]), smem_addr(&taken[1])};
    if constexpr (PAIR) {
      taken_bar[0] = cluster_address(taken_bar[0], 0);
      taken_bar[1] = cluster_address(taken_bar[1], 0);
    }
    int buffer = 0;
    uint32_t buffer_phase = 0;
    for (int i = worker; i < order.total; i += workers) {
      const Tile t = order.at(i);
      const int first_row = t.m + rank * kCtaRows + quad * 32, row = first_row + lane;
      const int column = t.n + half * (order.width / 2);
      // What the row needs is fetched while the products run.  Rows beyond the kept ones are zeros
      // up to a multiple of 128, which gives them P = 0 (the sums over rows reach up to the next
      // multiple of 64).
      int target = -1;
      float lse2 = 0.f, weight_of = 0.f;
      bool live = true;
      if constexpr (PASS != kGradients) {
        live = row < kept;
        if (live) target = p.kept_target[p.first_row + row];
      }
      if constexpr (PASS == kProbs) {
        target = target >= p.v0 ? target - p.v0 : -1;
        if (live) {
          lse2 = p.lse2[p.first_row + row];
          weight_of = p.weight_of[p.first_row + row];
        }
      }
      if (!mbar_wait(&done[buffer], buffer_phase, &abort_flag)) break;
      tcgen05_fence_after();
      uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + buffer * kTileN + half * (order.width / 2);
      auto release = [&] {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_cluster(taken_bar[buffer]);
          else mbar_arrive(&taken[buffer]);
        }
        buffer ^= 1;
        if (buffer == 0) buffer_phase ^= 1u;
      };
      const int columns = min(order.width / 2, p.D - column);  // of this half tile of a gradient
      if constexpr (PASS != kGradients) {
        // The row's 128 logits of the half tile, segment by segment, before anything is done with
        // them: the next tile's products can go on.
        float z[kTileN / 2];
#pragma unroll
        for (int c = 0; c < kTileN / 2; c += 32)
          tmem_load_32(src + c, *reinterpret_cast<uint32_t(*)[32]>(z + c));
        release();
        bool alive = true;
        for (int k = kSegmentSteps; k < t.k_steps; k += kSegmentSteps) {
          if (!mbar_wait(&done[buffer], buffer_phase, &abort_flag)) {
            alive = false;
            break;
          }
          tcgen05_fence_after();
          src = tmem + ((uint32_t)(quad * 32) << 16) + buffer * kTileN + half * (kTileN / 2);
#pragma unroll
          for (int c = 0; c < kTileN / 2; c += 16) {
            uint32_t r[16];
            tmem_load_16(src + c, r);
#pragma unroll
            for (int e = 0; e < 16; ++e) z[c + e] += __uint_as_float(r[e]);
          }
          release();
        }
        if (!alive) break;
        const int valid = p.vn - column, at = target - column;
        const bool rows_exist = first_row < p.row_limit;
        float top = -INFINITY, sums[2] = {0.f, 0.f};
        if constexpr (PASS == kStats || PASS == kCodes) {
          // The half tile's maximum first: sums and codes count from it.
#pragma unroll
          for (int e = 0; e < kTileN / 2; ++e) z[e] *= to_log2;
          if (valid < kTileN / 2) {  // the last tile: ids beyond the vocabulary
#pragma unroll
            for (int e = 0; e < kTileN / 2; ++e) z[e] = e < valid ? z[e] : -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < kTileN / 2; ++e) top = fmaxf(top, z[e]);
          if (at >= 0 && at < kTileN / 2) {
            float y = z[0];
#pragma unroll
            for (int e = 1; e < kTileN / 2; ++e) y = at == e ? z[e] : y;
            p.target_logit[p.first_row + row] = y;
          }
        }
        const float pivot = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int c = 0; c < kTileN / 2; c += 64) {
          if (column + c < p.vn) {
            if constexpr (PASS != kStats) {
              if (lane == 0) tensor_store_wait_read();
              __syncwarp();
            }
#pragma unroll
            for (int h = 0; h < 64; h += 8) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int e = c + h + 2 * q;
                if constexpr (PASS == kProbs) {
                  const float p0 = exp2_approx(fmaf(z[e], to_log2, -lse2));
                  const float p1 = exp2_approx(fmaf(z[e + 1], to_log2, -lse2));
                  const float v0 = weight_of * (at == e ? p0 - 1.f : p0);
                  const float v1 = weight_of * (at == e + 1 ? p1 - 1.f : p1);
                  w[q] = pack2<T>(v0, v1);
                } else {
                  const float down0 = z[e] - pivot, down1 = z[e + 1] - pivot;  // at most zero
                  sums[0] += exp2_approx(down0);
                  sums[1] += exp2_approx(down1);
                  if constexpr (PASS == kCodes) {
                    // Adding 2^23 leaves the rounded integer in the low bits.
                    const float most = 8388608.f + 65535.f;
                    const float code0 = fminf(fmaf(down0, -kCodeSteps, 8388608.f), most);
                    const float code1 = fminf(fmaf(down1, -kCodeSteps, 8388608.f), most);
                    w[q] = __byte_perm(__float_as_uint(code0), __float_as_uint(code1), 0x5410);
                  }
                }
              }
              if constexpr (PASS != kStats)
                store_shared16(block_slot(staging, lane, h / 8), w[0], w[1], w[2], w[3]);
            }
            if constexpr (PASS != kStats) {
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0 && rows_exist) tensor_store_2d(&map_2, column + c, first_row, staging);
            }
          }
        }
        if constexpr (PASS == kStats || PASS == kCodes) {
          // (a half tile beyond the vocabulary is all -inf: it adds nothing)
          if (live)
            p.partials[(int64_t)row * (2 * order.tiles_n) + 2 * (t.n / kTileN) + half] =
                make_float2(top, sums[0] + sums[1]);
        }
      } else if ((t.weight ? p.weight_out : p.slices_out) != nullptr) {
        // A part of the sum, in FP32: loss_slices_kernel adds the slices and rounds.
        int64_t place = -1;
        if (t.weight) {
          if (row < p.vn) place = ((int64_t)t.slice * p.V + p.v0 + row) * p.D + column;
        } else if (row < kept) {
          place = ((int64_t)t.slice * p.N + p.first_row + row) * p.D + column;
        }
        float* parts = t.weight ? p.weight_out : p.slices_out;
#pragma unroll 1
        for (int c = 0; c < columns; c += 32) {
          uint32_t r[32];
          tmem_load_32(src + c, r);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (t.k_steps > 0)
              store_shared16(block_slot(staging, lane, q), r[4 * q], r[4 * q + 1], r[4 * q + 2],
                             r[4 * q + 3]);
            else
              store_shared16(block_slot(staging, lane, q), 0u, 0u, 0u, 0u);
          }
          write_block<float>(staging, parts + c, place, columns - c, p.D % 4 == 0, lane,
                             t.weight ? p.add_weight : p.add_hidden);
        }
      } else {
        int64_t place = -1;
        if (t.weight) {
          if (row < p.vn) place = (int64_t)(p.v0 + row) * p.D + column;
        } else if (row < kept) {
          place = (int64_t)p.kept_index[p.first_row + row] * p.D + column;
        }
        T* out = static_cast<T*>(t.weight ? p.dweight : p.dhidden);
        const bool vector = t.weight ? p.vector_dweight : p.vector_dhidden;
#pragma unroll 1
        for (int c = 0; c < columns; c += 64) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_load_32(src + c + h * 32, r);
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = t.k_steps > 0 ? __uint_as_float(r[e]) * out_scale : 0.f;  // no kept row: zeros
#pragma unroll
            for (int q = 0; q < 4; ++q)
              store_shared16(block_slot(staging, lane, h * 4 + q), pack2<T>(v[8 * q], v[8 * q + 1]),
                             pack2<T>(v[8 * q + 2], v[8 * q + 3]),
                             pack2<T>(v[8 * q + 4], v[8 * q + 5]),
                             pack2<T>(v[8 * q + 6], v[8 * q + 7]));
          }
          write_block<T>(staging, out + c, place, columns - c, vector, lane);
        }
      }
      if constexpr (PASS == kGradients) release();
    }
    if ((PASS == kProbs || PASS == kCodes) && lane == 0) tensor_store_wait_read();
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (abort_flag != 0) {  // copies and products still in flight land before anything is given back
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 200000ull) {
    }
    __syncthreads();
  }
  // Nobody leaves while the other CTA may still read its memory or signal its barriers.
  if constexpr (PAIR) cluster_barrier();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc_512<PAIR>(tmem);
  if constexpr (PAIR) cluster_barrier();
}

// A gradient from its parts, added in order; a warp takes kSliceColumns of a row at a time, so that a
// gradient of three rows still fills the GPU (10 rows of 1590 in 21 parts: 170 us with a warp a row,
// 12 us so).  dH: the kept rows, to their places in the input.  dW (no `kept_index`): rows as
// they are.
constexpr int kSliceColumns = 256;

template <typename T>
__global__ void __launch_bounds__(256)
loss_slices_kernel(const float* __restrict__ slices, int count, const int32_t* kept_rows,
                   const int32_t* __restrict__ kept_index, const float* gradient_scale, float scale,
                   int64_t N, int D, T* out, int vector) {
  start_next_kernel();
  wait_for_previous_kernel();
  const float out_scale = scale * *gradient_scale * (__is_same(T, __half) ? 1.f / kHalfLift : 1.f);
  const int lane = threadIdx.x & 31;
  const int64_t kept = kept_index != nullptr ? *kept_rows : N;
  const int64_t all = N * D;
  const int blocks = (D + kSliceColumns - 1) / kSliceColumns;
  for (int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); item < kept * blocks;
       item += (int64_t)gridDim.x * 8) {
    const int64_t row = item / blocks;
    const int first = (int)(item - row * blocks) * kSliceColumns;
    const float* mine = slices + row * D;
    T* to = out + (kept_index != nullptr ? kept_index[row] : row) * D;
    float sum[8] = {};
    if (vector) {
      const int c = first + lane * 8;
      if (c >= D) continue;
#pragma unroll 4
      for (int s = 0; s < count; ++s) {
        const float4* from = reinterpret_cast<const float4*>(mine + s * all + c);
        const float4 a = __ldcs(from), b = __ldcs(from + 1);
        sum[0] += a.x;
        sum[1] += a.y;
        sum[2] += a.z;
        sum[3] += a.w;
        sum[4] += b.x;
        sum[5] += b.y;
        sum[6] += b.z;
        sum[7] += b.w;
      }
      uint4 v;
      v.x = pack2<T>(sum[0] * out_scale, sum[1] * out_scale);
      v.y = pack2<T>(sum[2] * out_scale, sum[3] * out_scale);
      v.z = pack2<T>(sum[4] * out_scale, sum[5] * out_scale);
      v.w = pack2<T>(sum[6] * out_scale, sum[7] * out_scale);
      *reinterpret_cast<uint4*>(to + c) = v;
    } else {
      const int c = first + lane;
#pragma unroll 2
      for (int s = 0; s < count; ++s) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + 32 * i < D) sum[i] += __ldcs(mine + s * all + c + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + 32 * i < D) to[c + 32 * i] = from_float<T>(sum[i] * out_scale);
    }
  }
}

// ------------------------------------------------------------------------------ joining the loss

constexpr int kJoinThreads = 256;

// log2 of a row's sum of exponentials from its (max, sum) pairs, and its loss: one warp a kept row.
__global__ void __launch_bounds__(kJoinThreads)
loss_join_kernel(const float2* __restrict__ partials, int pairs, const int32_t* count, int first_row,
                 int row_limit, const float* __restrict__ target_logit,
                 const int32_t* __restrict__ kept_index, float* __restrict__ lse2,
                 float* __restrict__ losses) {
  start_next_kernel();
  wait_for_previous_kernel();
  const int row = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= row_limit || first_row + row >= *count) return;
  const float2* mine = partials + (int64_t)row * pairs;
  float top = -INFINITY, sum = 0.f;
  auto add = [&](float other_top, float other_sum) {
    const float high = fmaxf(top, other_top), pivot = high == -INFINITY ? 0.f : high;
    sum = sum * exp2f(top - pivot) + other_sum * exp2f(other_top - pivot);
    top = high;
  };
  for (int i = lane; i < pairs; i += 256) {  // eight pairs at once: one trip to memory, one maximum
    float2 v[8];
    float high = -INFINITY, part = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = i + 32 * k < pairs ? mine[i + 32 * k] : make_float2(-INFINITY, 0.f);
      high = fmaxf(high, v[k].x);
    }
    const float pivot = high == -INFINITY ? 0.f : high;
#pragma unroll
    for (int k = 0; k < 8; ++k) part = fmaf(v[k].y, exp2f(v[k].x - pivot), part);
    add(high, part);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other_top = __shfl_xor_sync(0xffffffffu, top, o);
    const float other_sum = __shfl_xor_sync(0xffffffffu, sum, o);
    add(other_top, other_sum);
  }
  if (lane == 0) {
    const float at_target = target_logit[first_row + row];
    // No logit at the target (an id outside the vocabulary): the loss and the gradients of the
    // row are not numbers, so the mistake shows.
    const float over = log2f(sum);
    lse2[first_row + row] = isnan(at_target) ? at_target : top + over;
    // The two large numbers first: a small loss keeps its digits.
    losses[kept_index[first_row + row]] = ((top - at_target) + over) * kLn2;
  }
}

// Codes become P = p - [v = target] in place: a CTA takes 8192 columns of one kept row, a thread four
// chunks of eight, all loaded before the first is converted.  Memory bounds it: 4 bytes a logit.
constexpr int kProbsThreads = 256;
constexpr int kProbsChunks = 4;
constexpr int kProbsColumns = kProbsThreads * kProbsChunks * 8;

__global__ void __launch_bounds__(kProbsThreads)
loss_probs_kernel(const float2* __restrict__ partials, int pairs, const int32_t* count, int first_row,
                  int row_limit, const float* __restrict__ target_logit,
                  const int32_t* __restrict__ kept_target, const float* __restrict__ lse2,
                  unsigned short* codes, int64_t stride, int V) {
  // (The products' CTAs would take the L1 cache for their shared memory while they wait: they start
  // when this kernel's CTAs are done.)
  wait_for_previous_kernel();
  const int parts = (V + kProbsColumns - 1) / kProbsColumns, total = (V + 7) / 8;
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts;
  if (row >= row_limit || first_row + row >= *count) return;
  uint4* chunks = reinterpret_cast<uint4*>(codes + (int64_t)row * stride);
  const float2* mine = partials + (int64_t)row * pairs;
  const int first = part * (kProbsThreads * kProbsChunks) + threadIdx.x;
  uint4 raw[kProbsChunks];
  float base[kProbsChunks];
#pragma unroll
  for (int k = 0; k < kProbsChunks; ++k) {
    const int c = first + k * kProbsThreads;
    if (c < total) {
      raw[k] = __ldcs(chunks + c);
      base[k] = __ldg(&mine[c >> 4].x);  // sixteen chunks to a half tile
    }
  }
  const float sum2 = lse2[first_row + row];
  const float residue = exp2f(target_logit[first_row + row] - sum2) - 1.f;
  const int target = kept_target[first_row + row];
#pragma unroll
  for (int k = 0; k < kProbsChunks; ++k) {
    const int c = first + k * kProbsThreads;
    if (c >= total) continue;
    const float up = base[k] - sum2;
    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
    float p[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // 2^23 + code as a float, then minus 2^23: exact
      const float lo = __uint_as_float(__byte_perm(w[q], 0x4b000000u, 0x7610)) - 8388608.f;
      const float hi = __uint_as_float(__byte_perm(w[q], 0x4b000000u, 0x7632)) - 8388608.f;
      p[2 * q] = exp2_approx(fmaf(lo, -1.f / kCodeSteps, up));
      p[2 * q + 1] = exp2_approx(fmaf(hi, -1.f / kCodeSteps, up));
    }
    if (c == target >> 3) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e == (target & 7)) p[e] = residue;
    }
    chunks[c] = pack8(p);
  }
}

// Sum or mean of the losses, in a fixed order and FP64, by one CTA.
__global__ void __launch_bounds__(1024)
loss_reduce_kernel(const float* __restrict__ losses, int64_t N, const int32_t* count, int mean,
                   float* out) {
  start_next_kernel();
  wait_for_previous_kernel();
  __shared__ double sums[32];
  double sum = 0.0;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < N; n += 1024) sum += (double)losses[n];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int w = 0; w < 32; ++w) total += sums[w];
    *out = (float)(mean ? total / (double)*count : total);  // no kept row: not a number
  }
}

// Gradients for an upstream gradient of one, times the one that came: eight elements a thread.
__global__ void __launch_bounds__(256)
loss_scale_kernel(const __nv_bfloat16* __restrict__ in, const float* upstream, int64_t elements,
                  __nv_bfloat16* __restrict__ out) {
  const float g = *upstream;
  const int64_t chunks = elements / 8, stride = (int64_t)gridDim.x * 256;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
#pragma unroll 4
  for (int64_t i = first; i < chunks; i += stride) {
    float f[8];
    unpack8(__ldcs(reinterpret_cast<const uint4*>(in) + i), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= g;
    reinterpret_cast<uint4*>(out)[i] = pack8(f);
  }
  for (int64_t i = chunks * 8 + first; i < elements; i += stride)
    out[i] = __float2bfloat16_rn(__bfloat162float(in[i]) * g);
}

// ------------------------------------------------------------------------------ before the gradients

// What each kept row's loss weighs in the result, as a factor of at most one (times 2^15 for
// FP16) and one common scale that the products apply in FP32: whatever the upstream gradient is,
// P stays within its type.  CTA 0 does this; the others zero the gradient of ignored rows.
__global__ void __launch_bounds__(1024)
loss_weights_kernel(const float* upstream, int64_t upstream_stride, int per_row, int mean,
                    const int32_t* count, const int32_t* __restrict__ kept_index, float lift,
                    float* __restrict__ weight_of, float* gradient_scale, const void* targets,
                    int targets_64, int64_t ignored, int64_t N, unsigned short* dhidden, int D) {
  start_next_kernel();
  wait_for_previous_kernel();
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    if (dhidden == nullptr) return;
    const int lane = tid & 31;
    for (int64_t n = (int64_t)(blockIdx.x - 1) * 32 + (tid >> 5); n < N;
         n += (int64_t)(gridDim.x - 1) * 32) {
      if (load_target(targets, targets_64, n) == ignored)
        for (int i = lane; i < D; i += 32) dhidden[n * D + i] = 0;
    }
    return;
  }
  const int kept = *count;
  if (!per_row) {
    for (int i = tid; i < kept; i += 1024) weight_of[i] = lift;
    // no kept row: the gradients are zeros
    if (tid == 0) *gradient_scale = kept == 0 ? 0.f : mean ? *upstream / (float)kept : *upstream;
    return;
  }
  // The largest finite weight is the common scale; infinities and NaN stay with their rows.
  __shared__ float tops[32];
  float top = 0.f;
#pragma unroll 4
  for (int i = tid; i < kept; i += 1024) {
    const float g = fabsf(upstream[kept_index[i] * upstream_stride]);
    if (g <= 3.4028235e38f) top = fmaxf(top, g);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
  top = 0.f;
  for (int w = 0; w < 32; ++w) top = fmaxf(top, tops[w]);
  if (top == 0.f) top = 1.f;
  for (int i = tid; i < kept; i += 1024)
    weight_of[i] = upstream[kept_index[i] * upstream_stride] / top * lift;
  if (tid == 0) *gradient_scale = top;
}

}  // namespace attnres_b200
