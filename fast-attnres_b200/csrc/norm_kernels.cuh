// LayerNorm over the last axis, forward and backward, as an operator of its own (the LayerNorm
// that follows a read lives in the read's epilogue).
//
//   mean = sum(x) / D      rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)      xh = (x - mean) rstd
//   y  = xh w + b
//   gw = g w      dx = rstd (gw - mean(gw) - xh mean(gw xh))
//   dw = sum over rows of g xh         db = sum over rows of g
//
// A row belongs to a group of WARPS warps that keeps it in registers, so it is read once and the
// variance is the sum of squares of centred values (no cancellation, whatever the mean).  Groups
// walk rows with a stride, hold the weights (and the sums of the parameter gradients) of their
// columns in registers for the whole launch, and load rows ahead of the one they work on.
#pragma once

#include "typed_access.cuh"

namespace attnres_b200 {

struct NormParams {
  const void* x;
  int64_t x_row_stride;  // elements
  const void* grad;      // backward only
  int64_t grad_row_stride;
  const void* weight;  // NULL: ones
  const void* bias;    // NULL: zeros
  int32_t param_type;
  int32_t D;
  int64_t N;
  float eps;
  void* y;           // forward: [N,D] contiguous; backward: dx, NULL when not wanted
  float* stats;      // [2,N]: mean, rstd (forward: may be NULL)
  float* partials;   // backward: [gridDim.x, 2D], NULL when no parameter gradient is wanted
};

// Elements a thread owns: NJ chunks of CH consecutive ones (one 16-byte access each) with
// VECTOR, otherwise NJ*CH single elements a group's width apart.
template <typename T, bool VECTOR, int NJ, int WARPS>
struct NormShape {
  static constexpr int kChunk = 16 / (int)sizeof(T);
  static constexpr int kElements = NJ * kChunk;
  static constexpr int kThreads = WARPS * 32;  // of a row group
  static constexpr int kCapacity = kElements * kThreads;

  __device__ static int index(int k, int t) {
    return VECTOR ? ((k / kChunk) * kThreads + t) * kChunk + k % kChunk : k * kThreads + t;
  }

  __device__ static void load(T* dst, const T* row, int D, int t) {
    if constexpr (VECTOR) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = j * kThreads + t;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (c * kChunk < D) raw = __ldg(reinterpret_cast<const uint4*>(row) + c);
        *reinterpret_cast<uint4*>(dst + j * kChunk) = raw;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kElements; ++k) {
        const int i = k * kThreads + t;
        dst[k] = i < D ? row[i] : T(0.f);
      }
    }
  }

  __device__ static void store(T* row, const float* src, int D, int t) {
    if constexpr (VECTOR) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = j * kThreads + t;
        if (c * kChunk < D) {
          __align__(16) T out[kChunk];
#pragma unroll
          for (int e = 0; e < kChunk; ++e) out[e] = from_float<T>(src[j * kChunk + e]);
          *(reinterpret_cast<uint4*>(row) + c) = *reinterpret_cast<const uint4*>(out);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kElements; ++k) {
        const int i = k * kThreads + t;
        if (i < D) row[i] = from_float<T>(src[k]);
      }
    }
  }
};

// Sums K values over a row group; every thread gets the same result, warps are added in index
// order.  `slots` is the group's [2][K][WARPS] scratch; successive calls alternate its halves, so
// one barrier a call is enough.
template <int K, int WARPS>
__device__ __forceinline__ void group_sum(float* v, float* slots, int& parity, int group, int t) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (WARPS > 1) {
    float* half = slots + parity * (K * WARPS);
    parity ^= 1;
    if ((t & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) half[k * WARPS + (t >> 5)] = v[k];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WARPS * 32) : "memory");
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v[k] += half[k * WARPS + w];
    }
  }
}

constexpr int kNormThreads = 512;

template <typename T, bool VECTOR, int NJ, int WARPS>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_fwd_kernel(const NormParams p) {
  using Shape = NormShape<T, VECTOR, NJ, WARPS>;
  constexpr int E = Shape::kElements, TG = Shape::kThreads, GROUPS = kNormThreads / TG;
  __shared__ float scratch[GROUPS][2 * WARPS];
  const int group = threadIdx.x / TG, t = threadIdx.x % TG, D = p.D;
  const float inv_width = 1.0f / (float)D;
  float w[E], b[E];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const int i = Shape::index(k, t);
    w[k] = (p.weight != nullptr && i < D) ? load_typed(p.weight, p.param_type, i) : 1.f;
    b[k] = (p.bias != nullptr && i < D) ? load_typed(p.bias, p.param_type, i) : 0.f;
  }
  const T* x = static_cast<const T*>(p.x);
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  __align__(16) T next[E];
  if (row < p.N) Shape::load(next, x + row * p.x_row_stride, D, t);
  int parity = 0;
  for (; row < p.N; row += stride) {
    float f[E], sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) {
      f[k] = to_float(next[k]);
      sum[0] += f[k];
    }
    if (row + stride < p.N) Shape::load(next, x + (row + stride) * p.x_row_stride, D, t);
    group_sum<1, WARPS>(sum, scratch[group], parity, group, t);
    const float mean = sum[0] * inv_width;
    sum[0] = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      f[k] = Shape::index(k, t) < D ? f[k] - mean : 0.f;
      sum[0] = fmaf(f[k], f[k], sum[0]);
    }
    group_sum<1, WARPS>(sum, scratch[group], parity, group, t);
    const float rstd = rsqrtf(fmaf(sum[0], inv_width, p.eps));
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = fmaf(f[k] * rstd, w[k], b[k]);
    Shape::store(static_cast<T*>(p.y) + row * D, f, D, t);
    if (t == 0 && p.stats != nullptr) {
      p.stats[row] = mean;
      p.stats[p.N + row] = rstd;
    }
  }
}

template <typename T, bool VECTOR, int NJ, int WARPS>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_grad_kernel(const NormParams p) {
  using Shape = NormShape<T, VECTOR, NJ, WARPS>;
  constexpr int E = Shape::kElements, TG = Shape::kThreads, GROUPS = kNormThreads / TG;
  __shared__ float scratch[GROUPS][2 * 2 * WARPS];
  extern __shared__ float group_rows[];  // [GROUPS - 1][2][capacity], used once at the end
  const int group = threadIdx.x / TG, t = threadIdx.x % TG, D = p.D;
  const float inv_width = 1.0f / (float)D;
  float w[E], dw[E], db[E];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const int i = Shape::index(k, t);
    w[k] = (p.weight != nullptr && i < D) ? load_typed(p.weight, p.param_type, i) : 1.f;
    dw[k] = 0.f;
    db[k] = 0.f;
  }
  const T* x = static_cast<const T*>(p.x);
  const T* g = static_cast<const T*>(p.grad);
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  __align__(16) T next_x[E];
  __align__(16) T next_g[E];
  float next_mean = 0.f, next_rstd = 0.f;
  if (row < p.N) {
    Shape::load(next_x, x + row * p.x_row_stride, D, t);
    Shape::load(next_g, g + row * p.grad_row_stride, D, t);
    next_mean = p.stats[row];
    next_rstd = p.stats[p.N + row];
  }
  int parity = 0;
  for (; row < p.N; row += stride) {
    float xh[E], gw[E], sums[2] = {0.f, 0.f};
    const float mean = next_mean, rstd = next_rstd;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      // Elements beyond D were loaded as zeros: their gradient is zero, so whatever xh they
      // get adds nothing to any sum.
      xh[k] = (to_float(next_x[k]) - mean) * rstd;
      const float gk = to_float(next_g[k]);
      gw[k] = gk * w[k];
      sums[0] += gw[k];
      sums[1] = fmaf(gw[k], xh[k], sums[1]);
      dw[k] = fmaf(gk, xh[k], dw[k]);
      db[k] += gk;
    }
    if (row + stride < p.N) {
      Shape::load(next_x, x + (row + stride) * p.x_row_stride, D, t);
      Shape::load(next_g, g + (row + stride) * p.grad_row_stride, D, t);
      next_mean = p.stats[row + stride];
      next_rstd = p.stats[p.N + row + stride];
    }
    if (p.y != nullptr) {  // uniform over the grid
      group_sum<2, WARPS>(sums, scratch[group], parity, group, t);
      const float mean_gw = sums[0] * inv_width, mean_gwx = sums[1] * inv_width;
#pragma unroll
      for (int k = 0; k < E; ++k) gw[k] = rstd * (gw[k] - mean_gw - xh[k] * mean_gwx);
      Shape::store(static_cast<T*>(p.y) + row * D, gw, D, t);
    }
  }
  if (p.partials == nullptr) return;
  // The groups' sums are added in index order, so the result does not depend on timing.
  if (group > 0) {
    float* mine = group_rows + (group - 1) * (2 * Shape::kCapacity);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      mine[k * TG + t] = dw[k];
      mine[Shape::kCapacity + k * TG + t] = db[k];
    }
  }
  __syncthreads();
  if (group > 0) return;
  float* out = p.partials + (int64_t)blockIdx.x * (2 * D);
#pragma unroll
  for (int k = 0; k < E; ++k) {
    for (int other = 0; other < GROUPS - 1; ++other) {
      const float* theirs = group_rows + other * (2 * Shape::kCapacity);
      dw[k] += theirs[k * TG + t];
      db[k] += theirs[Shape::kCapacity + k * TG + t];
    }
    const int i = Shape::index(k, t);
    if (i < D) {
      out[i] = dw[k];
      out[D + i] = db[k];
    }
  }
}

// Column sums of the [rows, 2D] partials in a fixed order and FP64 (this stage adds no rounding
// of its own), written in the parameters' type; either output may be NULL.
constexpr int kNormReduceColumns = 16;
constexpr int kNormReduceGroups = 32;

__global__ void __launch_bounds__(kNormReduceColumns * kNormReduceGroups)
layer_norm_param_reduce_kernel(const float* __restrict__ partials, int rows, int D, void* dweight,
                               void* dbias, int param_type) {
  __shared__ double sums[kNormReduceGroups][kNormReduceColumns + 1];
  const int col = threadIdx.x % kNormReduceColumns, grp = threadIdx.x / kNormReduceColumns;
  const int c = blockIdx.x * kNormReduceColumns + col;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  if (c < 2 * D) {
    const float* column = partials + c;
    const int64_t width = 2 * (int64_t)D;
    int row = grp;
    for (; row + 3 * kNormReduceGroups < rows; row += 4 * kNormReduceGroups) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += (double)column[(row + k * kNormReduceGroups) * width];
    }
    for (; row < rows; row += kNormReduceGroups) s[0] += (double)column[row * width];
  }
  sums[grp][col] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (grp == 0 && c < 2 * D) {
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < kNormReduceGroups; ++k) total += sums[k][col];
    void* out = c < D ? dweight : dbias;
    if (out != nullptr) store_typed(out, param_type, c < D ? c : c - D, (float)total);
  }
}

}  // namespace attnres_b200
