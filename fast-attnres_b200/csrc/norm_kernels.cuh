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
// walk rows with a stride and hold the weights (and the sums of the parameter gradients) of their
// columns in registers for the whole launch.  With 16-byte accesses a thread copies its own chunks
// of the rows ahead into a shared-memory ring (cp.async: no barrier, each thread reads back only
// what it copied itself), otherwise the next row waits in registers.
//
// DRAM bounds it.  BF16, 16 384 rows, forward / backward with parameter gradients: 1024 features
// 11.4 / 22 us (5.9 / 4.5 TB/s), 4096 features 44 / 75 us (6.1 / 5.4 TB/s), of 6.6 for a copy;
// FP32, 8192 x 8192: 94 / 141 us (5.7 TB/s); element by element, FP32 4099 x 1537: 10.7 / 18 us.
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

// What a thread owns of a row: E elements as pairs, in 16-byte chunks of CH consecutive ones with
// VECTOR, otherwise single elements a group's width apart.
template <typename T, bool VECTOR, int E, int WARPS>
struct NormShape {
  static constexpr int kChunk = 16 / (int)sizeof(T);
  static constexpr int kChunks = E / kChunk;
  static constexpr int kThreads = WARPS * 32;  // of a row group
  static constexpr int kCapacity = E * kThreads;

  __device__ static int index(int k, int t) {
    return VECTOR ? ((k / kChunk) * kThreads + t) * kChunk + k % kChunk : k * kThreads + t;
  }

  // The pairs of chunk j from its 16 bytes.
  __device__ static void unpack(const uint4& raw, float2* f) {
    if constexpr (sizeof(T) == 4) {
      f[0] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
      f[1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
    } else {
      const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (__is_same(T, __half)) f[k] = __half22float2(*reinterpret_cast<const __half2*>(&words[k]));
        else f[k] = make_float2(bf16x2_lo(words[k]), bf16x2_hi(words[k]));
      }
    }
  }

  __device__ static void load(T* dst, const T* row, int D, int t) {
    static_assert(!VECTOR, "rows of 16-byte chunks come through the ring");
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int i = k * kThreads + t;
      dst[k] = i < D ? row[i] : T(0.f);
    }
  }

  __device__ static void store(T* row, const float2* src, int D, int t) {
    const float* flat = reinterpret_cast<const float*>(src);
    if constexpr (VECTOR) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int c = j * kThreads + t;
        if (c * kChunk < D) {
          __align__(16) T out[kChunk];
#pragma unroll
          for (int e = 0; e < kChunk; ++e) out[e] = from_float<T>(flat[j * kChunk + e]);
          *(reinterpret_cast<uint4*>(row) + c) = *reinterpret_cast<const uint4*>(out);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int i = k * kThreads + t;
        if (i < D) row[i] = from_float<T>(flat[k]);
      }
    }
  }

  // [D] parameters of any type as this thread's pairs.
  __device__ static void parameters(float2* dst, const void* base, int type, int D, int t,
                                    float otherwise) {
    if (base == nullptr) {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) dst[k] = make_float2(otherwise, otherwise);
      return;
    }
    if (VECTOR && (reinterpret_cast<uintptr_t>(base) & 15u) == 0) {  // chunk by chunk
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int c = j * kThreads + t;
        float f[8];
        if (c * kChunk < D) {
          if (type == ATTNRES_B200_FP32) {
#pragma unroll
            for (int k = 0; k < kChunk / 4; ++k) {
              const float4 v = __ldg(static_cast<const float4*>(base) + c * (kChunk / 4) + k);
              f[4 * k] = v.x;
              f[4 * k + 1] = v.y;
              f[4 * k + 2] = v.z;
              f[4 * k + 3] = v.w;
            }
          } else {
#pragma unroll
            for (int k = 0; k < kChunk / 4; ++k) {
              const uint2 v = __ldg(static_cast<const uint2*>(base) + c * (kChunk / 4) + k);
              const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
              const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
              const bool bf16 = type == ATTNRES_B200_BF16;
              f[4 * k] = bf16 ? bf16x2_lo(v.x) : lo.x;
              f[4 * k + 1] = bf16 ? bf16x2_hi(v.x) : lo.y;
              f[4 * k + 2] = bf16 ? bf16x2_lo(v.y) : hi.x;
              f[4 * k + 3] = bf16 ? bf16x2_hi(v.y) : hi.y;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < kChunk; ++e) f[e] = otherwise;
        }
#pragma unroll
        for (int k = 0; k < kChunk / 2; ++k)
          dst[j * (kChunk / 2) + k] = make_float2(f[2 * k], f[2 * k + 1]);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < E; k += 2) {
      const int i = index(k, t), j = index(k + 1, t);
      dst[k / 2].x = i < D ? load_typed(base, type, i) : otherwise;
      dst[k / 2].y = j < D ? load_typed(base, type, j) : otherwise;
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

// Ring stages by what a CTA's rows take, and resident CTAs by what a thread holds in registers
// (element-wise rows need registers for the next row as well).
constexpr int norm_fwd_ctas(int E, bool vector) {
  return vector ? (E <= 8 ? 3 : E <= 16 ? 2 : 1) : (E <= 8 ? 2 : 1);
}
constexpr int norm_grad_ctas(int E) { return E <= 8 ? 2 : 1; }

template <typename Shape, int OPERANDS>
struct NormRing {
  static constexpr int kChunks = Shape::kChunks * OPERANDS;  // a thread's, a row
  static constexpr int kStages = kChunks <= 1 ? 5 : kChunks <= 2 ? 4 : 3;
  static constexpr uint32_t kBytes = (uint32_t)kStages * kChunks * kNormThreads * 16;

  // Starts the copy of operand `which` of a row; chunks beyond D become zeros.
  template <typename T>
  __device__ static void copy(uint4* ring, int stage, int which, const T* row, int D, int t) {
#pragma unroll
    for (int j = 0; j < Shape::kChunks; ++j) {
      const int c = j * Shape::kThreads + t;
      const bool inside = c * Shape::kChunk < D;
      const uint4* src = reinterpret_cast<const uint4*>(row) + (inside ? c : 0);
      const uint4* dst = at(ring, stage, which, j);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                   "l"(src), "r"(inside ? 16 : 0)
                   : "memory");
    }
  }
  __device__ static uint4* at(uint4* ring, int stage, int which, int j) {
    return ring + ((stage * kChunks + which * Shape::kChunks + j) * kNormThreads + threadIdx.x);
  }
  __device__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // The oldest of the rows in flight has arrived.
  __device__ static void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
  }
  __device__ static void drain() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
  __device__ static void read(float2* dst, uint4* ring, int stage, int which) {
#pragma unroll
    for (int j = 0; j < Shape::kChunks; ++j)
      Shape::unpack(*at(ring, stage, which, j), dst + j * (Shape::kChunk / 2));
  }
};

extern __shared__ uint4 norm_smem[];

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <typename T, bool VECTOR, int E, int WARPS>
__global__ void __launch_bounds__(kNormThreads, norm_fwd_ctas(E, VECTOR))
layer_norm_fwd_kernel(const NormParams p) {
  using Shape = NormShape<T, VECTOR, E, WARPS>;
  using Ring = NormRing<Shape, 1>;
  constexpr int TG = Shape::kThreads, GROUPS = kNormThreads / TG;
  __shared__ float scratch[GROUPS][2 * WARPS];
  // (the same number in every lane, and known to be: rows are addressed with uniform registers)
  const int group = __shfl_sync(0xffffffffu, threadIdx.x / TG, 0), t = threadIdx.x % TG, D = p.D;
  const float inv_width = 1.0f / (float)D;
  const T* x = static_cast<const T*>(p.x);
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  T now[VECTOR ? 1 : E];
  int stage = 0;
  auto fetch = [&](int64_t which, int to) {
    if constexpr (VECTOR) {
      if (which < p.N) Ring::copy(norm_smem, to, 0, x + which * p.x_row_stride, D, t);
      Ring::commit();
    } else {
      if (which < p.N) Shape::load(now, x + which * p.x_row_stride, D, t);
    }
  };
  if constexpr (VECTOR) {
#pragma unroll
    for (int k = 0; k < Ring::kStages - 1; ++k) fetch(row + k * stride, k);
  } else {
    fetch(row, 0);
  }
  float2 w[E / 2], b[E / 2];
  Shape::parameters(w, p.weight, p.param_type, D, t, 1.f);
  Shape::parameters(b, p.bias, p.param_type, D, t, 0.f);
  int parity = 0;
  for (; row < p.N; row += stride) {
    float2 f[E / 2], part[2] = {both(0.f), both(0.f)};
    if constexpr (VECTOR) {
      // the stage that the previous row was read from
      fetch(row + (Ring::kStages - 1) * stride, stage == 0 ? Ring::kStages - 1 : stage - 1);
      Ring::wait();
      Ring::read(f, norm_smem, stage, 0);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) f[k] = make_float2(to_float(now[2 * k]), to_float(now[2 * k + 1]));
      fetch(row + stride, 0);
    }
#pragma unroll
    for (int k = 0; k < E / 2; ++k) part[k & 1] = __fadd2_rn(part[k & 1], f[k]);
    float sum[1] = {(part[0].x + part[0].y) + (part[1].x + part[1].y)};
    group_sum<1, WARPS>(sum, scratch[group], parity, group, t);
    const float mean = sum[0] * inv_width;
#pragma unroll
    for (int k = 0; k < E / 2; ++k) f[k] = __fadd2_rn(f[k], both(-mean));
    if (D != Shape::kCapacity) {  // what lies beyond the row adds nothing to the variance
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        if (Shape::index(2 * k, t) >= D) f[k].x = 0.f;
        if (Shape::index(2 * k + 1, t) >= D) f[k].y = 0.f;
      }
    }
    part[0] = part[1] = both(0.f);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) part[k & 1] = __ffma2_rn(f[k], f[k], part[k & 1]);
    sum[0] = (part[0].x + part[0].y) + (part[1].x + part[1].y);
    group_sum<1, WARPS>(sum, scratch[group], parity, group, t);
    const float rstd = rsqrtf(fmaf(sum[0], inv_width, p.eps));
#pragma unroll
    for (int k = 0; k < E / 2; ++k) f[k] = __ffma2_rn(__fmul2_rn(f[k], both(rstd)), w[k], b[k]);
    Shape::store(static_cast<T*>(p.y) + row * D, f, D, t);
    if (t == 0 && p.stats != nullptr) {
      p.stats[row] = mean;
      p.stats[p.N + row] = rstd;
    }
  }
  if constexpr (VECTOR) Ring::drain();
}

template <typename T, bool VECTOR, int E, int WARPS>
__global__ void __launch_bounds__(kNormThreads, norm_grad_ctas(E))
layer_norm_grad_kernel(const NormParams p) {
  start_next_kernel();  // the reduction of the partial sums waits for the end
  using Shape = NormShape<T, VECTOR, E, WARPS>;
  using Ring = NormRing<Shape, 2>;
  constexpr int TG = Shape::kThreads, GROUPS = kNormThreads / TG;
  __shared__ float scratch[GROUPS][2 * 2 * WARPS];
  const int group = __shfl_sync(0xffffffffu, threadIdx.x / TG, 0), t = threadIdx.x % TG, D = p.D;
  const float inv_width = 1.0f / (float)D;
  const T* x = static_cast<const T*>(p.x);
  const T* g = static_cast<const T*>(p.grad);
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  T now_x[VECTOR ? 1 : E], now_g[VECTOR ? 1 : E];
  float next_mean = 0.f, next_rstd = 0.f;
  int stage = 0;
  auto fetch = [&](int64_t which, int to) {
    if constexpr (VECTOR) {
      if (which < p.N) {
        Ring::copy(norm_smem, to, 0, x + which * p.x_row_stride, D, t);
        Ring::copy(norm_smem, to, 1, g + which * p.grad_row_stride, D, t);
      }
      Ring::commit();
    } else {
      if (which < p.N) {
        Shape::load(now_x, x + which * p.x_row_stride, D, t);
        Shape::load(now_g, g + which * p.grad_row_stride, D, t);
      }
    }
  };
  auto fetch_stats = [&](int64_t which) {
    if (which < p.N) {
      next_mean = p.stats[which];
      next_rstd = p.stats[p.N + which];
    }
  };
  if constexpr (VECTOR) {
#pragma unroll
    for (int k = 0; k < Ring::kStages - 1; ++k) fetch(row + k * stride, k);
  } else {
    fetch(row, 0);
  }
  fetch_stats(row);
  float2 w[E / 2], dw[E / 2], db[E / 2];
  Shape::parameters(w, p.weight, p.param_type, D, t, 1.f);
#pragma unroll
  for (int k = 0; k < E / 2; ++k) dw[k] = db[k] = both(0.f);
  int parity = 0;
  for (; row < p.N; row += stride) {
    float2 xh[E / 2], gw[E / 2];
    if constexpr (VECTOR) {
      fetch(row + (Ring::kStages - 1) * stride, stage == 0 ? Ring::kStages - 1 : stage - 1);
      Ring::wait();
      Ring::read(xh, norm_smem, stage, 0);
      Ring::read(gw, norm_smem, stage, 1);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        xh[k] = make_float2(to_float(now_x[2 * k]), to_float(now_x[2 * k + 1]));
        gw[k] = make_float2(to_float(now_g[2 * k]), to_float(now_g[2 * k + 1]));
      }
      fetch(row + stride, 0);
    }
    const float mean = next_mean, rstd = next_rstd;
    fetch_stats(row + stride);
    float2 sum_gw = both(0.f), sum_gwx = both(0.f);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      // Elements beyond D were loaded as zeros: their gradient is zero, so whatever xh they
      // get adds nothing to any sum.
      xh[k] = __fmul2_rn(__fadd2_rn(xh[k], both(-mean)), both(rstd));
      dw[k] = __ffma2_rn(gw[k], xh[k], dw[k]);
      db[k] = __fadd2_rn(db[k], gw[k]);
      gw[k] = __fmul2_rn(gw[k], w[k]);
      sum_gw = __fadd2_rn(sum_gw, gw[k]);
      sum_gwx = __ffma2_rn(gw[k], xh[k], sum_gwx);
    }
    if (p.y != nullptr) {  // uniform over the grid
      float sums[2] = {sum_gw.x + sum_gw.y, sum_gwx.x + sum_gwx.y};
      group_sum<2, WARPS>(sums, scratch[group], parity, group, t);
      const float mean_gw = sums[0] * inv_width, mean_gwx = sums[1] * inv_width;
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        gw[k] = __ffma2_rn(xh[k], both(-mean_gwx), __fadd2_rn(gw[k], both(-mean_gw)));
        gw[k] = __fmul2_rn(gw[k], both(rstd));
      }
      Shape::store(static_cast<T*>(p.y) + row * D, gw, D, t);
    }
  }
  if constexpr (VECTOR) Ring::drain();
  if (p.partials == nullptr) return;
  // The groups' sums are added in index order, so the result does not depend on timing.  They
  // meet in the ring's memory, which nobody needs any more.
  float* group_rows = reinterpret_cast<float*>(norm_smem);
  float* sums_w = reinterpret_cast<float*>(dw);
  float* sums_b = reinterpret_cast<float*>(db);
  __syncthreads();
  if (group > 0) {
    float* mine = group_rows + (group - 1) * (2 * Shape::kCapacity);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      mine[k * TG + t] = sums_w[k];
      mine[Shape::kCapacity + k * TG + t] = sums_b[k];
    }
  }
  __syncthreads();
  if (group > 0) return;
  float* out = p.partials + (int64_t)blockIdx.x * (2 * D);
#pragma unroll
  for (int k = 0; k < E; ++k) {
    for (int other = 0; other < GROUPS - 1; ++other) {
      const float* theirs = group_rows + other * (2 * Shape::kCapacity);
      sums_w[k] += theirs[k * TG + t];
      sums_b[k] += theirs[Shape::kCapacity + k * TG + t];
    }
    const int i = Shape::index(k, t);
    if (i < D) {
      out[i] = sums_w[k];
      out[D + i] = sums_b[k];
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
  wait_for_previous_kernel();
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
