// C ABI of the LayerNorm operator (declared in include/attnres_b200.h).
#include <cmath>

#include "norm_kernels.cuh"
#include "tma_common.cuh"

namespace attnres_b200 {
namespace {

enum NormPass { kForward, kBackward };

// What a thread holds of a row, and the warps that share one.  More elements to a thread mean
// fewer reductions to an element: with eight everywhere, BF16 rows of 4096 ran at 3.9 TB/s where
// FP32 rows of as many bytes ran at 6.0.  The forward holds three values an element, the backward
// five; element-wise rows keep the next row in registers too.  A forward of so few rows that every
// SM gets one at most is all latency and takes eight elements to a thread (8 x 4096: 3.0 us
// against 6.4 us with 32).
struct NormPlan {
  int elements, warps;
};

inline NormPlan norm_plan(NormPass pass, int64_t N, int D, bool vector, int sms) {
  const bool few = pass == kForward && vector && N <= sms && D <= 4096;
  const int most = few ? 8 : pass == kForward && vector ? 32 : 16;
  int elements = 8;
  while (elements < most && D > elements * 32) elements *= 2;
  int warps = 1;
  while (D > elements * warps * 32) warps *= 2;
  return {elements, warps};
}

int norm_grid(NormPass pass, int64_t N, int D, bool vector, int sms) {
  const NormPlan plan = norm_plan(pass, N, D, vector, sms);
  const int64_t groups = kNormThreads / (plan.warps * 32);
  const int64_t needed = (N + groups - 1) / groups;
  const int64_t cap = (int64_t)sms * (pass == kForward ? norm_fwd_ctas(plan.elements, vector)
                                                       : norm_grad_ctas(plan.elements));
  return (int)(needed < cap ? needed : cap);
}

template <NormPass PASS, typename T, bool VECTOR, int E, int WARPS>
int launch_norm(const NormParams& p, int grid, cudaStream_t stream) {
  using Shape = NormShape<T, VECTOR, E, WARPS>;
  static SmemGrant grant;
  if constexpr (PASS == kForward) {
    constexpr uint32_t smem = VECTOR ? NormRing<Shape, 1>::kBytes : 0;
    if (int st = prepare_kernel(layer_norm_fwd_kernel<T, VECTOR, E, WARPS>, smem, grant)) return st;
    layer_norm_fwd_kernel<T, VECTOR, E, WARPS><<<grid, kNormThreads, smem, stream>>>(p);
  } else {
    constexpr uint32_t ring = VECTOR ? NormRing<Shape, 2>::kBytes : 0;
    constexpr uint32_t meeting =
        (kNormThreads / Shape::kThreads - 1) * 2 * Shape::kCapacity * (uint32_t)sizeof(float);
    constexpr uint32_t smem = ring < meeting ? meeting : ring;
    if (int st = prepare_kernel(layer_norm_grad_kernel<T, VECTOR, E, WARPS>, smem, grant)) return st;
    layer_norm_grad_kernel<T, VECTOR, E, WARPS><<<grid, kNormThreads, smem, stream>>>(p);
  }
  return launched();
}

template <NormPass PASS, typename T, bool VECTOR>
int dispatch_norm(const NormParams& p, int sms, cudaStream_t st) {
  constexpr int kMost = PASS == kForward && VECTOR ? 32 : 16;
  const NormPlan plan = norm_plan(PASS, p.N, p.D, VECTOR, sms);
  const int grid = norm_grid(PASS, p.N, p.D, VECTOR, sms);
  if (plan.elements == 8) {
    if (plan.warps == 1) return launch_norm<PASS, T, VECTOR, 8, 1>(p, grid, st);
    if constexpr (kMost == 32) {
      switch (plan.warps) {
        case 2: return launch_norm<PASS, T, VECTOR, 8, 2>(p, grid, st);
        case 4: return launch_norm<PASS, T, VECTOR, 8, 4>(p, grid, st);
        case 8: return launch_norm<PASS, T, VECTOR, 8, 8>(p, grid, st);
        default: return launch_norm<PASS, T, VECTOR, 8, 16>(p, grid, st);
      }
    }
  }
  if (plan.elements == 16 && plan.warps == 1) return launch_norm<PASS, T, VECTOR, 16, 1>(p, grid, st);
  switch (plan.warps) {
    case 1:
      if constexpr (kMost == 32) return launch_norm<PASS, T, VECTOR, 32, 1>(p, grid, st);
    case 2: return launch_norm<PASS, T, VECTOR, kMost, 2>(p, grid, st);
    case 4: return launch_norm<PASS, T, VECTOR, kMost, 4>(p, grid, st);
    case 8: return launch_norm<PASS, T, VECTOR, kMost, 8>(p, grid, st);
    default:
      if constexpr (kMost == 16) return launch_norm<PASS, T, VECTOR, 16, 16>(p, grid, st);
      return ATTNRES_B200_ERR_BAD_WIDTH;
  }
}

template <NormPass PASS>
int dispatch_norm_type(const NormParams& p, int32_t type, bool vector, int sms, cudaStream_t st) {
  if (type == ATTNRES_B200_BF16)
    return vector ? dispatch_norm<PASS, __nv_bfloat16, true>(p, sms, st)
                  : dispatch_norm<PASS, __nv_bfloat16, false>(p, sms, st);
  if (type == ATTNRES_B200_FP16)
    return vector ? dispatch_norm<PASS, __half, true>(p, sms, st)
                  : dispatch_norm<PASS, __half, false>(p, sms, st);
  return vector ? dispatch_norm<PASS, float, true>(p, sms, st)
                : dispatch_norm<PASS, float, false>(p, sms, st);
}

int check_norm(int64_t N, int32_t D, int32_t type, int32_t param_type) {
  if (D < 1 || D > kMaxWidth) return ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1) return ATTNRES_B200_ERR_BAD_ROWS;
  if (!type_ok(type) || !type_ok(param_type)) return ATTNRES_B200_ERR_BAD_TYPE;
  return ATTNRES_B200_OK;
}

bool rows_vector(const void* base, int64_t row_stride, int64_t N, int32_t D, int32_t type) {
  const int chunk = 16 / type_bytes(type);
  return aligned16(base) && D % chunk == 0 && (N == 1 || row_stride % chunk == 0);
}

}  // namespace
}  // namespace attnres_b200

using namespace attnres_b200;

extern "C" int attnres_b200_norm_forward(
    const void* x, int64_t x_row_stride, const void* weight, const void* bias, int64_t N, int32_t D,
    int32_t type, int32_t param_type, float eps, void* y, float* stats, void* stream) {
  if (int st = check_norm(N, D, type, param_type)) return st;
  if (!std::isfinite(eps) || eps < 0.f) return ATTNRES_B200_ERR_BAD_SCALAR;
  if (!x || !y) return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned_type(x, type) || !aligned_type(y, type) || !aligned_type(weight, param_type) ||
      !aligned_type(bias, param_type))
    return ATTNRES_B200_ERR_MISALIGNED;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  NormParams p{};
  p.x = x;
  p.x_row_stride = x_row_stride;
  p.weight = weight;
  p.bias = bias;
  p.param_type = param_type;
  p.D = D;
  p.N = N;
  p.eps = eps;
  p.y = y;
  p.stats = stats;
  const bool vector = rows_vector(x, x_row_stride, N, D, type) && aligned16(y);
  return dispatch_norm_type<kForward>(p, type, vector, sms, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t attnres_b200_norm_workspace_rows(int64_t N, int32_t D, int32_t device) {
  if (D < 1 || D > kMaxWidth) return -ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1) return -ATTNRES_B200_ERR_BAD_ROWS;
  int sms = 0;
  if (int st = sm_count(device, &sms)) return -st;
  // the same plan for both kinds of access: the backward's does not depend on it
  return norm_grid(kBackward, N, D, true, sms);
}

extern "C" int attnres_b200_norm_backward(
    const void* grad, int64_t grad_row_stride, const void* x, int64_t x_row_stride,
    const float* stats, const void* weight, int64_t N, int32_t D, int32_t type, int32_t param_type,
    void* dx, float* partials, int32_t partial_rows, void* dweight, void* dbias, void* stream) {
  if (int st = check_norm(N, D, type, param_type)) return st;
  if (!grad || !x || !stats) return ATTNRES_B200_ERR_NULL_POINTER;
  const bool want_params = dweight != nullptr || dbias != nullptr;
  if (!dx && !want_params) return ATTNRES_B200_ERR_NOTHING_TO_DO;
  if (want_params && !partials) return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned_type(grad, type) || !aligned_type(x, type) || !aligned_type(dx, type) ||
      !aligned_type(weight, param_type) || !aligned_type(dweight, param_type) ||
      !aligned_type(dbias, param_type))
    return ATTNRES_B200_ERR_MISALIGNED;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  const int grid = norm_grid(kBackward, N, D, true, sms);
  if (want_params && partial_rows < grid) return ATTNRES_B200_ERR_WORKSPACE;
  NormParams p{};
  p.x = x;
  p.x_row_stride = x_row_stride;
  p.grad = grad;
  p.grad_row_stride = grad_row_stride;
  p.weight = weight;
  p.param_type = param_type;
  p.D = D;
  p.N = N;
  p.y = dx;
  p.stats = const_cast<float*>(stats);
  p.partials = want_params ? partials : nullptr;
  const bool vector = rows_vector(x, x_row_stride, N, D, type) &&
                      rows_vector(grad, grad_row_stride, N, D, type) && aligned16(dx);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (int st = dispatch_norm_type<kBackward>(p, type, vector, sms, cs)) return st;
  if (!want_params) return ATTNRES_B200_OK;
  return launch_behind(layer_norm_param_reduce_kernel,
                       (2 * D + kNormReduceColumns - 1) / kNormReduceColumns,
                       kNormReduceColumns * kNormReduceGroups, 0, true, cs, (const float*)partials,
                       grid, D, dweight, dbias, param_type);
}
