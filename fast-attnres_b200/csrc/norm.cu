// C ABI of the LayerNorm operator (declared in include/attnres_b200.h).
#include <cmath>

#include "norm_kernels.cuh"
#include "tma_common.cuh"

namespace attnres_b200 {
namespace {

enum NormPass { kForward, kBackward };

template <typename T, bool VECTOR, int NJ, int WARPS>
int launch_norm(NormPass pass, const NormParams& p, int grid, cudaStream_t stream) {
  using Shape = NormShape<T, VECTOR, NJ, WARPS>;
  if (pass == kForward) {
    layer_norm_fwd_kernel<T, VECTOR, NJ, WARPS><<<grid, kNormThreads, 0, stream>>>(p);
    return launched();
  }
  static SmemGrant grant;
  constexpr int groups = kNormThreads / Shape::kThreads;
  constexpr uint32_t smem = (groups - 1) * 2 * Shape::kCapacity * (uint32_t)sizeof(float);
  if (smem > 0) {
    if (int st = prepare_kernel(layer_norm_grad_kernel<T, VECTOR, NJ, WARPS>, smem, grant)) return st;
  }
  layer_norm_grad_kernel<T, VECTOR, NJ, WARPS><<<grid, kNormThreads, smem, stream>>>(p);
  return launched();
}

// Warps of a row group: eight elements to a thread up to 4096 features, sixteen beyond.
inline int norm_warps(int D) {
  for (int warps = 1; warps < 16; warps *= 2)
    if (D <= warps * 256) return warps;
  return 16;
}

template <typename T, bool VECTOR>
int dispatch_norm(NormPass pass, const NormParams& p, int grid, cudaStream_t st) {
  constexpr int NJ = (int)sizeof(T) / 2;
  switch (norm_warps(p.D)) {
    case 1: return launch_norm<T, VECTOR, NJ, 1>(pass, p, grid, st);
    case 2: return launch_norm<T, VECTOR, NJ, 2>(pass, p, grid, st);
    case 4: return launch_norm<T, VECTOR, NJ, 4>(pass, p, grid, st);
    case 8: return launch_norm<T, VECTOR, NJ, 8>(pass, p, grid, st);
    default:
      if (p.D <= 4096) return launch_norm<T, VECTOR, NJ, 16>(pass, p, grid, st);
      return launch_norm<T, VECTOR, 2 * NJ, 16>(pass, p, grid, st);
  }
}

int dispatch_norm_type(NormPass pass, const NormParams& p, int32_t type, bool vector, int grid,
                       cudaStream_t st) {
  if (type == ATTNRES_B200_BF16)
    return vector ? dispatch_norm<__nv_bfloat16, true>(pass, p, grid, st)
                  : dispatch_norm<__nv_bfloat16, false>(pass, p, grid, st);
  if (type == ATTNRES_B200_FP16)
    return vector ? dispatch_norm<__half, true>(pass, p, grid, st)
                  : dispatch_norm<__half, false>(pass, p, grid, st);
  return vector ? dispatch_norm<float, true>(pass, p, grid, st)
                : dispatch_norm<float, false>(pass, p, grid, st);
}

int norm_grid(int64_t N, int D, int sms, int ctas_per_sm) {
  const int64_t groups = kNormThreads / (norm_warps(D) * 32);
  const int64_t needed = (N + groups - 1) / groups, cap = (int64_t)sms * ctas_per_sm;
  return (int)(needed < cap ? needed : cap);
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
  return dispatch_norm_type(kForward, p, type, vector, norm_grid(N, D, sms, 3),
                            static_cast<cudaStream_t>(stream));
}

extern "C" int32_t attnres_b200_norm_workspace_rows(int64_t N, int32_t D, int32_t device) {
  if (D < 1 || D > kMaxWidth) return -ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1) return -ATTNRES_B200_ERR_BAD_ROWS;
  int sms = 0;
  if (int st = sm_count(device, &sms)) return -st;
  return norm_grid(N, D, sms, 2);
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
  const int grid = norm_grid(N, D, sms, 2);
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
  if (int st = dispatch_norm_type(kBackward, p, type, vector, grid, cs)) return st;
  if (!want_params) return ATTNRES_B200_OK;
  layer_norm_param_reduce_kernel<<<(2 * D + kNormReduceColumns - 1) / kNormReduceColumns,
                                   kNormReduceColumns * kNormReduceGroups, 0, cs>>>(
      partials, grid, D, dweight, dbias, param_type);
  return launched();
}
