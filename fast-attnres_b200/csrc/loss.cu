// C ABI of the vocabulary loss (declared in include/attnres_b200.h).
#include <cmath>

#include "loss_kernels.cuh"

namespace attnres_b200 {

int loss_error_flag(int* flag, int clear) {
  int value = 0;
  if (cudaMemcpyFromSymbol(&value, g_error_flag, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return ATTNRES_B200_ERR_CUDA;
  }
  *flag = value;
  if (clear && value != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_error_flag, &zero, sizeof(int)) != cudaSuccess) {
      cudaGetLastError();
      return ATTNRES_B200_ERR_CUDA;
    }
  }
  return ATTNRES_B200_OK;
}

namespace {

constexpr int64_t kMaxLossRows = 1 << 30;
constexpr int32_t kMaxLossVocabulary = 1 << 25;
// Bytes of (max, sum) pairs held at a time (65 536 rows of 32 000 ids take 131 MB).
constexpr int64_t kPairBytes = 256ll << 20;
// Bytes of P held at a time.  With more than one piece a gradient is added up in FP32 in memory;
// 16 384 rows of 32 000 ids are one piece.
constexpr int64_t kPieceBytes = 1024ll << 20;
constexpr int64_t kPieceMinimum = 4096;

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled find_encode_tiled() {
  void* found = nullptr;
  cudaDriverEntryPointQueryResult result;
  if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault,
                                       &result) == cudaSuccess &&
      result == cudaDriverEntryPointSuccess)
    return reinterpret_cast<EncodeTiled>(found);
  cudaGetLastError();
  return nullptr;
}

EncodeTiled encode_tiled() {
  static const EncodeTiled function = find_encode_tiled();
  return function;
}

// A 16-bit row-major matrix read (or written) in boxes of 64 columns.
int make_map(CUtensorMap* map, const void* base, int32_t type, int64_t rows, int64_t columns,
             int64_t row_stride, int box_rows) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return ATTNRES_B200_ERR_CUDA;
  const cuuint64_t sizes[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_stride * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, steps[2] = {1, 1};
  const CUtensorMapDataType element = type == ATTNRES_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encode(map, element, 2, const_cast<void*>(base), sizes, strides, box, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
                 CUDA_SUCCESS
             ? ATTNRES_B200_OK
             : ATTNRES_B200_ERR_CUDA;
}

int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int check_loss(int64_t N, int32_t V, int32_t D, int32_t type, float scale) {
  if (D < 1 || D > kMaxWidth) return ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1 || N > kMaxLossRows) return ATTNRES_B200_ERR_BAD_ROWS;
  if (V < 1 || V > kMaxLossVocabulary) return ATTNRES_B200_ERR_BAD_VOCABULARY;
  if (type != ATTNRES_B200_BF16 && type != ATTNRES_B200_FP16) return ATTNRES_B200_ERR_BAD_TYPE;
  if (!std::isfinite(scale)) return ATTNRES_B200_ERR_BAD_SCALAR;
  return ATTNRES_B200_OK;
}

int32_t padded_width(int32_t D) { return (D + 7) / 8 * 8; }

bool needs_padding(const void* weight, int64_t row_stride, int32_t V, int32_t D) {
  return D % 8 != 0 || !aligned16(weight) || (V > 1 && (row_stride % 8 != 0 || row_stride < D));
}

struct LossPlan {
  int64_t padded_weight;  // bytes of a padded copy of the weight
  int64_t stats_rows, partials;
  int64_t piece, pieces;  // ids of a piece
  int64_t slices, weight_slices;
  int64_t probs, slices_out, weight_out, weights;
};

int64_t tiles_of(int64_t rows, int64_t columns, bool pair) {
  return ((rows + tile_rows(pair) - 1) / tile_rows(pair)) * ((columns + kTileN - 1) / kTileN);
}

// Pairs of CTAs load a third less for the same products; single CTAs make twice as many, smaller
// tiles, which is what counts when there are few.
bool use_pairs(int64_t tiles_of_pairs) { return tiles_of_pairs >= 296; }

// Slices that a gradient's sum is cut into: few rows (or few ids) make few tiles, each a long sum over
// the vocabulary (or the rows).  One for every SM, but of sixteen steps at least.  Whole and cut, with
// the adding up: 10 rows of 49115 ids of 1590 features 363 and 162 us, 19318 rows of 13 ids of 111
// features 107 and 22 us; whole steps over 1024 and 2048 rows of 32000 ids of 1024 features 356 and 265,
// 454 and 389 us, and over 4096 rows of 1000 ids of 2048 features (64 steps in two) 100 and 95 us.
int64_t slices_of(int64_t tiles, int64_t sum_over) {
  const int64_t wanted = 148 / tiles, most = (sum_over + kTileK - 1) / kTileK / 16;
  return wanted < 1 || most < 1 ? 1 : wanted < most ? wanted : most;
}

LossPlan plan_loss(int64_t N, int32_t V, int32_t D) {
  LossPlan plan;
  plan.padded_weight = align256((int64_t)V * padded_width(D) * 2);
  const int64_t tiles_n = (V + kTileN - 1) / kTileN;
  plan.stats_rows = kPairBytes / (2 * tiles_n * (int64_t)sizeof(float2)) / 256 * 256;
  if (plan.stats_rows < 256) plan.stats_rows = 256;
  if (plan.stats_rows > N) plan.stats_rows = N;
  plan.partials = align256(plan.stats_rows * 2 * tiles_n * (int64_t)sizeof(float2));
  int64_t most = kPieceBytes / (2 * N) / kTileN * kTileN;
  if (most < kPieceMinimum) most = kPieceMinimum;
  plan.pieces = (V + most - 1) / most;
  plan.piece = ((V + plan.pieces - 1) / plan.pieces + kTileN - 1) / kTileN * kTileN;
  plan.pieces = (V + plan.piece - 1) / plan.piece;
  const int64_t columns = plan.piece < V ? plan.piece : padded_width(V);
  plan.probs = align256(N * columns * 2);
  const int64_t numbers = (int64_t)sizeof(float) * D;
  plan.slices = slices_of(tiles_of(N, D, false), plan.piece);
  plan.slices_out = plan.slices * plan.pieces > 1 ? align256(plan.slices * N * numbers) : 0;
  plan.weight_slices = plan.pieces > 1 ? 1 : slices_of(tiles_of(V, D, false), N);
  plan.weight_out = plan.weight_slices > 1 ? align256(plan.weight_slices * V * numbers) : 0;
  plan.weights = align256((N + 1) * (int64_t)sizeof(float));
  return plan;
}

// The forward that forms the gradients as well works on pieces of the rows.
struct GradientPlan {
  int64_t piece, pieces;  // rows
  int64_t slices, weight_slices;
  int64_t partials, codes, slices_out, weight_out;
};

GradientPlan plan_gradients(int64_t N, int32_t V, int32_t D) {
  GradientPlan plan;
  int64_t most = kPieceBytes / (2 * (int64_t)padded_width(V)) / 256 * 256;
  if (most < 256) most = 256;
  plan.pieces = (N + most - 1) / most;
  plan.piece = ((N + plan.pieces - 1) / plan.pieces + 255) / 256 * 256;
  if (plan.piece > N) plan.piece = N;
  plan.pieces = (N + plan.piece - 1) / plan.piece;
  const int64_t tiles_n = (V + kTileN - 1) / kTileN;
  plan.partials = align256(plan.piece * 2 * tiles_n * (int64_t)sizeof(float2));
  plan.codes = align256(plan.piece * (int64_t)padded_width(V) * 2);
  const int64_t numbers = (int64_t)sizeof(float) * D;
  plan.slices = slices_of(tiles_of(plan.piece, D, false), V);
  plan.slices_out = plan.slices > 1 ? align256(plan.slices * N * numbers) : 0;
  plan.weight_slices = slices_of(tiles_of(V, D, false), plan.piece);
  plan.weight_out =
      plan.weight_slices * plan.pieces > 1 ? align256(plan.weight_slices * V * numbers) : 0;
  return plan;
}

template <int PASS, typename T, bool PAIR>
int launch_product(const CUtensorMap (&maps)[3], const ProductParams& p, int64_t tiles, int sms,
                   cudaStream_t stream) {
  static SmemGrant grant;
  constexpr uint32_t smem = product_smem(PAIR);
  if (int st = prepare_kernel(loss_product_kernel<PASS, T, PAIR>, smem, grant)) return st;
  const int64_t workers = PAIR ? sms / 2 : sms;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((tiles < workers ? tiles : workers) * (PAIR ? 2 : 1)));
  config.blockDim = dim3(kProductThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = 2;
  attributes[1].val.clusterDim.y = 1;
  attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&config, loss_product_kernel<PASS, T, PAIR>, maps[0], maps[1], maps[2],
                         p) != cudaSuccess) {
    cudaGetLastError();
    return ATTNRES_B200_ERR_CUDA;
  }
  return ATTNRES_B200_OK;
}

// `tiles(pair)` counts the launch's tiles for pairs and for single CTAs.
template <int PASS, typename Count>
int launch_product_type(int32_t type, const CUtensorMap (&maps)[3], const ProductParams& p,
                        Count tiles, int sms, cudaStream_t stream) {
  const bool pair = use_pairs(tiles(true));
  if (type == ATTNRES_B200_BF16)
    return pair ? launch_product<PASS, __nv_bfloat16, true>(maps, p, tiles(true), sms, stream)
                : launch_product<PASS, __nv_bfloat16, false>(maps, p, tiles(false), sms, stream);
  return pair ? launch_product<PASS, __half, true>(maps, p, tiles(true), sms, stream)
              : launch_product<PASS, __half, false>(maps, p, tiles(false), sms, stream);
}

// The gradients that were formed in parts.
template <typename T>
int launch_slices_type(const ProductParams& p, int sms, cudaStream_t stream) {
  const int64_t most = 8 * sms, blocks = (p.D + kSliceColumns - 1) / kSliceColumns;
  if (p.slices_out != nullptr) {
    const int64_t ctas = (p.N * blocks + 7) / 8;
    if (int st = launch_behind(loss_slices_kernel<T>, ctas < most ? ctas : most, 256, 0, true, stream,
                               p.slices_out, p.slices, p.count, p.kept_index, p.gradient_scale,
                               p.scale, (int64_t)p.N, p.D, static_cast<T*>(p.dhidden),
                               p.vector_dhidden))
      return st;
  }
  if (p.weight_out != nullptr) {
    const int64_t ctas = (p.V * blocks + 7) / 8;
    if (int st = launch_behind(loss_slices_kernel<T>, ctas < most ? ctas : most, 256, 0, true, stream,
                               p.weight_out, p.weight_slices, nullptr, nullptr, p.gradient_scale,
                               p.scale, (int64_t)p.V, p.D, static_cast<T*>(p.dweight),
                               p.vector_dweight))
      return st;
  }
  return ATTNRES_B200_OK;
}

int launch_slices(const ProductParams& p, int32_t type, int sms, cudaStream_t stream) {
  return type == ATTNRES_B200_BF16 ? launch_slices_type<__nv_bfloat16>(p, sms, stream)
                                   : launch_slices_type<__half>(p, sms, stream);
}

// The weight as the TMA can read it: in place, or copied into rows of a multiple of eight.
int lay_out_weight(const void** weight, int64_t* row_stride, int32_t V, int32_t D, void* copy,
                   bool behind, int sms, cudaStream_t stream) {
  if (!needs_padding(*weight, *row_stride, V, D)) return ATTNRES_B200_OK;
  if (int st = launch_behind(loss_pad_kernel, sms * 8, 256, 0, behind, stream,
                             static_cast<unsigned short*>(copy),
                             static_cast<const unsigned short*>(*weight), *row_stride, (int64_t)V, D,
                             padded_width(D)))
    return st;
  *weight = copy;
  *row_stride = padded_width(D);
  return ATTNRES_B200_OK;
}

}  // namespace
}  // namespace attnres_b200

using namespace attnres_b200;

extern "C" int64_t attnres_b200_loss_workspace_bytes(int64_t N, int32_t V, int32_t D,
                                                     int32_t pass) {
  if (int st = check_loss(N, V, D, ATTNRES_B200_BF16, 1.f)) return -st;
  const LossPlan plan = plan_loss(N, V, D);
  const int64_t logits = align256(N * (int64_t)sizeof(float));
  if (pass == ATTNRES_B200_LOSS_FORWARD) return plan.padded_weight + plan.partials + logits;
  if (pass == ATTNRES_B200_LOSS_FORWARD_GRADIENTS) {
    const GradientPlan gradients = plan_gradients(N, V, D);
    return plan.padded_weight + gradients.partials + 2 * logits + 256 + gradients.codes +
           gradients.slices_out + gradients.weight_out;
  }
  if (pass != ATTNRES_B200_LOSS_BACKWARD) return -ATTNRES_B200_ERR_BAD_FLAGS;
  return plan.padded_weight + plan.probs + plan.slices_out + plan.weight_out + plan.weights;
}

extern "C" int attnres_b200_loss_forward(
    const void* hidden, int64_t hidden_row_stride, const void* weight, int64_t weight_row_stride,
    const void* targets, int32_t targets_64, int64_t N, int32_t V, int32_t D, int32_t type,
    int64_t ignored, float scale, int32_t reduction, void* kept, int32_t* kept_index,
    int32_t* kept_target, int32_t* count, float* lse2, float* losses, float* loss, void* dhidden,
    void* dweight, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int st = check_loss(N, V, D, type, scale)) return st;
  const bool gradients = dhidden != nullptr || dweight != nullptr;
  if (gradients && type != ATTNRES_B200_BF16) return ATTNRES_B200_ERR_BAD_TYPE;
  if (gradients && reduction == ATTNRES_B200_LOSS_NONE) return ATTNRES_B200_ERR_BAD_FLAGS;
  if (reduction < ATTNRES_B200_LOSS_NONE || reduction > ATTNRES_B200_LOSS_MEAN)
    return ATTNRES_B200_ERR_BAD_FLAGS;
  if (!hidden || !weight || !targets || !kept || !kept_index || !kept_target || !count ||
      (!gradients && !lse2) || !losses || !workspace ||
      (reduction != ATTNRES_B200_LOSS_NONE && !loss))
    return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned2(hidden) || !aligned2(weight) || !aligned16(kept) || !aligned16(workspace) ||
      !aligned2(dhidden) || !aligned2(dweight) ||
      (reinterpret_cast<uintptr_t>(targets) & (targets_64 ? 7u : 3u)) != 0)
    return ATTNRES_B200_ERR_MISALIGNED;
  const int32_t pass = gradients ? ATTNRES_B200_LOSS_FORWARD_GRADIENTS : ATTNRES_B200_LOSS_FORWARD;
  if (workspace_bytes < attnres_b200_loss_workspace_bytes(N, V, D, pass))
    return ATTNRES_B200_ERR_WORKSPACE;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const LossPlan plan = plan_loss(N, V, D);
  const int32_t Dp = padded_width(D);
  char* space = static_cast<char*>(workspace);
  const GradientPlan pieces = plan_gradients(N, V, D);
  float2* partials = reinterpret_cast<float2*>(space + plan.padded_weight);
  char* rest = space + plan.padded_weight + (gradients ? pieces.partials : plan.partials);
  float* target_logit = reinterpret_cast<float*>(rest);
  rest += align256(N * (int64_t)sizeof(float));
  float* gradient_scale = reinterpret_cast<float*>(rest);  // from here on with gradients only
  float* sums = gradient_scale + 64;
  rest += 256 + align256(N * (int64_t)sizeof(float));
  unsigned short* codes = reinterpret_cast<unsigned short*>(rest);
  float* slices_out = reinterpret_cast<float*>(rest + pieces.codes);
  float* weight_out = reinterpret_cast<float*>(rest + pieces.codes + pieces.slices_out);

  GatherParams g{};
  g.hidden = hidden;
  g.hidden_row_stride = hidden_row_stride;
  g.targets = targets;
  g.targets_64 = targets_64;
  g.N = N;
  g.D = D;
  g.Dp = Dp;
  g.V = V;
  g.ignored = ignored;
  // Every CTA counts the kept rows before its own, so their number is bounded (512).
  g.block_rows = (int32_t)(32 * ((N + 32 * 512 - 1) / (32 * 512)));
  g.kept = static_cast<unsigned short*>(kept);
  g.kept_index = kept_index;
  g.kept_target = kept_target;
  g.count = count;
  g.target_logit = target_logit;
  g.losses = losses;
  if (gradients) {
    g.gradient_scale = gradient_scale;
    g.mean = reduction == ATTNRES_B200_LOSS_MEAN;
    g.dhidden = static_cast<unsigned short*>(dhidden);
  }
  const int gather_grid = (int)((N + g.block_rows - 1) / g.block_rows);
  if (D % 8 == 0 && aligned16(hidden) && (N == 1 || hidden_row_stride % 8 == 0))
    loss_gather_kernel<true><<<gather_grid, kGatherThreads, 0, cs>>>(g);
  else
    loss_gather_kernel<false><<<gather_grid, kGatherThreads, 0, cs>>>(g);
  if (int st = launched()) return st;
  if (int st = lay_out_weight(&weight, &weight_row_stride, V, D, space, true, sms, cs)) return st;

  CUtensorMap maps[3];
  if (int st = make_map(&maps[0], kept, type, N, D, Dp, 64)) return st;
  if (int st = make_map(&maps[1], weight, type, V, D, V > 1 ? weight_row_stride : Dp, 64)) return st;
  maps[2] = maps[1];  // nothing is stored through a map here
  ProductParams p{};
  p.count = count;
  p.N = (int32_t)N;
  p.V = V;
  p.D = D;
  p.v0 = 0;
  p.vn = V;
  p.scale = scale;
  p.kept_target = kept_target;
  p.partials = partials;
  p.target_logit = target_logit;
  const int pairs = 2 * ((V + kTileN - 1) / kTileN);
  if (gradients) {
    const int64_t stride = padded_width(V);
    p.kept_index = kept_index;
    p.gradient_scale = gradient_scale;
    p.dhidden = dhidden;
    p.dweight = dweight;
    p.vector_dhidden = D % 8 == 0 && aligned16(dhidden);
    p.vector_dweight = D % 8 == 0 && aligned16(dweight);
    p.slices = (int32_t)pieces.slices;
    p.weight_slices = (int32_t)pieces.weight_slices;
    p.slices_out = dhidden != nullptr && pieces.slices_out > 0 ? slices_out : nullptr;
    p.weight_out = dweight != nullptr && pieces.weight_out > 0 ? weight_out : nullptr;
    for (int64_t piece = 0; piece < pieces.pieces; ++piece) {
      p.first_row = (int32_t)(piece * pieces.piece);
      p.row_limit = (int32_t)(N - p.first_row < pieces.piece ? N - p.first_row : pieces.piece);
      CUtensorMap form[3] = {maps[0], maps[1], maps[1]}, use[3] = {maps[0], maps[1], maps[0]};
      if (int st = make_map(&form[2], codes, type, p.row_limit, V, stride, 32)) return st;
      if (int st = make_map(&use[0], codes, type, p.row_limit, V, stride, 64)) return st;
      const auto logits = [&](bool pair) { return tiles_of(p.row_limit, V, pair); };
      if (int st = launch_product_type<kCodes>(type, form, p, logits, sms, cs)) return st;
      if (int st = launch_behind(loss_join_kernel, (p.row_limit + 7) / 8, kJoinThreads, 0, true, cs,
                                 partials, pairs, count, p.first_row, p.row_limit, target_logit,
                                 kept_index, sums, losses))
        return st;
      const int64_t parts = (V + kProbsColumns - 1) / kProbsColumns;
      if (int st = launch_behind(loss_probs_kernel, p.row_limit * parts, kProbsThreads, 0, true, cs,
                                 partials, pairs, count, p.first_row, p.row_limit, target_logit,
                                 kept_target, sums, codes, stride, V))
        return st;
      p.add_weight = piece > 0;  // a piece's rows of dH are its own
      const auto both = [&](bool pair) {
        return (dhidden ? tiles_of(p.row_limit, D, pair) * p.slices : 0) +
               (dweight ? tiles_of(V, D, pair) * p.weight_slices : 0);
      };
      if (int st = launch_product_type<kGradients>(type, use, p, both, sms, cs)) return st;
    }
    if (int st = launch_slices(p, type, sms, cs)) return st;
  }
  for (int64_t row = 0; row < N && !gradients; row += plan.stats_rows) {
    p.first_row = (int32_t)row;
    p.row_limit = (int32_t)(N - row < plan.stats_rows ? N - row : plan.stats_rows);
    const auto tiles = [&](bool pair) { return tiles_of(p.row_limit, V, pair); };
    if (int st = launch_product_type<kStats>(type, maps, p, tiles, sms, cs)) return st;
    if (int st = launch_behind(loss_join_kernel, (p.row_limit + 7) / 8, kJoinThreads, 0, true, cs,
                               partials, pairs, count, p.first_row, p.row_limit, target_logit,
                               kept_index, lse2, losses))
      return st;
  }
  if (reduction == ATTNRES_B200_LOSS_NONE) return ATTNRES_B200_OK;
  return launch_behind(loss_reduce_kernel, 1, 1024, 0, true, cs, losses, N, count,
                       (int)(reduction == ATTNRES_B200_LOSS_MEAN), loss);
}

extern "C" int attnres_b200_loss_backward(
    const float* upstream, int64_t upstream_stride, const void* weight, int64_t weight_row_stride,
    const void* targets, int32_t targets_64, int64_t N, int32_t V, int32_t D, int32_t type,
    int64_t ignored, float scale, int32_t reduction, const void* kept, const int32_t* kept_index,
    const int32_t* kept_target, const int32_t* count, const float* lse2, void* dhidden,
    void* dweight, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int st = check_loss(N, V, D, type, scale)) return st;
  if (reduction < ATTNRES_B200_LOSS_NONE || reduction > ATTNRES_B200_LOSS_MEAN)
    return ATTNRES_B200_ERR_BAD_FLAGS;
  if (!dhidden && !dweight) return ATTNRES_B200_ERR_NOTHING_TO_DO;
  if (!upstream || !weight || !targets || !kept || !kept_index || !kept_target || !count || !lse2 ||
      !workspace)
    return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned2(weight) || !aligned16(kept) || !aligned16(workspace) || !aligned2(dhidden) ||
      !aligned2(dweight) || (reinterpret_cast<uintptr_t>(targets) & (targets_64 ? 7u : 3u)) != 0)
    return ATTNRES_B200_ERR_MISALIGNED;
  if (workspace_bytes < attnres_b200_loss_workspace_bytes(N, V, D, ATTNRES_B200_LOSS_BACKWARD))
    return ATTNRES_B200_ERR_WORKSPACE;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const LossPlan plan = plan_loss(N, V, D);
  const int32_t Dp = padded_width(D);
  char* space = static_cast<char*>(workspace);
  void* probs = space + plan.padded_weight;
  float* slices_out = reinterpret_cast<float*>(space + plan.padded_weight + plan.probs);
  float* weight_out =
      reinterpret_cast<float*>(space + plan.padded_weight + plan.probs + plan.slices_out);
  float* gradient_scale = reinterpret_cast<float*>(space + plan.padded_weight + plan.probs +
                                                   plan.slices_out + plan.weight_out);
  float* weight_of = gradient_scale + 1;

  const bool padded = needs_padding(weight, weight_row_stride, V, D);
  if (int st = lay_out_weight(&weight, &weight_row_stride, V, D, space, false, sms, cs)) return st;
  const int64_t zero_ctas = (N + 31) / 32;
  if (int st = launch_behind(loss_weights_kernel, 1 + (zero_ctas < 2 * sms ? zero_ctas : 2 * sms), 1024,
                             0, padded, cs, upstream, upstream_stride,
                             (int)(reduction == ATTNRES_B200_LOSS_NONE),
                             (int)(reduction == ATTNRES_B200_LOSS_MEAN), count, kept_index,
                             type == ATTNRES_B200_FP16 ? kHalfLift : 1.f, weight_of, gradient_scale,
                             targets, targets_64, ignored, N, static_cast<unsigned short*>(dhidden), D))
    return st;

  CUtensorMap map_h, map_w;
  if (int st = make_map(&map_h, kept, type, N, D, Dp, 64)) return st;
  if (int st = make_map(&map_w, weight, type, V, D, V > 1 ? weight_row_stride : Dp, 64)) return st;
  ProductParams p{};
  p.count = count;
  p.N = (int32_t)N;
  p.V = V;
  p.D = D;
  p.scale = scale;
  p.kept_index = kept_index;
  p.kept_target = kept_target;
  p.lse2 = lse2;
  p.weight_of = weight_of;
  p.row_limit = (int32_t)N;
  p.gradient_scale = gradient_scale;
  p.dhidden = dhidden;
  p.dweight = dweight;
  p.vector_dhidden = D % 8 == 0 && aligned16(dhidden);
  p.vector_dweight = D % 8 == 0 && aligned16(dweight);
  p.slices = (int32_t)plan.slices;
  p.weight_slices = (int32_t)plan.weight_slices;
  p.slices_out = dhidden != nullptr && plan.slices_out > 0 ? slices_out : nullptr;
  p.weight_out = dweight != nullptr && plan.weight_out > 0 ? weight_out : nullptr;
  for (int64_t v0 = 0; v0 < V; v0 += plan.piece) {
    p.v0 = (int32_t)v0;
    p.vn = (int32_t)(V - v0 < plan.piece ? V - v0 : plan.piece);
    const int64_t stride = padded_width(p.vn);
    CUtensorMap form[3] = {map_h, map_w, map_w}, use[3] = {map_h, map_w, map_h};
    if (int st = make_map(&form[2], probs, type, N, p.vn, stride, 32)) return st;
    if (int st = make_map(&use[0], probs, type, N, p.vn, stride, 64)) return st;
    const auto logits = [&](bool pair) { return tiles_of(N, p.vn, pair); };
    if (int st = launch_product_type<kProbs>(type, form, p, logits, sms, cs)) return st;
    const auto gradients = [&](bool pair) {
      return (dhidden ? tiles_of(N, D, pair) * plan.slices : 0) +
             (dweight ? tiles_of(p.vn, D, pair) * plan.weight_slices : 0);
    };
    if (int st = launch_product_type<kGradients>(type, use, p, gradients, sms, cs)) return st;
    p.add_hidden = 1;  // a piece's rows of dW are its own
  }
  return launch_slices(p, type, sms, cs);
}

extern "C" int32_t attnres_b200_loss_gradients_in_forward(int32_t D, int32_t type, int32_t reduction) {
  // The gradients' own forward saves the second z (2 N V D products) and spends 4 N V bytes on
  // turning codes into P, which ties near D = 450 at 1.4 PFLOP/s and 6.5 TB/s.  FP16 stays with the
  // backward: its gradients before the upstream factor may be too small for the type.
  return type == ATTNRES_B200_BF16 && reduction != ATTNRES_B200_LOSS_NONE && D >= 512;
}

extern "C" int attnres_b200_loss_scale_gradient(const void* gradient, const float* upstream,
                                                int64_t elements, void* out, void* stream) {
  if (elements < 1) return ATTNRES_B200_ERR_BAD_ROWS;
  if (!gradient || !upstream || !out) return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned16(gradient) || !aligned16(out)) return ATTNRES_B200_ERR_MISALIGNED;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  const int64_t ctas = (elements / 8 + 1023) / 1024 + 1;
  loss_scale_kernel<<<(unsigned)(ctas < 16 * sms ? ctas : 16 * sms), 256, 0,
                      static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(gradient), upstream, elements,
      static_cast<__nv_bfloat16*>(out));
  return launched();
}
