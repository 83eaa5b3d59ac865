// C ABI of the embedding operator (declared in include/attnres_b200.h).
#include <cmath>

#include "embedding_kernels.cuh"
#include "tma_common.cuh"

namespace attnres_b200 {
namespace {

constexpr int64_t kMaxTokens = (1ll << 31) - 1;  // positions are 32-bit inside the sort
constexpr int32_t kMaxVocabulary = 1 << 25;

int check_embedding(int64_t N, int64_t T, int32_t V, int32_t D, int32_t type, int32_t out_type,
                    int32_t position_type, float scale) {
  if (D < 1 || D > kMaxWidth) return ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1 || N > kMaxTokens || T < 1 || N % T != 0) return ATTNRES_B200_ERR_BAD_ROWS;
  if (V < 1 || V > kMaxVocabulary) return ATTNRES_B200_ERR_BAD_VOCABULARY;
  if (!type_ok(type) || !type_ok(out_type) || !type_ok(position_type))
    return ATTNRES_B200_ERR_BAD_TYPE;
  if (!std::isfinite(scale)) return ATTNRES_B200_ERR_BAD_SCALAR;
  return ATTNRES_B200_OK;
}

int64_t tile_pairs(int64_t N) {
  // 32 pairs a tile keep enough tiles for every SM at the usual sizes (16 384 ids: 512 tiles for
  // each 256 columns); beyond 131 072 ids the tiles grow, so that the pieces' workspace and the
  // joining of one very frequent id stay bounded (4096 tiles).
  const int64_t grown = (N + 4095) / 4096;
  return grown <= 32 ? 32 : (grown + 7) / 8 * 8;
}

template <bool VECTOR, bool WIDE>
int launch_embedding_forward(const EmbedParams& p, int lanes, dim3 grid, cudaStream_t stream) {
  if (p.positions == nullptr)
    embedding_fwd_kernel<VECTOR, WIDE, kNoPositions><<<grid, kEmbedThreads, 0, stream>>>(p, lanes);
  else if (p.position_type != ATTNRES_B200_FP32)
    embedding_fwd_kernel<VECTOR, WIDE, kNarrowPositions><<<grid, kEmbedThreads, 0, stream>>>(p, lanes);
  else
    embedding_fwd_kernel<VECTOR, WIDE, kWidePositions><<<grid, kEmbedThreads, 0, stream>>>(p, lanes);
  return launched();
}

template <bool VECTOR, bool WIDE>
int launch_embedding_backward(const EmbedParams& p, int sms, cudaStream_t cs) {
  static SmemGrant grant;
  int64_t fill_ctas = 0, position_ctas = 0;
  const bool few = p.dtable != nullptr && p.N <= kFewTokens;
  if (p.dtable != nullptr && !few) {
    if (int st = prepare_kernel(embedding_sort_kernel, kSortSmem, grant)) return st;
    embedding_sort_kernel<<<kSortCluster, kSortThreads, kSortSmem, cs>>>(p);
    if (int st = launched()) return st;
  }
  if (p.dtable != nullptr) {
    // Every filling CTA reads all ids: few of them where that takes longer than the filling.
    fill_ctas = p.N <= 65536 ? 4 * sms : sms;
    const int64_t ranges = ((int64_t)p.V + kFillRange - 2) / (kFillRange - 1);
    if (fill_ctas < ranges) fill_ctas = ranges;  // a bitmap holds its CTA's range
    if (fill_ctas > p.V) fill_ctas = p.V;
  }
  if (p.dpositions != nullptr)
    position_ctas = (p.T * ((p.D + 7) / 8) + kEarlyThreads - 1) / kEarlyThreads;
  if (few) {
    const int64_t columns = 32 * gradient_columns<VECTOR>();
    const int64_t sums = (p.N * ((p.D + columns - 1) / columns) * 32 + kEarlyThreads - 1) / kEarlyThreads;
    embedding_early_kernel<VECTOR, WIDE, true>
        <<<(unsigned)(fill_ctas + position_ctas + sums), kEarlyThreads, 0, cs>>>(
            p, type_bytes(p.table_type), (int)fill_ctas, (int)sums);
    return launched();
  }
  if (int st = launch_behind(embedding_early_kernel<VECTOR, WIDE, false>, fill_ctas + position_ctas,
                             kEarlyThreads, 0, p.dtable != nullptr, cs, p, type_bytes(p.table_type),
                             (int)fill_ctas, 0))
    return st;
  if (p.dtable == nullptr) return ATTNRES_B200_OK;
  const int64_t tiles = (p.N + p.tile - 1) / p.tile;
  const auto [lanes, blocks] = columns_of(p.D, gradient_columns<VECTOR>());
  const int64_t units = tiles * blocks;
  const int per_cta = kSumThreads / lanes;
  embedding_sum_kernel<VECTOR, WIDE>
      <<<(unsigned)((units + per_cta - 1) / per_cta), kSumThreads, 0, cs>>>(p, lanes, blocks, tiles);
  if (int st = launched()) return st;
  if (tiles == 1) return ATTNRES_B200_OK;
  constexpr int warps = kEmbedThreads / 32;
  const int64_t joins = (units + warps - 1) / warps;
  return launch_behind(embedding_join_kernel<VECTOR>, joins < 2 * sms ? joins : 2 * sms,
                       kEmbedThreads, 0, true, cs, p, lanes, blocks, tiles);
}

int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace
}  // namespace attnres_b200

using namespace attnres_b200;

extern "C" int attnres_b200_embedding_forward(
    const void* tokens, int32_t tokens_64, int64_t N, int64_t T, int32_t V, int32_t D,
    const void* table, int64_t table_row_stride, int32_t table_type, const void* positions,
    int64_t position_row_stride, int32_t position_type, float scale, void* out, int32_t out_type,
    void* stream) {
  if (int st = check_embedding(N, T, V, D, table_type, out_type, position_type, scale)) return st;
  if (!tokens || !table || !out) return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned_type(table, table_type) || !aligned_type(positions, position_type) ||
      !aligned_type(out, out_type) ||
      (reinterpret_cast<uintptr_t>(tokens) & (tokens_64 ? 7u : 3u)) != 0)
    return ATTNRES_B200_ERR_MISALIGNED;
  EmbedParams p{};
  p.tokens = tokens;
  p.tokens_64 = tokens_64;
  p.V = V;
  p.N = N;
  p.T = T;
  p.D = D;
  p.scale = scale;
  p.table = table;
  p.table_row_stride = table_row_stride;
  p.table_type = table_type;
  p.positions = positions;
  p.position_row_stride = position_row_stride;
  p.position_type = position_type;
  p.out = out;
  p.out_type = out_type;
  const bool vector = D % 8 == 0 && aligned16(table) && table_row_stride % 8 == 0 &&
                      aligned16(out) &&
                      (!positions || (aligned16(positions) && position_row_stride % 8 == 0));
  const auto [lanes, blocks] = columns_of(D, 8);
  const int rows = kEmbedThreads / lanes;
  const dim3 grid((unsigned)((N + rows - 1) / rows),
                  (unsigned)((blocks + kEmbedBlocks - 1) / kEmbedBlocks));
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (table_type == ATTNRES_B200_FP32)
    return vector ? launch_embedding_forward<true, true>(p, lanes, grid, cs)
                  : launch_embedding_forward<false, true>(p, lanes, grid, cs);
  return vector ? launch_embedding_forward<true, false>(p, lanes, grid, cs)
                : launch_embedding_forward<false, false>(p, lanes, grid, cs);
}

extern "C" int64_t attnres_b200_embedding_workspace_bytes(int64_t N, int32_t D) {
  if (D < 1 || D > kMaxWidth) return -ATTNRES_B200_ERR_BAD_WIDTH;
  if (N < 1 || N > kMaxTokens) return -ATTNRES_B200_ERR_BAD_ROWS;
  const int64_t tile = tile_pairs(N), tiles = (N + tile - 1) / tile;
  return 2 * align256(N * (int64_t)sizeof(uint2)) + align256((tiles + 1) * (int64_t)sizeof(int32_t)) +
         tiles * 2 * D * (int64_t)sizeof(float);
}

extern "C" int attnres_b200_embedding_backward(
    const void* tokens, int32_t tokens_64, int64_t N, int64_t T, int32_t V, int32_t D,
    int64_t padding_id, const void* grad, int64_t grad_row_stride, int32_t grad_type, float scale,
    void* dtable, int32_t table_type, void* dpositions, int32_t position_type, void* workspace,
    int64_t workspace_bytes, void* stream) {
  if (int st = check_embedding(N, T, V, D, table_type, grad_type, position_type, scale)) return st;
  if (!dtable && !dpositions) return ATTNRES_B200_ERR_NOTHING_TO_DO;
  if (!tokens || !grad || (dtable && !workspace)) return ATTNRES_B200_ERR_NULL_POINTER;
  if (!aligned_type(grad, grad_type) || !aligned_type(dtable, table_type) ||
      !aligned_type(dpositions, position_type) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(tokens) & (tokens_64 ? 7u : 3u)) != 0)
    return ATTNRES_B200_ERR_MISALIGNED;
  if (dtable && workspace_bytes < attnres_b200_embedding_workspace_bytes(N, D))
    return ATTNRES_B200_ERR_WORKSPACE;
  int device = 0, sms = 0;
  if (int st = current_device(&device)) return st;
  if (int st = sm_count(device, &sms)) return st;
  EmbedParams p{};
  p.tokens = tokens;
  p.tokens_64 = tokens_64;
  p.V = V;
  p.N = N;
  p.T = T;
  p.padding = padding_id;
  p.D = D;
  p.scale = scale;
  p.out_type = grad_type;
  p.grad = grad;
  p.grad_row_stride = grad_row_stride;
  p.dtable = dtable;
  p.table_type = table_type;
  p.dpositions = dpositions;
  p.position_type = position_type;
  p.pairs[0] = static_cast<uint2*>(workspace);
  p.pairs[1] = reinterpret_cast<uint2*>(static_cast<char*>(workspace) +
                                        align256(N * (int64_t)sizeof(uint2)));
  p.tile = (int32_t)tile_pairs(N);
  const int64_t tiles = (N + p.tile - 1) / p.tile;
  char* rest = static_cast<char*>(workspace) + 2 * align256(N * (int64_t)sizeof(uint2));
  p.runs = reinterpret_cast<int32_t*>(rest);
  p.pieces = reinterpret_cast<float*>(rest + align256((tiles + 1) * (int64_t)sizeof(int32_t)));
  int bits = 1;  // of the ids and of V itself, which marks a token without a gradient
  while ((V >> bits) != 0) ++bits;
  p.passes = (bits + kSortMaxDigitBits - 1) / kSortMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const bool vector = D % 8 == 0 && aligned16(grad) && (N == 1 || grad_row_stride % 8 == 0) &&
                      (!dtable || aligned16(dtable)) && (!dpositions || aligned16(dpositions));
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (grad_type == ATTNRES_B200_FP32)
    return vector ? launch_embedding_backward<true, true>(p, sms, cs)
                  : launch_embedding_backward<false, true>(p, sms, cs);
  return vector ? launch_embedding_backward<true, false>(p, sms, cs)
                : launch_embedding_backward<false, false>(p, sms, cs);
}
