// extern "C" entry points of the row operators with gradients (rows.h): LayerNorm, tokens
// in the order of their experts and back.
#include <climits>

#include "capi_detail.h"
#include "rows.h"

using namespace moe355;

namespace {

bool bad_element(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % elem_size(dtype) != 0;
}

int check_norm(int T, int H, int dtype, int weight_dtype) {
  if (T < 0 || H <= 0) return fail(MOE355_EINVAL, "bad sizes T=%d H=%d", T, H);
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype))
    return fail(MOE355_EINVAL, "unknown dtype %d / weight dtype %d", dtype, weight_dtype);
  if (H > norm_max_hidden(dtype))
    return fail(MOE355_EUNSUPPORTED, "LayerNorm needs H <= %d", norm_max_hidden(dtype));
  // a launch holds less than 2^32 threads, 256 a row
  if (T >= 1 << 24) return fail(MOE355_EUNSUPPORTED, "T=%d: a call takes less than 2^24 rows", T);
  return MOE355_OK;
}

int check_slots(int T, int K, int E, int H, int dtype) {
  if (T < 0 || K < 1) return fail(MOE355_EINVAL, "bad sizes T=%d K=%d", T, K);
  if (E < 1 || E > MOE355_MAX_EXPERTS)
    return fail(MOE355_EUNSUPPORTED, "E=%d outside [1, %d]", E, MOE355_MAX_EXPERTS);
  if (T >= 1 << 26) return fail(MOE355_EUNSUPPORTED, "T=%d: a call takes less than 2^26 tokens", T);
  if (static_cast<long long>(T) * K > INT_MAX / 2)
    return fail(MOE355_EUNSUPPORTED, "T*K=%lld too large", static_cast<long long>(T) * K);
  if (H <= 0) return fail(MOE355_EINVAL, "bad H=%d", H);
  if (H >= 1 << 24) return fail(MOE355_EUNSUPPORTED, "H=%d: rows are less than 2^24 wide", H);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  return MOE355_OK;
}

int check_moves(int T, int K, int E, int H, int dtype) {
  if (int rc = check_slots(T, K, E, H, dtype)) return rc;
  // a launch holds less than 2^32 threads, 256 for four tokens or the rest of them
  if (T > (1 << 26) - 4) return fail(MOE355_EUNSUPPORTED, "T=%d: a call moves 2^26 - 4 tokens at most", T);
  return MOE355_OK;
}

int order_blocks(int R) {
  return R <= kPermuteSingleMax ? 1 : (R + kPermuteChunk - 1) / kPermuteChunk;
}

// The permute also lists the experts' tiles; nothing reads that list here, so its tiles
// are as large as it may be.
constexpr int kOrderTileRows = 1 << 20;

int order_tiles(int R, int E) { return E + R / kOrderTileRows; }

size_t order_bytes(int R, int E) {
  return align256(static_cast<size_t>(order_blocks(R)) * E * 4) +
         (2 + 2 * static_cast<size_t>(order_tiles(R, E))) * 4;
}

}  // namespace

extern "C" {

int moe355_layer_norm(const void* x, const void* residual, void* residual_out, const void* weight,
                      const void* bias, int weight_dtype, float eps, int T, int H, int dtype,
                      void* out, float* mean, float* rstd, void* stream) {
  if (int rc = check_norm(T, H, dtype, weight_dtype)) return rc;
  if (!(eps >= 0.0f)) return fail(MOE355_EINVAL, "eps must be >= 0");
  if (T == 0) return MOE355_OK;
  if (!x || !weight || !out) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (residual && !residual_out) return fail(MOE355_EINVAL, "residual given without residual_out");
  if (!mean != !rstd) return fail(MOE355_EINVAL, "mean and rstd belong together");
  if (bad_element(x, dtype) || bad_element(residual, dtype) || bad_element(residual_out, dtype) ||
      bad_element(out, dtype) || bad_element(weight, weight_dtype) || bad_element(bias, weight_dtype))
    return fail(MOE355_EINVAL, "tensor not aligned to its elements");
  LayerNormArgs a{};
  a.x = x; a.residual = residual; a.residual_out = residual_out; a.weight = weight; a.bias = bias;
  a.out = out; a.mean = mean; a.rstd = rstd;
  a.T = T; a.H = H; a.weight_dtype = weight_dtype; a.eps = eps;
  return check_hip(launch_layer_norm(a, dtype, as_stream(stream)), "layer_norm launch");
}

int moe355_layer_norm_bwd_workspace_bytes(int T, int H, int dtype, size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  if (int rc = check_norm(T, H, dtype, dtype)) return rc;
  *bytes = static_cast<size_t>(layer_norm_bwd_parts(T, H, dtype)) * 2 * H * 4;
  return MOE355_OK;
}

int moe355_layer_norm_bwd(const void* dy, const void* dres, const void* r, const void* weight,
                          int weight_dtype, const float* mean, const float* rstd, int T, int H,
                          int dtype, void* dx, void* dw, void* db, void* workspace,
                          size_t workspace_bytes, void* stream) {
  size_t bytes;
  if (int rc = check_norm(T, H, dtype, weight_dtype)) return rc;
  if (int rc = moe355_layer_norm_bwd_workspace_bytes(T, H, dtype, &bytes)) return rc;
  if (T == 0) return fail(MOE355_EINVAL, "no rows to sum over");
  if (!dy || !r || !weight || !mean || !rstd) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (bad_element(dy, dtype) || bad_element(dres, dtype) || bad_element(r, dtype) ||
      bad_element(dx, dtype) || bad_element(weight, weight_dtype) ||
      bad_element(dw, weight_dtype) || bad_element(db, weight_dtype))
    return fail(MOE355_EINVAL, "tensor not aligned to its elements");
  if ((dw || db) && (!workspace || workspace_bytes < bytes))
    return fail(MOE355_EWORKSPACE, "workspace of %zu bytes, the call needs %zu", workspace_bytes,
                bytes);
  if (!aligned16(workspace)) return fail(MOE355_EINVAL, "workspace not 16-byte aligned");
  LayerNormBwdArgs a{};
  a.dy = dy; a.dres = dres; a.r = r; a.weight = weight; a.mean = mean; a.rstd = rstd;
  a.dx = dx; a.dw = dw; a.db = db;
  a.part = dw || db ? static_cast<float*>(workspace) : nullptr;
  a.T = T; a.H = H; a.weight_dtype = weight_dtype;
  return check_hip(launch_layer_norm_bwd(a, dtype, as_stream(stream)), "layer_norm_bwd launch");
}

int moe355_token_order_workspace_bytes(int T, int K, int E, size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  if (int rc = check_slots(T, K, E, 1, MOE355_F32)) return rc;
  *bytes = order_bytes(T * K, E);
  return MOE355_OK;
}

int moe355_token_order(const void* topk_ids, int ids_int64, int T, int K, int E, int32_t* offsets,
                       int32_t* slot_to_row, int32_t* row_src, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (int rc = check_slots(T, K, E, 1, MOE355_F32)) return rc;
  if (T == 0) return fail(MOE355_EINVAL, "no slots to order");
  if (!topk_ids || !offsets || !slot_to_row || !row_src)
    return fail(MOE355_EINVAL, "NULL tensor argument");
  const int R = T * K;
  if (!workspace || workspace_bytes < order_bytes(R, E))
    return fail(MOE355_EWORKSPACE, "workspace of %zu bytes, the call needs %zu", workspace_bytes,
                order_bytes(R, E));
  if (!aligned16(workspace)) return fail(MOE355_EINVAL, "workspace not 16-byte aligned");
  PermuteArgs a{};
  a.ids = topk_ids;
  a.n_blocks = order_blocks(R);
  a.block_counts = static_cast<int32_t*>(workspace);
  a.tile_map = at<int32_t>(workspace, align256(static_cast<size_t>(a.n_blocks) * E * 4));
  a.offsets = offsets; a.slot_to_row = slot_to_row; a.row_src = row_src;
  a.R = R; a.K = K; a.E = E;
  a.tile_rows = kOrderTileRows; a.max_tiles = order_tiles(R, E);
  a.ids_int64 = ids_int64 != 0;
  return check_hip(launch_permute(a, as_stream(stream)), "token_order launch");
}

int moe355_permute_rows(const void* x, const int32_t* offsets, const int32_t* slot_to_row, int T,
                        int H, int K, int E, int dtype, void* rows, void* stream) {
  if (int rc = check_moves(T, K, E, H, dtype)) return rc;
  if (T == 0) return MOE355_OK;
  if (!x || !offsets || !slot_to_row || !rows) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (bad_element(x, dtype) || bad_element(rows, dtype))
    return fail(MOE355_EINVAL, "tensor not aligned to its elements");
  TokenRowsArgs a{};
  a.src = x; a.dst = rows; a.slot_to_row = slot_to_row; a.n_rows = offsets + E;
  a.T = T; a.K = K; a.H = H; a.R = T * K;
  return check_hip(launch_permute_rows(a, dtype, as_stream(stream)), "permute_rows launch");
}

int moe355_combine_rows(const void* rows, const float* topk_w, const int32_t* slot_to_row, int T,
                        int H, int K, int dtype, void* out, void* stream) {
  if (int rc = check_moves(T, K, 1, H, dtype)) return rc;
  if (T == 0) return MOE355_OK;
  if (!rows || !slot_to_row || !out) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (bad_element(rows, dtype) || bad_element(out, dtype))
    return fail(MOE355_EINVAL, "tensor not aligned to its elements");
  TokenRowsArgs a{};
  a.src = rows; a.dst = out; a.topk_w = topk_w; a.slot_to_row = slot_to_row;
  a.T = T; a.K = K; a.H = H; a.R = T * K;
  return check_hip(launch_combine_rows(a, dtype, as_stream(stream)), "combine_rows launch");
}

int moe355_combine_rows_bwd(const void* dout, const void* rows, const float* topk_w,
                            const int32_t* offsets, const int32_t* slot_to_row, int T, int H, int K,
                            int E, int dtype, void* drows, float* dw, void* stream) {
  if (int rc = check_moves(T, K, E, H, dtype)) return rc;
  if (T == 0 || (!drows && !dw)) return MOE355_OK;
  if (!dout || !topk_w || !offsets || !slot_to_row || (dw && !rows))
    return fail(MOE355_EINVAL, "NULL tensor argument");
  if (bad_element(dout, dtype) || bad_element(rows, dtype) || bad_element(drows, dtype))
    return fail(MOE355_EINVAL, "tensor not aligned to its elements");
  CombineBwdArgs a{};
  a.dout = dout; a.rows = rows; a.topk_w = topk_w; a.slot_to_row = slot_to_row;
  a.n_rows = offsets + E; a.drows = drows; a.dw = dw;
  a.T = T; a.K = K; a.H = H; a.R = T * K;
  return check_hip(launch_combine_rows_bwd(a, dtype, as_stream(stream)), "combine_rows_bwd launch");
}

}  // extern "C"
