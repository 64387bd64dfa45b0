// extern "C" entry points of the 8-bit format with a scale per block of 128 (fp8.h):
// argument checks, the plan of the expert FFN, and dispatch.
#include <algorithm>
#include <climits>

#include "capi_detail.h"
#include "fp8.h"

using namespace moe355;

namespace {

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

int check_matrix(long long rows, int cols) {
  if (rows < 0 || cols <= 0) return fail(MOE355_EINVAL, "bad sizes %lld x %d", rows, cols);
  if (cols > (1 << 20)) return fail(MOE355_EUNSUPPORTED, "%d columns, at most 2^20", cols);
  return MOE355_OK;
}

int check_weights(int N, int K, int E) {
  if (int rc = check_matrix(N, K)) return rc;
  if (N == 0) return fail(MOE355_EINVAL, "bad N=%d", N);
  if (E < 1 || E > MOE355_MAX_EXPERTS)
    return fail(MOE355_EUNSUPPORTED, "E=%d outside [1, %d]", E, MOE355_MAX_EXPERTS);
  // the kernels address a matrix by 31-bit offsets
  if (static_cast<long long>(f8_pad(N)) * f8_pad(K) > INT_MAX)
    return fail(MOE355_EUNSUPPORTED, "a matrix of %d x %d is over 2 GB", N, K);
  return MOE355_OK;
}

int check_rows(int M, int dtype) {
  if (M < 0) return fail(MOE355_EINVAL, "bad M=%d", M);
  if (M > INT_MAX / 2) return fail(MOE355_EUNSUPPORTED, "M=%d too large", M);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  return MOE355_OK;
}

hipError_t launch_matmul(const F8Path& p, const F8MatmulArgs& a, bool gate_up, hipStream_t s) {
  return p.tile_rows ? launch_f8_tiled(a, gate_up, p.tile_rows, s) : launch_f8_stream(a, gate_up, s);
}

// Where the data of an expert call lies in the workspace.
struct F8Plan {
  int rows, n_blocks, max_tiles;
  F8Experts path;
  size_t block_counts, offsets, slot_to_row, row_src, tile_map, xq, xq_scales, inter, inter_scales,
      y, y_scales, parts, bytes;
};

int y_blocks(int H) { return (H + kScaled16Block - 1) / kScaled16Block; }

int f8_plan(int T, int H, int I, int E, int K, int dtype, F8Plan* p) {
  if (T < 0) return fail(MOE355_EINVAL, "bad T=%d", T);
  if (H <= 0 || I <= 0) return fail(MOE355_EINVAL, "bad sizes H=%d I=%d", H, I);
  if (H % 16 || I % 16) return fail(MOE355_EUNSUPPORTED, "H=%d and I=%d must be multiples of 16", H, I);
  if (H > (1 << 20) || I > (1 << 19)) return fail(MOE355_EUNSUPPORTED, "H=%d or I=%d over 2^20 / 2^19", H, I);
  if (int rc = check_weights(2 * f8_pad(I), H, E)) return rc;
  if (int rc = check_weights(H, I, E)) return rc;
  if (K < 1 || K > E) return fail(MOE355_EINVAL, "top-k K=%d outside [1, E=%d]", K, E);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  const long long R = static_cast<long long>(T) * K;
  if (R > INT_MAX / 2) return fail(MOE355_EUNSUPPORTED, "T*K=%lld too large", R);
  *p = F8Plan{};
  p->rows = static_cast<int>(R);
  p->n_blocks = R <= kPermuteSingleMax ? 1 : static_cast<int>((R + kPermuteChunk - 1) / kPermuteChunk);
  p->max_tiles = E + p->rows / kF8StreamTile;
  p->path = f8_experts(p->rows, H, I, E, K, dtype, device_cu_count());
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align256(off + bytes);
    return at;
  };
  p->block_counts = take(static_cast<size_t>(p->n_blocks) * E * 4);
  p->offsets = take(static_cast<size_t>(E + 1) * 4);
  p->slot_to_row = take(static_cast<size_t>(R) * 4);
  p->row_src = take(static_cast<size_t>(R) * 4);
  p->tile_map = take((2 + 2 * static_cast<size_t>(p->max_tiles)) * 4);
  p->xq = take(static_cast<size_t>(T) * f8_pad(H));
  p->xq_scales = take(static_cast<size_t>(T) * f8_blocks(H) * 4);
  p->inter = take(static_cast<size_t>(R) * f8_pad(I));
  p->inter_scales = take(static_cast<size_t>(R) * f8_blocks(I) * 4);
  p->y = take(static_cast<size_t>(R) * H * (p->path.narrow ? 2 : 4));
  p->y_scales = take(p->path.narrow ? static_cast<size_t>(R) * y_blocks(H) : 0);
  p->parts = take(std::max(p->path.up.part_bytes, p->path.down.part_bytes));
  p->bytes = off;
  return MOE355_OK;
}

// Token rows gathered by the kernels lie at 31-bit offsets: a call of more 8-bit bytes
// than that runs in parts.
int max_tokens(int H) { return INT_MAX / f8_pad(H); }

}  // namespace

extern "C" {

int moe355_fp8_quantize(const void* x, int M, int K, int dtype, void* codes, float* scales,
                        void* stream) {
  if (int rc = check_matrix(M, K)) return rc;
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  // a launch holds less than 2^32 threads, 256 for 16 blocks or the rest of them
  if (static_cast<long long>(M) * f8_blocks(K) > (1 << 28) - 16)
    return fail(MOE355_EUNSUPPORTED, "M=%d rows of K=%d: a call takes less than 2^28 blocks, 2^28 - 16 at most",
                M, K);
  if (M == 0) return MOE355_OK;
  if (!x || !codes || !scales) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (reinterpret_cast<uintptr_t>(x) % elem_size(dtype) || !aligned16(codes) || !aligned4(scales))
    return fail(MOE355_EINVAL, "x/codes/scales not aligned");
  F8QuantArgs a{x, static_cast<uint8_t*>(codes), scales, M, K};
  return check_hip(launch_f8_quantize(a, dtype, as_stream(stream)), "fp8_quantize launch");
}

int moe355_fp8_quantize_weight(const void* w, int N, int K, int dtype, void* cells, float* scales,
                               void* stream) {
  if (int rc = check_weights(N, K, 1)) return rc;
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  if (f8_blocks(N) > 65535) return fail(MOE355_EUNSUPPORTED, "N=%d too large", N);
  if (!w || !cells || !scales) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (reinterpret_cast<uintptr_t>(w) % elem_size(dtype) || !aligned16(cells) || !aligned4(scales))
    return fail(MOE355_EINVAL, "w/cells/scales not aligned");
  F8QuantArgs a{w, static_cast<uint8_t*>(cells), scales, N, K};
  return check_hip(launch_f8_quantize_weight(a, dtype, as_stream(stream)), "fp8_quantize_weight launch");
}

int moe355_fp8_pack(const void* codes, int N, int K, void* cells, void* stream) {
  if (int rc = check_weights(N, K, 1)) return rc;
  if (!codes || !cells) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(cells)) return fail(MOE355_EINVAL, "cells not 16-byte aligned");
  F8PackArgs a{static_cast<const uint8_t*>(codes), static_cast<uint8_t*>(cells), N, K};
  return check_hip(launch_f8_pack(a, as_stream(stream)), "fp8_pack launch");
}

int moe355_fp8_matmul_workspace_bytes(int M, int N, int K, int E, int dtype, size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  if (int rc = check_weights(N, K, E)) return rc;
  if (int rc = check_rows(M, dtype)) return rc;
  *bytes = M == 0 ? 0 : f8_path(M, N, f8_pad(K), E, dtype == MOE355_F32, device_cu_count()).part_bytes;
  return MOE355_OK;
}

int moe355_fp8_matmul(const void* x, const float* x_scales, const void* w, const float* w_scales,
                      const int32_t* offsets, int M, int N, int K, int E, int dtype, void* out,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_weights(N, K, E)) return rc;
  if (int rc = check_rows(M, dtype)) return rc;
  if (!offsets && E != 1) return fail(MOE355_EINVAL, "%d matrices without offsets", E);
  if (M == 0) return MOE355_OK;
  if (!x || !x_scales || !w || !w_scales || !out) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(x) || !aligned16(w) || !aligned4(x_scales) || !aligned4(w_scales) ||
      !aligned4(offsets) || !aligned16(out) || !aligned16(workspace))
    return fail(MOE355_EINVAL, "x/w/scales/offsets/out/workspace not aligned");
  const F8Path p = f8_path(M, N, f8_pad(K), E, dtype == MOE355_F32, device_cu_count());
  if (p.part_bytes > 0 && (!workspace || workspace_bytes < p.part_bytes))
    return fail(MOE355_EWORKSPACE, "workspace of %zu bytes, the call needs %zu", workspace_bytes,
                p.part_bytes);
  F8MatmulArgs a{};
  a.x = static_cast<const uint8_t*>(x); a.x_scales = x_scales; a.offsets = offsets;
  a.w = static_cast<const uint8_t*>(w); a.w_scales = w_scales; a.out = out;
  a.M = M; a.N = N; a.Kp = f8_pad(K); a.E = E; a.out_dtype = dtype; a.zero_rest = 1;
  a.exact = dtype == MOE355_F32;
  a.parts = static_cast<float*>(workspace); a.max_parts = p.max_parts;
  return check_hip(launch_matmul(p, a, false, as_stream(stream)), "fp8_matmul launch");
}

int moe355_fp8_workspace_bytes(int T, int H, int I, int E, int K, int dtype, size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  F8Plan p;
  const int most = H > 0 ? max_tokens(H) : T;
  if (int rc = f8_plan(std::min(T, most), H, I, E, K, dtype, &p)) return rc;
  if (static_cast<long long>(T) * K > INT_MAX / 2)
    return fail(MOE355_EUNSUPPORTED, "T*K=%lld too large", static_cast<long long>(T) * K);
  *bytes = p.bytes;
  if (T > most) {  // the last part has fewer rows, which may take other kernels and more memory
    if (int rc = f8_plan(T % most, H, I, E, K, dtype, &p)) return rc;
    *bytes = std::max(*bytes, p.bytes);
  }
  return MOE355_OK;
}

int moe355_fp8_fused_experts(const void* x, const float* x_scales, const void* w1,
                             const float* w1_scales, const void* w2, const float* w2_scales,
                             const float* topk_w, const void* topk_ids, int ids_int64, int T, int H,
                             int I, int E, int K, int dtype, int act, void* out, void* workspace,
                             size_t workspace_bytes, void* stream) {
  size_t bytes;
  if (int rc = moe355_fp8_workspace_bytes(T, H, I, E, K, dtype, &bytes)) return rc;
  if (act < MOE355_ACT_SILU || act > MOE355_ACT_GELU_TANH)
    return fail(MOE355_EINVAL, "unknown activation %d", act);
  if (T == 0) return MOE355_OK;
  if (!x || !w1 || !w1_scales || !w2 || !w2_scales || !topk_w || !topk_ids || !out)
    return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(x) || !aligned16(w1) || !aligned4(w1_scales) || !aligned16(w2) ||
      !aligned4(w2_scales) || !aligned16(out) || !aligned4(x_scales))
    return fail(MOE355_EINVAL, "x/w1/w2/scales/out not aligned");
  if (!workspace || workspace_bytes < bytes)
    return fail(MOE355_EWORKSPACE, "workspace of %zu bytes, the call needs %zu", workspace_bytes,
                bytes);
  if (!aligned16(workspace)) return fail(MOE355_EINVAL, "workspace not 16-byte aligned");
  const hipStream_t s = as_stream(stream);
  const int Hp = f8_pad(H), esz = elem_size(dtype);
  for (int t = 0; t < T; t += max_tokens(H)) {
    const int n = std::min(T - t, max_tokens(H));
    F8Plan p;
    if (int rc = f8_plan(n, H, I, E, K, dtype, &p)) return rc;
    const size_t first = t;
    const float* weights = topk_w + first * K;

    F8MatmulArgs a{};
    F8QuantArgs qa{};
    if (x_scales) {
      a.x = static_cast<const uint8_t*>(x) + first * Hp;
      a.x_scales = x_scales + first * (Hp / kF8Block);
    } else {
      qa = F8QuantArgs{static_cast<const char*>(x) + first * H * esz, at<uint8_t>(workspace, p.xq),
                       at<float>(workspace, p.xq_scales), n, H};
      a.x = qa.codes;
      a.x_scales = qa.scales;
    }
    PermuteArgs pa{};
    pa.ids = static_cast<const char*>(topk_ids) + first * K * (ids_int64 ? 8 : 4);
    pa.block_counts = at<int32_t>(workspace, p.block_counts);
    pa.offsets = at<int32_t>(workspace, p.offsets);
    pa.slot_to_row = at<int32_t>(workspace, p.slot_to_row);
    pa.row_src = at<int32_t>(workspace, p.row_src);
    pa.tile_map = at<int32_t>(workspace, p.tile_map);
    pa.R = p.rows; pa.K = K; pa.E = E; pa.n_blocks = p.n_blocks;
    pa.tile_rows = kF8StreamTile; pa.max_tiles = p.max_tiles;
    pa.ids_int64 = ids_int64 != 0;
    pa.weights = weights;
    if (int rc = check_hip(launch_f8_prepare(pa, qa, dtype, s), "fp8 prepare launch")) return rc;

    a.row_src = pa.row_src; a.offsets = pa.offsets;
    a.w = static_cast<const uint8_t*>(w1); a.w_scales = w1_scales;
    a.out_codes = at<uint8_t>(workspace, p.inter);
    a.out_scales = at<float>(workspace, p.inter_scales);
    a.M = p.rows; a.N = 2 * I; a.Kp = Hp; a.E = E; a.act = act;
    a.parts = at<float>(workspace, p.parts); a.max_parts = p.path.up.max_parts; a.exact = p.path.exact_up;
    if (int rc = check_hip(launch_matmul(p.path.up, a, true, s), "fp8 gate_up launch")) return rc;

    F8MatmulArgs d{};
    d.x = a.out_codes; d.x_scales = a.out_scales; d.offsets = pa.offsets;
    d.w = static_cast<const uint8_t*>(w2); d.w_scales = w2_scales;
    d.out = at<void>(workspace, p.y);
    d.M = p.rows; d.N = H; d.Kp = f8_pad(I); d.E = E; d.out_dtype = MOE355_F32;
    if (p.path.narrow) d.slot_scales = at<uint8_t>(workspace, p.y_scales);
    d.parts = a.parts; d.max_parts = p.path.down.max_parts; d.exact = p.path.exact_down;
    if (int rc = check_hip(launch_matmul(p.path.down, d, false, s), "fp8 down launch")) return rc;

    CombineArgs c{};
    c.y = d.out; c.topk_w = weights; c.slot_to_row = pa.slot_to_row;
    c.out = static_cast<char*>(out) + first * H * esz;
    c.T = n; c.K = K; c.H = H; c.R = p.rows; c.splits = 1;
    c.y16 = p.path.narrow; c.y_scales = d.slot_scales; c.y_blocks = y_blocks(H);
    if (int rc = check_hip(launch_combine(c, dtype, s), "combine launch")) return rc;
  }
  return MOE355_OK;
}

}  // extern "C"
