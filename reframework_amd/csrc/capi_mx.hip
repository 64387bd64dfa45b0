// extern "C" entry points of the 8-bit and 4-bit formats (mx.h) and of the routing
// by groups: argument checks, the plan of the expert FFN, and dispatch.
#include <algorithm>
#include <climits>
#include <cmath>

#include "capi_detail.h"
#include "mx.h"

using namespace moe355;

namespace {

bool bad_blocks(int n) { return n <= 0 || n % kMxBlock; }

// Average rows per active expert up to which the weights are streamed past 16-row
// tiles (ffn_mx.hip), and below which the tiled kernels (ffn_mx_tiled.hip) take tiles
// of 64 rows; from there on, 256 (exact products: 128). Whole calls of random routing, us.
// Streaming (exact) / 64 rows (scaled): 8 experts of H 4096, I 14336 at 8 rows 138 / 149, 10 rows
// 133 / 148, 12 rows 159 / 150, 14 rows 172 / 152, 20 rows 251 / 155; 64 of H 2048, I 1408 (6 slots)
// at 12 rows 70 / 75, 14 rows 78 / 76; 8 of H 2048, I 8192 at 10 rows 51 / 56, 12 rows 56 / 56; 32
// of H 1280, I 3328 (4 slots) at 12 rows 58 / 68, 16 rows 69 / 69.
// 64 / 256 rows: the taller tile costs more at the start
// and end of an item, which few columns do not hide. 16 experts of H 7168, I 2048 at 60 rows
// 134 / 121, 120 rows 171 / 148; 8 of H 4096, I 14336 at 60 rows 227 / 254, 75 rows 246 / 238,
// 135 rows 346 / 294; 64 of H 2048, I 1408 (6 slots) at 105 rows 120 / 126, 135 rows 150 / 137;
// 32 of H 1280, I 3328 (4 slots) at 180 rows 123 / 132, 200 rows 151 / 136; 16 of H 768, I
// 1536 at 180 rows 41 / 51, 220 rows 44 / 55.
// Exact products, 64 / 128 rows: the second at 160 rows 519 / 547, 230 rows 691 / 622, 420 rows
// 1159 / 1088; the third at 160 rows 261 / 272, 230 rows 333 / 323, 420 rows 565 / 527; the fourth
// at 230 rows 244 / 258, 300 rows 312 / 304.
// The rule goes by the mean, as the host does not know the routing. Where popularity is
// skewed, a call that streams reads a popular expert's weights once per 16 rows, from the
// caches: 128 tokens of 6 of 64 experts (H 2048, I 1408) 69 us, 73 where one expert is every
// token's; 48 of 2 of 8 (H 4096, I 14336) 151, 183; 256 of 8 of 256 (H 7168, I 2048) 1126, 1142.
constexpr int kMxStreamRows = 12, kMxTile64RowsExact = 224;
int tile64_rows(int steps, bool exact) {
  return exact ? kMxTile64RowsExact : std::min(std::max(2000 / steps, 56), 224);
}

// The stages of one expert call and where their data lies in the workspace.
struct MxPlan {
  int rows, n_blocks, tiled, tile_rows, max_tiles, down_splits, down_steps, y16;
  int Hp, Ip;
  size_t block_counts, offsets, slot_to_row, row_src, tile_map, xq, xq_scales, inter,
      inter_scales, y, y_scales, bytes;
};

int mx_plan(int T, int H, int I, int E, int K, int dtype, bool accumulate, MxPlan* p) {
  if (T < 0) return fail(MOE355_EINVAL, "bad T=%d", T);
  if (H <= 0 || I <= 0) return fail(MOE355_EINVAL, "bad sizes H=%d I=%d", H, I);
  if (bad_blocks(H) || bad_blocks(I))
    return fail(MOE355_EUNSUPPORTED, "H=%d and I=%d must be multiples of %d", H, I, kMxBlock);
  if (H > (1 << 20) || I > (1 << 20)) return fail(MOE355_EUNSUPPORTED, "H=%d or I=%d over 2^20", H, I);
  if (E < 1 || E > MOE355_MAX_EXPERTS)
    return fail(MOE355_EUNSUPPORTED, "E=%d outside [1, %d]", E, MOE355_MAX_EXPERTS);
  if (K < 1 || K > E) return fail(MOE355_EINVAL, "top-k K=%d outside [1, E=%d]", K, E);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  const long long R = static_cast<long long>(T) * K;
  if (R > INT_MAX / 2) return fail(MOE355_EUNSUPPORTED, "T*K=%lld too large", R);

  *p = MxPlan{};
  p->rows = static_cast<int>(R);
  p->Hp = mx_pad(H);
  p->Ip = mx_pad(I);
  p->n_blocks = R <= kPermuteSingleMax ? 1 : static_cast<int>((R + kPermuteChunk - 1) / kPermuteChunk);
  const int active = static_cast<int>(std::max<long long>(1, std::min<long long>(R, E)));
  const long long avg = R / active;
  p->tiled = avg > kMxStreamRows;
  const bool exact = dtype != MOE355_BF16;
  p->tile_rows = !p->tiled                                      ? kMxStreamTile
                 : avg < tile64_rows(p->Hp / kMxStep, exact) ? 64
                 : exact                                      ? 128
                                                              : 256;
  p->max_tiles = static_cast<int>((R + static_cast<long long>(active) * (p->tile_rows - 1)) / p->tile_rows);
  // A bf16 call of several slots per token keeps their results in 16 bits until they are
  // weighed and added: half the bytes (4096 tokens of 6 slots, H 2048: 259 us instead of
  // 286). They are f16 with a scale per 64 columns, whose 11 bits take the error of the
  // bf16 sum from 0.0017 of the results' size to 0.0018 (kept in bf16 it was 0.0024). Sums
  // that go on in fp32 keep fp32 slots: there the 11 bits would be most of the error.
  const bool narrow = p->tiled && !exact && K > 1 && !accumulate;
  const int steps = p->Ip / kMxStep;
  int s = 1;
  if (p->tiled) {
    // The columns of the down projection are cut where that shortens its rounds of
    // workgroups by more than the planes of y cost: a step of a CU takes 1.25 us on
    // 256-row tiles (and 128-row ones of exact products) and 0.85 on 64-row ones, an item 3 steps more, y 5 TB/s (us with 1 /
    // 2 / 4 parts: 8 experts of I 14336 at 49 rows 92 / 54 / 53, at 1085 rows 444 / 434 / 498;
    // 12 of H 1280, I 3328 at 83 rows 20.8 / 14.7 / 16.0).
    const double fill = static_cast<double>(R) / active / p->tile_rows;
    const double est = std::min<double>(p->max_tiles, active * (fill < 0.8 ? 1.0 : fill + 0.5));
    const long long items = static_cast<long long>((p->Hp + 255) / 256) * static_cast<long long>(est + 0.5);
    const int cus = device_cu_count();
    double best = 0.0;
    for (int c = 1; c <= 4 && steps >= 4 * c; c *= 2) {
      const double rounds = static_cast<double>((items * c + cus - 1) / cus);
      const double y_bytes = c == 1 && narrow ? 4.0 : 8.0 * c;
      const double us = rounds * ((steps + c - 1) / c + 3.0) * (p->tile_rows > 64 ? 1.25 : 0.85) +
                        static_cast<double>(R) * H * y_bytes / 5e6;
      if (c == 1 || us < 0.97 * best) {
        best = us;
        s = c;
      }
    }
  } else {
    // Columns of the down projection over workgroups, until there are 512 of them.
    const long long groups = static_cast<long long>(p->Hp / kMxSuper) * std::max(p->max_tiles, 1);
    while (s < 8 && groups * s < 512 && steps >= 8 * s) s *= 2;
  }
  p->down_splits = s;
  p->y16 = narrow && s == 1;
  p->down_steps = (steps + s - 1) / s;

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
  p->xq = take(static_cast<size_t>(T) * p->Hp);
  p->xq_scales = take(static_cast<size_t>(T) * p->Hp / kMxBlock);
  p->inter = take(static_cast<size_t>(R) * p->Ip);
  p->inter_scales = take(static_cast<size_t>(R) * p->Ip / kMxBlock);
  p->y = take(static_cast<size_t>(p->down_splits) * R * H * (p->y16 ? 2 : 4));
  p->y_scales = take(p->y16 ? static_cast<size_t>(R) * (p->Hp / kMxSuper) : 0);
  p->bytes = off;
  return MOE355_OK;
}

// The tiled kernels address token rows by 32-bit byte offsets whose bit 31 marks
// padding: a call of more 8-bit bytes than that runs in parts.
int max_tokens(int H) { return INT_MAX / mx_pad(H); }

// Bytes that a call of T tokens needs: those of its full parts or of its last one, whose
// plan may cut the columns into more parts.
int mx_bytes(int T, int H, int I, int E, int K, int dtype, bool accumulate, size_t* bytes) {
  MxPlan p;
  if (int rc = mx_plan(T, H, I, E, K, dtype, accumulate, &p)) return rc;
  if (T > max_tokens(H)) {
    const int rest = T % max_tokens(H);
    if (int rc = mx_plan(max_tokens(H), H, I, E, K, dtype, accumulate, &p)) return rc;
    *bytes = p.bytes;
    if (rest == 0) return MOE355_OK;
    if (int rc = mx_plan(rest, H, I, E, K, dtype, accumulate, &p)) return rc;
    *bytes = std::max(*bytes, p.bytes);
    return MOE355_OK;
  }
  *bytes = p.bytes;
  return MOE355_OK;
}

struct MxCall {
  const void* x;
  const uint8_t* x_scales;  // nullptr: x is to be quantised
  const uint8_t *w1, *w2;
  const uint32_t *w1_scales, *w2_scales;
  const float* topk_w;
  const void* topk_ids;
  void* out;
  int ids_int64, accumulate, T, H, E, K, dtype, act;
};

int mx_run(const MxPlan& p, const MxCall& a, void* workspace, hipStream_t s) {
  PermuteArgs pa{};
  pa.ids = a.topk_ids;
  pa.block_counts = at<int32_t>(workspace, p.block_counts);
  pa.offsets = at<int32_t>(workspace, p.offsets);
  pa.slot_to_row = at<int32_t>(workspace, p.slot_to_row);
  pa.row_src = at<int32_t>(workspace, p.row_src);
  pa.tile_map = at<int32_t>(workspace, p.tile_map);
  pa.R = p.rows; pa.K = a.K; pa.E = a.E; pa.n_blocks = p.n_blocks;
  pa.tile_rows = p.tile_rows; pa.max_tiles = p.max_tiles;
  pa.ids_int64 = a.ids_int64;
  pa.weights = a.topk_w;
  pa.full_tiles = 1;
  MxQuantArgs qa{};
  qa.T = a.T; qa.H = a.H; qa.Hp = p.Hp;
  if (!a.x_scales) {
    qa.x = a.x;
    qa.codes = at<uint8_t>(workspace, p.xq);
    qa.scales = at<uint8_t>(workspace, p.xq_scales);
  }
  if (int rc = check_hip(launch_mx_prepare(pa, qa, a.dtype, s), "mx prepare launch")) return rc;

  MxFfnArgs f{};
  f.row_src = pa.row_src; f.tile_map = pa.tile_map; f.offsets = pa.offsets;
  f.max_tiles = p.max_tiles; f.tile_rows = p.tile_rows;
  f.R = p.rows; f.H = a.H; f.Ip = p.Ip; f.act = a.act;
  // Tiled calls of a bf16 result take the scaled MFMA (mx_mma.h says what that costs the
  // result and saves in time); the others, and all streaming ones, exact products.
  f.exact = a.dtype != MOE355_BF16;
  f.out_codes = at<uint8_t>(workspace, p.inter);
  f.out_scales = at<uint8_t>(workspace, p.inter_scales);
  f.y = at<void>(workspace, p.y);
  f.y_scales = at<uint8_t>(workspace, p.y_scales);
  f.y16 = p.y16;

  f.x = a.x_scales ? static_cast<const uint8_t*>(a.x) : qa.codes;
  f.x_scales = a.x_scales ? a.x_scales : qa.scales;
  f.w = a.w1; f.w_scales = a.w1_scales;
  f.w_stride = mx_code_bytes(2 * p.Ip, p.Hp); f.ws_stride = mx_scale_bytes(2 * p.Ip, p.Hp) / 4;
  f.Kp = p.Hp; f.n_super = 2 * p.Ip / kMxSuper;
  f.splits = 1; f.steps_per_split = p.Hp / kMxStep;
  if (int rc = check_hip(p.tiled ? launch_mx_gate_up_tiled(f, s) : launch_mx_gate_up(f, s), "mx gate_up launch"))
    return rc;

  f.x = f.out_codes; f.x_scales = f.out_scales;
  f.w = a.w2; f.w_scales = a.w2_scales;
  f.w_stride = mx_code_bytes(p.Hp, p.Ip); f.ws_stride = mx_scale_bytes(p.Hp, p.Ip) / 4;
  f.Kp = p.Ip; f.n_super = p.Hp / kMxSuper;
  f.splits = p.down_splits; f.steps_per_split = p.down_steps;
  if (int rc = check_hip(p.tiled ? launch_mx_down_tiled(f, s) : launch_mx_down(f, s), "mx down launch"))
    return rc;

  CombineArgs c{};
  c.y = f.y; c.topk_w = a.topk_w; c.slot_to_row = pa.slot_to_row; c.out = a.out;
  c.T = a.T; c.K = a.K; c.H = a.H; c.R = p.rows; c.splits = p.down_splits;
  c.accumulate = a.accumulate;
  c.y16 = p.y16;
  if (p.y16) {
    c.y_scales = f.y_scales;
    c.y_blocks = f.n_super;
  }
  return check_hip(launch_combine(c, a.dtype, s), "combine launch");
}

}  // namespace

extern "C" {

int moe355_mx_quantize(const void* x, int T, int H, int dtype, void* codes, void* scales,
                       void* stream) {
  if (T < 0) return fail(MOE355_EINVAL, "bad T=%d", T);
  if (bad_blocks(H)) return fail(MOE355_EUNSUPPORTED, "H=%d must be a multiple of %d", H, kMxBlock);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  if (T == 0) return MOE355_OK;
  if (!x || !codes || !scales) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(x) || !aligned16(codes)) return fail(MOE355_EINVAL, "x/codes not 16-byte aligned");
  // In parts that a grid's 32 bits of threads hold.
  for (int t = 0; t < T; t += max_tokens(H)) {
    const size_t row = t, Hp = mx_pad(H);
    const MxQuantArgs a{static_cast<const char*>(x) + row * H * elem_size(dtype),
                        static_cast<uint8_t*>(codes) + row * Hp,
                        static_cast<uint8_t*>(scales) + row * (Hp / kMxBlock),
                        std::min(T - t, max_tokens(H)), H, mx_pad(H)};
    if (int rc = check_hip(launch_mx_quantize(a, dtype, as_stream(stream)), "mx_quantize launch")) return rc;
  }
  return MOE355_OK;
}

int moe355_add_rmsnorm_mxfp8(const void* x, const void* residual, void* residual_out,
                             const void* weight, const void* bias, int weight_dtype, float eps,
                             int T, int H, int dtype, void* normed_out, void* codes, void* scales,
                             void* stream) {
  if (T < 0 || H <= 0) return fail(MOE355_EINVAL, "bad sizes T=%d H=%d", T, H);
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype))
    return fail(MOE355_EINVAL, "unknown dtype %d / weight dtype %d", dtype, weight_dtype);
  if (bad_blocks(H) || H > norm_max_hidden(dtype))
    return fail(MOE355_EUNSUPPORTED, "norm with 8-bit rows needs H %% %d == 0 and H <= %d", kMxBlock,
                norm_max_hidden(dtype));
  if (!(eps >= 0.0f)) return fail(MOE355_EINVAL, "eps must be >= 0");
  if (T == 0) return MOE355_OK;
  if (!x || !weight || !normed_out || !codes || !scales)
    return fail(MOE355_EINVAL, "NULL tensor argument");
  if (residual && !residual_out) return fail(MOE355_EINVAL, "residual given without residual_out");
  if (!aligned16(x) || !aligned16(normed_out) || !aligned16(codes) ||
      (residual && (!aligned16(residual) || !aligned16(residual_out))))
    return fail(MOE355_EINVAL, "x/residual/out/codes not 16-byte aligned");
  if (!aligned16(weight) || (bias && !aligned16(bias)))
    return fail(MOE355_EINVAL, "norm weight/bias not 16-byte aligned");
  NormArgs a{};
  a.x = x; a.residual = residual; a.residual_out = residual_out; a.weight = weight;
  a.bias = bias; a.out = normed_out;
  a.T = T; a.H = H; a.weight_dtype = weight_dtype; a.eps = eps;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.Hp = mx_pad(H);
  return check_hip(launch_add_rmsnorm(a, dtype, as_stream(stream)), "add_rmsnorm_mxfp8 launch");
}

int moe355_grouped_topk(const float* logits, const float* bias, int T, int E, int K, int scoring,
                        int num_groups, int topk_groups, int group_score, int renormalize,
                        float scale, float* topk_w, void* topk_ids, int ids_int64, int out_ld,
                        void* stream) {
  if (T < 0) return fail(MOE355_EINVAL, "bad T=%d", T);
  if (E < 1 || E > MOE355_MAX_EXPERTS)
    return fail(MOE355_EUNSUPPORTED, "E=%d outside [1, %d]", E, MOE355_MAX_EXPERTS);
  if (scoring != MOE355_SCORE_SOFTMAX && scoring != MOE355_SCORE_SIGMOID)
    return fail(MOE355_EINVAL, "unknown scoring %d", scoring);
  if (group_score != MOE355_GROUP_MAX && group_score != MOE355_GROUP_TOP2)
    return fail(MOE355_EINVAL, "unknown group score %d", group_score);
  if (num_groups < 1 || E % num_groups)
    return fail(MOE355_EINVAL, "%d groups do not divide E=%d experts", num_groups, E);
  if (num_groups > MOE355_MAX_GROUPS)
    return fail(MOE355_EUNSUPPORTED, "%d groups, at most %d", num_groups, MOE355_MAX_GROUPS);
  if (topk_groups < 1 || topk_groups > num_groups)
    return fail(MOE355_EINVAL, "topk_groups=%d outside [1, %d]", topk_groups, num_groups);
  if (K < 1 || K > topk_groups * (E / num_groups))
    return fail(MOE355_EINVAL, "top-k K=%d outside [1, %d], the experts of %d groups", K,
                topk_groups * (E / num_groups), topk_groups);
  if (K > MOE355_MAX_GROUPED_TOPK)
    return fail(MOE355_EUNSUPPORTED, "top-k K=%d over %d", K, MOE355_MAX_GROUPED_TOPK);
  if (!std::isfinite(scale)) return fail(MOE355_EINVAL, "scale must be finite");
  if (out_ld < K) return fail(MOE355_EINVAL, "output row stride %d < K=%d", out_ld, K);
  if (T == 0) return MOE355_OK;
  if (!logits || !topk_w || !topk_ids) return fail(MOE355_EINVAL, "NULL tensor argument");
  GroupTopkArgs a{};
  a.logits = logits; a.bias = bias; a.topk_w = topk_w; a.topk_ids = topk_ids;
  a.T = T; a.E = E; a.K = K; a.G = num_groups; a.KG = topk_groups;
  a.sigmoid = scoring == MOE355_SCORE_SIGMOID;
  a.top2 = group_score == MOE355_GROUP_TOP2;
  a.renormalize = renormalize != 0; a.ids_int64 = ids_int64 != 0; a.out_ld = out_ld;
  a.scale = scale;
  return check_hip(launch_group_topk(a, as_stream(stream)), "grouped_topk launch");
}

int moe355_router_logits(const void* x, const void* gate, int T, int H, int E, int dtype,
                         int round_logits, float* logits_out, void* stream) {
  if (T < 0 || H <= 0) return fail(MOE355_EINVAL, "bad sizes T=%d H=%d", T, H);
  if (E < 1 || E > MOE355_MAX_EXPERTS)
    return fail(MOE355_EUNSUPPORTED, "E=%d outside [1, %d]", E, MOE355_MAX_EXPERTS);
  if (!valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  const int vec = 16 / elem_size(dtype);
  if (H % vec) return fail(MOE355_EUNSUPPORTED, "router needs H %% %d == 0", vec);
  if (T == 0) return MOE355_OK;
  if (!x || !gate || !logits_out) return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(x) || !aligned16(gate)) return fail(MOE355_EINVAL, "x/gate not 16-byte aligned");
  RouterArgs a{};
  a.x = x; a.gate = gate; a.logits_out = logits_out;
  a.T = T; a.H = H; a.E = E; a.K = 0; a.round_logits = round_logits != 0;
  return check_hip(launch_router_logits(a, dtype, as_stream(stream)), "router_logits launch");
}

int moe355_mx_matrix_bytes(int rows, int cols, int gate_up, size_t* codes, size_t* scales) {
  if (!codes || !scales) return fail(MOE355_EINVAL, "NULL result");
  if (rows <= 0 || (gate_up && rows % 2)) return fail(MOE355_EINVAL, "bad rows=%d", rows);
  if (bad_blocks(cols) || bad_blocks(gate_up ? rows / 2 : rows) || rows > (1 << 21) || cols > (1 << 20))
    return fail(MOE355_EUNSUPPORTED, "a 4-bit matrix of %d x %d: sizes must be multiples of %d", rows,
                cols, kMxBlock);
  const int rows_p = gate_up ? 2 * mx_pad(rows / 2) : mx_pad(rows);
  *codes = mx_code_bytes(rows_p, mx_pad(cols));
  *scales = mx_scale_bytes(rows_p, mx_pad(cols));
  return MOE355_OK;
}

int moe355_mx_pack(const void* src, const void* src_scales, int rows, int cols, int gate_up,
                   int dtype, void* codes, void* scales, void* stream) {
  size_t nc, ns;
  if (int rc = moe355_mx_matrix_bytes(rows, cols, gate_up, &nc, &ns)) return rc;
  const bool is_codes = dtype == MOE355_MX_CODES;
  if (!is_codes && !valid_dtype(dtype)) return fail(MOE355_EINVAL, "unknown dtype %d", dtype);
  if (!src || !codes || !scales || (is_codes && !src_scales))
    return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(codes) || (is_codes && !aligned16(src)) ||
      (!is_codes && reinterpret_cast<uintptr_t>(src) % elem_size(dtype)))
    return fail(MOE355_EINVAL, "src/codes not aligned");
  MxPackArgs a{};
  a.src = src; a.scales = static_cast<const uint8_t*>(src_scales);
  a.codes_out = static_cast<uint8_t*>(codes); a.scales_out = static_cast<uint8_t*>(scales);
  a.rows = rows; a.cols = cols;
  a.rows_p = gate_up ? 2 * mx_pad(rows / 2) : mx_pad(rows);
  a.cols_p = mx_pad(cols);
  a.gate_up = gate_up != 0;
  return check_hip(launch_mx_pack(a, is_codes ? -1 : dtype, as_stream(stream)), "mx_pack launch");
}

int moe355_mx_workspace_bytes(int T, int H, int I, int E, int K, int dtype, size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  size_t stored, added;
  if (int rc = mx_bytes(T, H, I, E, K, dtype, false, &stored)) return rc;
  if (int rc = mx_bytes(T, H, I, E, K, dtype, true, &added)) return rc;
  *bytes = std::max(stored, added);
  return MOE355_OK;
}

int moe355_mx_call_workspace_bytes(int T, int H, int I, int E, int K, int dtype, int accumulate_f32,
                                   size_t* bytes) {
  if (!bytes) return fail(MOE355_EINVAL, "NULL result");
  return mx_bytes(T, H, I, E, K, dtype, accumulate_f32 != 0, bytes);
}

int moe355_mx_fused_experts(const void* x, const void* x_scales, const void* w1,
                            const void* w1_scales, const void* w2, const void* w2_scales,
                            const float* topk_w, const void* topk_ids, int ids_int64, int T, int H,
                            int I, int E, int K, int dtype, int act, void* out, int accumulate_f32,
                            void* workspace, size_t workspace_bytes, void* stream) {
  size_t bytes;
  if (int rc = mx_bytes(T, H, I, E, K, dtype, accumulate_f32 != 0, &bytes)) return rc;
  if (act < MOE355_ACT_SILU || act > MOE355_ACT_GELU_TANH)
    return fail(MOE355_EINVAL, "unknown activation %d", act);
  if (T == 0) return MOE355_OK;
  if (!x || !w1 || !w1_scales || !w2 || !w2_scales || !topk_w || !topk_ids || !out)
    return fail(MOE355_EINVAL, "NULL tensor argument");
  if (!aligned16(x) || !aligned16(w1) || !aligned16(w1_scales) || !aligned16(w2) ||
      !aligned16(w2_scales) || !aligned16(out) ||
      (x_scales && reinterpret_cast<uintptr_t>(x_scales) % 4))
    return fail(MOE355_EINVAL, "x/w1/w2/scales/out not 16-byte aligned");
  if (!workspace || workspace_bytes < bytes)
    return fail(MOE355_EWORKSPACE, "workspace of %zu bytes, the call needs %zu", workspace_bytes,
                bytes);
  if (!aligned16(workspace)) return fail(MOE355_EINVAL, "workspace not 16-byte aligned");
  const size_t x_row = x_scales ? mx_pad(H) : static_cast<size_t>(H) * elem_size(dtype);
  const size_t out_row = static_cast<size_t>(H) * (accumulate_f32 ? 4 : elem_size(dtype));
  for (int t = 0; t < T; t += max_tokens(H)) {
    const int n = std::min(T - t, max_tokens(H));
    MxPlan p;
    if (int rc = mx_plan(n, H, I, E, K, dtype, accumulate_f32 != 0, &p)) return rc;
    MxCall c{};
    c.x = static_cast<const char*>(x) + t * x_row;
    c.x_scales = x_scales ? static_cast<const uint8_t*>(x_scales) + t * static_cast<size_t>(p.Hp / kMxBlock) : nullptr;
    c.w1 = static_cast<const uint8_t*>(w1); c.w1_scales = static_cast<const uint32_t*>(w1_scales);
    c.w2 = static_cast<const uint8_t*>(w2); c.w2_scales = static_cast<const uint32_t*>(w2_scales);
    c.topk_w = topk_w + static_cast<size_t>(t) * K;
    c.topk_ids = static_cast<const char*>(topk_ids) + static_cast<size_t>(t) * K * (ids_int64 ? 8 : 4);
    c.out = static_cast<char*>(out) + t * out_row;
    c.ids_int64 = ids_int64 != 0; c.accumulate = accumulate_f32 != 0;
    c.T = n; c.H = H; c.E = E; c.K = K; c.dtype = dtype; c.act = act;
    if (int rc = mx_run(p, c, workspace, as_stream(stream))) return rc;
  }
  return MOE355_OK;
}

}  // extern "C"
