// Kernel arguments and launchers of the row operators with gradients: LayerNorm
// (layer_norm.hip) and tokens in the order of their experts (tokens.hip).
#pragma once

#include "common.h"

namespace moe355 {

struct LayerNormArgs {
  const void* x;         // [T,H]
  const void* residual;  // [T,H] added to x, or nullptr
  void* residual_out;    // [T,H] x + residual (may alias x or residual)
  const void* weight;    // [H] (weight_dtype)
  const void* bias;      // [H] (weight_dtype) or nullptr
  void* out;             // [T,H]
  float* mean;           // [T] with rstd, or nullptr
  float* rstd;           // [T]
  int T, H, weight_dtype;
  float eps;
};

struct LayerNormBwdArgs {
  const void* dy;      // [T,H]
  const void* dres;    // [T,H] or nullptr
  const void* r;       // [T,H] what was normed
  const void* weight;  // [H] (weight_dtype)
  const float* mean;   // [T]
  const float* rstd;   // [T]
  void* dx;            // [T,H] or nullptr
  void* dw;            // [H] (weight_dtype) or nullptr
  void* db;            // [H] or nullptr
  float* part;         // [parts, 2, H], or nullptr without dw and db
  int T, H, weight_dtype;
};

struct TokenRowsArgs {
  const void* src;             // gather: tokens [T,H]; combine: rows [R,H]
  void* dst;                   // gather: rows [R,H]; combine: tokens [T,H]
  const float* topk_w;         // [T,K], or nullptr: 1
  const int32_t* slot_to_row;  // [T,K], -1: to no expert
  const int32_t* n_rows;       // rows that have a slot; the others become zeros
  int T, K, H, R;
};

struct CombineBwdArgs {
  const void* dout;            // [T,H]
  const void* rows;            // [R,H], needed for dw
  const float* topk_w;         // [T,K]
  const int32_t* slot_to_row;  // [T,K]
  const int32_t* n_rows;
  void* drows;                 // [R,H] or nullptr
  float* dw;                   // [T,K] or nullptr
  int T, K, H, R;
};

// Workgroups of the backward pass, each leaving one part of the sums over rows.
int layer_norm_bwd_parts(int T, int H, int dtype);
hipError_t launch_layer_norm(const LayerNormArgs& a, int dtype, hipStream_t s);
hipError_t launch_layer_norm_bwd(const LayerNormBwdArgs& a, int dtype, hipStream_t s);
hipError_t launch_permute_rows(const TokenRowsArgs& a, int dtype, hipStream_t s);
hipError_t launch_combine_rows(const TokenRowsArgs& a, int dtype, hipStream_t s);
hipError_t launch_combine_rows_bwd(const CombineBwdArgs& a, int dtype, hipStream_t s);

}  // namespace moe355
