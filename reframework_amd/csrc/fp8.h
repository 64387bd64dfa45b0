// Values in 8 bits (e4m3 codes, largest magnitude 448) with fp32 scales: rows have a scale
// per 128 consecutive values, weights one per 128 x 128 block, blocks starting at multiples of
// 128. With m the block's largest finite magnitude, at least 448 * 2^-126, its scale is m / 448
// and a value's code is v * 448 / m rounded to nearest even. The quotient is formed from m, not
// from the rounded scale: 16-bit values over 16-bit maxima are often ties, and
// those would fall to the side the scale was rounded to. Infinities and NaN become NaN.
//
// Rows of tokens are padded to whole 128-value steps with codes of 0, so that the matrix kernels
// never see a partial step. Matrices are laid out once, as cells of 128 x 128 codes (16 KB, one
// scale) in rows of cells, padded with codes of 0. A cell holds 8 tiles of 16 rows (2 KB), each as
// the matrix instruction takes it: lane 16 q + r has row r, columns 16 q .. + 15 in the
// first KB and 64 + 16 q .. + 15 in the second. So every load of a wave is 1 KB in a row, and a
// workgroup's step 16 or 32. Row by row, a step's 256 rows are as many pieces of 128 bytes: loaded
// to LDS by one workgroup a CU that way 3.8 TB/s, as cells 4.9, by two 4.2 and 6.1.
#pragma once

#include "common.h"
#include "fp8_path.h"

namespace moe355 {

// What a value times 448 is divided by, of a block's largest finite magnitude. Where the
// product could overflow (of fp32 values) both are brought down by 2^-64.
struct F8Div {
  float mul, by, inv, scale;
};

__device__ __forceinline__ F8Div f8_div(float amax) {
  const float m = fmaxf(amax, 448.0f * 0x1p-126f);
  const bool large = m > 0x1p100f;
  const float by = large ? m * 0x1p-64f : m;
  return F8Div{large ? 448.0f * 0x1p-64f : 448.0f, by, __builtin_amdgcn_rcpf(by), m / 448.0f};
}

__device__ __forceinline__ float f8_finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}

// v over its block's scale; NaN of infinities and NaN. One correction of the product with the
// reciprocal by its remainder, which is exact: where the quotient has few bits, as a tie between
// two codes has, it comes out as it is. The product with 448 of a 24-bit value is rounded, so
// that the largest may come out a little over 448, which the conversion rounds to 448. (A
// division by the compiler takes three times the instructions: 8192 x 4096 bf16 29 us, so 27.)
__device__ __forceinline__ float f8_quotient(float v, const F8Div& d) {
  const float n = v * d.mul, q = n * d.inv;
  return fmaf(fmaf(-q, d.by, n), d.inv, q);
}

// Codes of four values, the first in the low byte.
__device__ __forceinline__ uint32_t f8_codes4(const float* v, const F8Div& d) {
  int c = 0;
  c = __builtin_amdgcn_cvt_pk_fp8_f32(f8_quotient(v[0], d), f8_quotient(v[1], d), c, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(f8_quotient(v[2], d), f8_quotient(v[3], d), c, true);
  return static_cast<uint32_t>(c);
}

constexpr int kF8Cell = kF8Block * kF8Block;  // bytes
constexpr int kF8Tile = 16 * kF8Block;

// Place in its matrix of the 16 codes of row n from column k on (a multiple of 16).
__host__ __device__ __forceinline__ size_t f8_place(int n, int k, int k_blocks) {
  const size_t cell = static_cast<size_t>(n / kF8Block) * k_blocks + k / kF8Block;
  const int q = k / 16 % 4, half = k / 64 % 2;
  return cell * kF8Cell + n % kF8Block / 16 * kF8Tile + half * (kF8Tile / 2) + (16 * q + n % 16) * 16;
}

struct F8QuantArgs {
  const void* x;    // [M, K]
  uint8_t* codes;   // rows: [M, Kp]; weights: cells
  float* scales;    // rows: [M, blocks]; weights: [row blocks, blocks]
  int M, K;
};

struct F8PackArgs {
  const uint8_t* src;  // codes [N, K]
  uint8_t* cells;
  int N, K;
};

// Rows of cells of a matrix of n rows; gate_up: of gate's and up's together.
__host__ __device__ constexpr int f8_cell_rows(int n, bool gate_up) {
  return gate_up ? 2 * f8_blocks(n / 2) : f8_blocks(n);
}

// One product, grouped: rows [offsets[e], offsets[e + 1]) of x times matrix e, transposed.
struct F8MatmulArgs {
  const uint8_t* x;        // [*, Kp]
  const float* x_scales;   // [*, blocks of K]
  const int32_t* row_src;  // x row of each row, or nullptr: the row itself
  const int32_t* offsets;  // [E + 1], or nullptr: one matrix, all rows
  const uint8_t* w;        // [E] matrices of cells (gate_up: gate's, then up's)
  const float* w_scales;   // [E, blocks of N, blocks of K]; gate_up: of I twice
  void* out;               // [M, N] (out_dtype)
  uint8_t* slot_scales;    // 256-row tiles, with it: out is Scaled16 with bytes [M, ceil(N/64)]
  uint8_t* out_codes;      // gate_up: [M, Ip]
  float* out_scales;       // gate_up: [M, blocks of I]
  int M, N, Kp, E;         // gate_up: N = 2 I
  int out_dtype, act;
  int exact;               // products in bf16 (fp8_mma.h); out_dtype is fp32 then
  int zero_rest;           // rows of no matrix become zeros in out
  float* parts;            // tiled: sums of parts of the last round's items
  int max_parts;           // room there, 0: items are not cut
};

hipError_t launch_f8_quantize(const F8QuantArgs& a, int dtype, hipStream_t s);
// The first launches of an expert call: slots grouped by expert, and x quantised beside that
// (x.x NULL: it is in 8 bits already).
hipError_t launch_f8_prepare(const PermuteArgs& p, const F8QuantArgs& x, int dtype, hipStream_t s);
hipError_t launch_f8_quantize_weight(const F8QuantArgs& a, int dtype, hipStream_t s);
hipError_t launch_f8_pack(const F8PackArgs& a, hipStream_t s);
// gate_up: out_codes, out_scales = act(gate) * up in 8 bits, of gate rows 0 .. I - 1 and up
// rows I .. 2 I - 1; else out.
hipError_t launch_f8_stream(const F8MatmulArgs& a, bool gate_up, hipStream_t s);
// tile_rows: 32, 64, 128 or 256 (not of exact products).
hipError_t launch_f8_tiled(const F8MatmulArgs& a, bool gate_up, int tile_rows, hipStream_t s);

}  // namespace moe355
