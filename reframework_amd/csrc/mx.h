// Formats with one power-of-two scale per 32 consecutive values of a row: 8 bits
// (e4m3 codes) for tokens and intermediates, 4 bits (e2m1 codes, two per byte, the
// even column in the low half) for expert weights. A scale is a byte b that
// stands for 2^(b - 127); in weights 255 stands for NaN.
//
// Rows of 8 bits are padded to whole 128-value steps with codes of 0, so that the
// matrix kernels never see a partial step.
//
// 4-bit matrices are laid out once, in the order in which the kernels stream them.
// A tile is 16 rows x 128 columns, 1 KB: lane 16 q + r of a wave holds row r,
// columns 32 q .. 32 q + 31 (one block, 16 bytes), which is the operand of
// v_mfma_scale_f32_16x16x128_f8f6f4 as it stands, so one load instruction fetches
// one tile from 1 KB of consecutive bytes and no lane moves data afterwards.
// Four groups of 16 rows make a supergroup, whose four tiles of a 128-column step
// follow each other (4 KB), then the next step's; its scales are one dword per lane
// and step, byte g for group g, so that a wave working on a supergroup loads all of
// a step's scales at once and the instruction picks its byte. A gate|up matrix is
// interleaved so that a supergroup holds one 32-value block of the intermediate: its
// groups are gate, up, gate, up, and row r of the first (second) pair is feature
// 8 (r / 4) + r % 4 (+ 4) of the block. The matrix core leaves rows 4 q .. 4 q + 3 of
// every group in lane q of a token, which so has features 8 q .. 8 q + 7, gate and
// up, and stores their codes as 8 consecutive bytes. Rows and columns are padded to
// multiples of 128 with zeros.
#pragma once

#include "common.h"

namespace moe355 {

constexpr int kMxBlock = 32;    // values per scale
constexpr int kMxStep = 128;    // columns per matrix instruction
constexpr int kMxSuper = 64;    // rows per supergroup
constexpr int kMxTileBytes = 1024;
constexpr int kMxStreamTile = 16;  // token rows of a tile of the weight-streaming kernels

__host__ __device__ constexpr int mx_pad(int n) { return (n + kMxStep - 1) / kMxStep * kMxStep; }

// Bytes of the codes and scales of a 4-bit matrix of [rows, cols], both padded.
__host__ __device__ constexpr size_t mx_code_bytes(int rows, int cols) {
  return static_cast<size_t>(rows) * cols / 2;
}
__host__ __device__ constexpr size_t mx_scale_bytes(int rows, int cols) {
  return static_cast<size_t>(rows) * cols / kMxBlock;
}

// Scale byte of a block whose largest finite magnitude is amax: the smallest power
// of two with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3 value), so
// that no value is clipped; 0 for a block of zeros. The addition carries into the
// exponent where the significand is over 1.75.
__device__ __forceinline__ int mx8_scale(float amax) {
  return max(static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8, 0);
}

// 2^(127 - b), the factor that brings a block's values to the range of the codes.
__device__ __forceinline__ float mx_inverse(int b) {
  return __uint_as_float(static_cast<uint32_t>(254 - b) << 23);
}

// Magnitude that counts for a block's scale: 0 for infinities and NaN, whose
// codes become NaN whatever the scale is.
__device__ __forceinline__ float mx_finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}

// Four or eight e4m3 codes of values of a block with scale byte b, rounded to nearest
// even; infinities and NaN become NaN. The conversion divides by 2^(b - 127), for
// b = 0 too (a probe over all bytes and 2^20 pairs of values found the codes of
// v * 2^(127 - b)).
typedef short mx_half2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t mx8_codes4(const float* v, int b) {
  const float s = __uint_as_float(static_cast<uint32_t>(b) << 23);
  mx_half2 c = {0, 0};
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[0], v[1], s, false);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[2], v[3], s, true);
  return __builtin_bit_cast(uint32_t, c);
}
__device__ __forceinline__ u32x2 mx8_codes(const float* v, int b) {
  return u32x2{mx8_codes4(v, b), mx8_codes4(v + 4, b)};
}

struct MxQuantArgs {
  const void* x;    // [T, H]
  uint8_t* codes;   // [T, Hp]
  uint8_t* scales;  // [T, Hp / 32]
  int T, H, Hp;
};

struct MxPackArgs {
  const void* src;        // codes [rows, cols / 2], or weights [rows, cols] to be rounded
  const uint8_t* scales;  // [rows, cols / 32] of codes
  uint8_t* codes_out;
  uint8_t* scales_out;
  int rows, cols;         // of the source
  int rows_p, cols_p;     // padded (both halves of a gate|up matrix each)
  int gate_up;            // rows 0 .. rows / 2 - 1 gate, the others up
};

struct MxFfnArgs {
  const uint8_t* x;         // token rows in 8 bits, [*, Kp]
  const uint8_t* x_scales;  // [*, Kp / 32]
  const int32_t* row_src;   // gate_up: x row of each permuted row
  const int32_t* tile_map;  // [2 + 2 * max_tiles]
  const int32_t* offsets;   // [E + 1]
  const uint8_t* w;         // 4-bit matrices, w_stride bytes apart
  const uint32_t* w_scales; // dwords, ws_stride apart
  size_t w_stride, ws_stride;
  int Kp, n_super;          // padded columns, supergroups of rows
  int max_tiles, tile_rows, splits, steps_per_split;
  int R, H;                 // down: rows and features of y
  void* y;                  // down: fp32 [splits, R, H], or Scaled16 [R, H] (y16: one split)
  uint8_t* y_scales;        // [R, n_super]
  int y16;
  uint8_t* out_codes;       // gate_up: [R, Ip]
  uint8_t* out_scales;      // [R, Ip / 32]
  int Ip, act;
  int exact;                // multiply in bf16 (exactly) instead of the scaled MFMA
};

hipError_t launch_mx_gate_up(const MxFfnArgs& a, hipStream_t s);
hipError_t launch_mx_down(const MxFfnArgs& a, hipStream_t s);
hipError_t launch_mx_gate_up_tiled(const MxFfnArgs& a, hipStream_t s);
hipError_t launch_mx_down_tiled(const MxFfnArgs& a, hipStream_t s);
// The first launch of an expert call: the routed slots grouped by expert (all of the
// permute up to kPermuteSingleMax slots, its counts above) by the first workgroups,
// x quantised by the others (x.x NULL: it is in 8 bits already).
hipError_t launch_mx_prepare(const PermuteArgs& p, const MxQuantArgs& x, int dtype, hipStream_t s);
hipError_t launch_mx_quantize(const MxQuantArgs& a, int dtype, hipStream_t s);
// dtype -1: src holds codes.
hipError_t launch_mx_pack(const MxPackArgs& a, int dtype, hipStream_t s);

}  // namespace moe355
