// The matrix products of 4-bit weights and 8-bit tokens and the epilogue of gate|up,
// shared by the weight-streaming (ffn_mx.hip) and the tiled kernels
// (ffn_mx_tiled.hip). Included inside their anonymous namespaces.
#pragma once

typedef int i32x8 __attribute__((ext_vector_type(8)));

// One 16-row tile times 16 tokens over 128 columns on the scaled MFMA: the
// instruction applies the blocks' scales. It aligns a step's products to their
// largest and keeps about 14 bits below it (measured: an error of 5e-6 of a sum's
// typical size for normal data); sums over the steps are in fp32. In gate|up this moves
// one intermediate in some thousands across a border of its 8-bit code. A bf16 result,
// whose rounding is off by 1.66e-3 of its size, is off by 1.73e-3 to 1.78e-3 with that (333
// tokens of 12 experts of H 1248, I 3296; 1024 of 64 of H 2048, I 1408). The tiled kernels of
// bf16 results take it because exact products cost them 13 to 50 % (us, scaled / exact, 64-row
// tiles: 8 experts of H 4096, I 14336 at 49 rows 169 / 200; 64 of H 2048, I 1408 at 94 rows
// 116 / 171; 32 of H 1280, I 3328 at 150 rows 116 / 172).
template <int g>
__device__ __forceinline__ f32x4 mma_scaled(u32x4 w, uint32_t ws, const u32x4* x, uint32_t xs, f32x4 c) {
  const i32x8 a = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]),
                   static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 b = {static_cast<int>(x[0][0]), static_cast<int>(x[0][1]), static_cast<int>(x[0][2]),
                   static_cast<int>(x[0][3]), static_cast<int>(x[1][0]), static_cast<int>(x[1][1]),
                   static_cast<int>(x[1][2]), static_cast<int>(x[1][3])};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, /*A e2m1*/ 4, /*B e4m3*/ 0, g,
                                                          static_cast<int>(ws), 0,
                                                          static_cast<int>(xs));
}

// The same product in bf16, which holds every code times its scale exactly (4
// significant bits at most), summed in fp32: for results of more bits than bf16, and
// where the weights' stream hides it. That holds for scale bytes 3 to 246 of tokens and up
// to 252 of weights: over them the largest codes are past bf16's range (of tokens in
// 16 or 32 bits none is), under 3 the smallest are rounded to multiples of 2^-133.
// Lane (r, q) multiplies columns 32 q + 8 j .. + 7 in the j-th of four MFMAs (the
// order of columns is free as long as both operands share it).
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bf16x8 join(bf16x2 a, bf16x2 b, bf16x2 c, bf16x2 d) {
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ bf16x8 weights_bf16(uint32_t w, float s) {
  return join(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
}

__device__ __forceinline__ bf16x8 tokens_bf16(uint32_t lo, uint32_t hi, float s) {
  return join(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false),
              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
}

// The gated activation of one supergroup for one token, to be stored in 8 bits: lane q
// holds features 8 q .. 8 q + 7 of the block (v: gate, up of the lower four, then of
// the upper four). Returns the bits of their largest magnitude.
template <int kAct, bool kExact>
__device__ __forceinline__ uint32_t gated_block(const f32x4* v, float* h) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float g = v[i / 4 * 2][i % 4], u = v[i / 4 * 2 + 1][i % 4];
    h[i] = (kExact ? gate_act(kAct, g) : gate_act_fast(kAct, g)) * u;
    amax = fmaxf(amax, fabsf(h[i]));  // ignores NaN
  }
  return __float_as_uint(amax);
}

// The same without infinities, which have no part in a block's scale. This and what
// follows runs while the matrix cores wait, so instructions count: infinities cost a
// branch that is seldom taken instead of a test per value.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t finite_max(const float* h) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, mx_finite_abs(h[i]));
  return __float_as_uint(amax);
}

// The largest of the token's four lanes (rows of 16 are exchanged without the LDS).
__device__ __forceinline__ uint32_t block_max(uint32_t amax) {
  const auto a = __builtin_amdgcn_permlane16_swap(amax, amax, false, false);
  amax = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
  return max(b[0], b[1]);
}

// f(activation as a compile-time constant).
template <typename F>
__device__ __forceinline__ void by_activation(int act, F f) {
  if (act == MOE355_ACT_SILU)
    f(std::integral_constant<int, MOE355_ACT_SILU>());
  else if (act == MOE355_ACT_GELU)
    f(std::integral_constant<int, MOE355_ACT_GELU>());
  else
    f(std::integral_constant<int, MOE355_ACT_GELU_TANH>());
}
