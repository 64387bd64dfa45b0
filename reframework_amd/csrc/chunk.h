// Rows of any length and alignment in 16-byte chunks: what the row kernels that take any
// size (layer_norm.hip, tokens.hip) share. Included inside their anonymous namespaces.
#pragma once

// N consecutive elements (16 bytes) from p on, of which the first n (1..N) exist: as stored.
// gfx950 loads 16 bytes at any element address in one instruction.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p, int n) {
  constexpr int N = Vec16<T>::N;
  if (n >= N) return load16_any(p);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= n) continue;
    if constexpr (sizeof(T) == 4)
      v[i] = __builtin_bit_cast(uint32_t, p[i]);
    else
      v[i / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, p[i])) << (16 * (i & 1));
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, u32x4 v, int n) {
  constexpr int N = Vec16<T>::N;
  if (n >= N) {
    *reinterpret_cast<u32x4_any*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= n) continue;
    if constexpr (sizeof(T) == 4)
      p[i] = __builtin_bit_cast(T, static_cast<uint32_t>(v[i]));
    else
      p[i] = __builtin_bit_cast(T, static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1))));
  }
}

// N fp32 values rounded to T, as stored.
template <typename T>
__device__ __forceinline__ u32x4 pack_chunk(const float* v) {
  if constexpr (sizeof(T) == 4) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                 __float_as_uint(v[3])};
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(v[i]);
    return __builtin_bit_cast(u32x4, h);
  }
}

// N consecutive parameters of type W from e on (n of them exist), in fp32.
template <typename W, int N>
__device__ __forceinline__ void load_params(const W* p, int n, float* o) {
  constexpr int kPer = Vec16<W>::N;
  if constexpr (N < kPer) {  // 4 of 8
    float t[kPer];
    if (n >= N) {
      typedef u32x2 u32x2_any __attribute__((aligned(2)));
      const u32x2 v = *reinterpret_cast<const u32x2_any*>(p);
      Vec16<W>::unpack(u32x4{v[0], v[1], 0u, 0u}, t);
    } else {
      Vec16<W>::unpack(load_chunk<W>(p, n), t);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
      if (i < n) {
        Vec16<W>::unpack(load_chunk<W>(p + i, n - i), o + i);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) o[i + j] = 0.f;
      }
    }
  }
}
