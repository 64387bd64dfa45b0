// Conversions into the formats of mx.h: token rows to 8 bits (alone, or in the first
// launch of an expert call beside the grouping of its slots), and expert weights
// (codes of a checkpoint, or 16/32-bit weights) to the 4-bit tile order.
#include <climits>

#include "mx.h"

namespace moe355 {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = kMxStreamTile;
#include "group_slots.h"
#include "permute_body.h"

// Thread i of a launch quantises 8 consecutive values (4 threads per block of 32); bound
// by reading T * H elements and writing half (16 bits) or a quarter of their bytes: some
// 10 us for 4096 x 4096 bf16 (50 MB).
template <typename T>
__device__ __forceinline__ void quantize8(const MxQuantArgs& a, size_t i) {
  const int per_row = a.Hp / 8;
  if (i >= static_cast<size_t>(a.T) * per_row) return;  // whole blocks: per_row % 16 == 0
  const int t = static_cast<int>(i / per_row), c = static_cast<int>(i % per_row) * 8;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (c < a.H) {
    const T* p = static_cast<const T*>(a.x) + static_cast<size_t>(t) * a.H + c;
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int j = 0; j < 8; j += N) Vec16<T>::unpack(*reinterpret_cast<const u32x4*>(p + j), v + j);
  }
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, mx_finite_abs(v[j]));
  amax = fmaxf(amax, __shfl_xor(amax, 1, kWave));
  amax = fmaxf(amax, __shfl_xor(amax, 2, kWave));
  const int b = mx8_scale(amax);
  *reinterpret_cast<u32x2*>(a.codes + static_cast<size_t>(t) * a.Hp + c) = mx8_codes(v, b);
  if ((threadIdx.x & 3) == 0)
    a.scales[static_cast<size_t>(t) * (a.Hp / kMxBlock) + c / kMxBlock] = static_cast<uint8_t>(b);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const MxQuantArgs a) {
  quantize8<T>(a, static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x);
}

// The first launch of an expert call. Its first workgroups group the slots: one wave
// up to 64 slots on 16-row tiles, one workgroup of a thread per slot up to
// kPermuteSingleMax, above it the permute's counts; the others quantise x. Two
// launches in a row took some 4 us longer. Latency bound but for prompts: 3 us for one
// token, 5 for 999 slots, 8 and 13 for 4096 tokens of H 2048 and 4096.
enum class Group { kWave, kOne, kCount };

template <typename T, Group kGroup>
__global__ __launch_bounds__(kGroup == Group::kOne ? kOneThreads : kThreads) void mx_prepare_kernel(
    const PermuteArgs p, const MxQuantArgs x) {
  const int n_group = kGroup == Group::kCount ? p.n_blocks : 1, b = blockIdx.x;
  if (b >= n_group) {
    quantize8<T>(x, static_cast<size_t>(b - n_group) * blockDim.x + threadIdx.x);
  } else if constexpr (kGroup == Group::kCount) {
    permute_count(p, b);
  } else if constexpr (kGroup == Group::kOne) {
    permute_one(p);
  } else if (threadIdx.x < kWave) {
    __shared__ int meta[4], rowsrc[kWave], estart[kGroupExpertsPerLane * kWave];
    __shared__ unsigned long long emask[kGroupExpertsPerLane * kWave];
    group_slots(p, 0, true, meta, rowsrc, emask, estart);
  }
}

// e2m1 code of v (|v| <= 6): the values 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even
// code.
__device__ __forceinline__ uint32_t mx4_code(float v) {
  const float m = fabsf(v);
  const uint32_t c = (m > 0.25f) + (m >= 0.75f) + (m > 1.25f) + (m >= 1.75f) + (m > 2.5f) +
                     (m >= 3.5f) + (m > 5.0f);
  return c | (v < 0.f ? 8u : 0u);
}

// One thread per lane of a tile (16 output bytes, one block of one row). T void:
// the source holds codes; else weights, each block scaled by the smallest power of
// two that keeps it within 6 (a block with an infinity or NaN gets the NaN scale).
// Runs once per weight matrix.
template <typename T>
__global__ __launch_bounds__(kThreads) void mx_pack_kernel(const MxPackArgs a) {
  constexpr bool kCodes = std::is_same<T, void>::value;
  const int steps = a.cols_p / kMxStep;
  const int groups = a.rows_p / 16;
  const size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= static_cast<size_t>(groups) * steps * kWave) return;
  const int lane = static_cast<int>(i % kWave);
  const size_t tile = i / kWave;
  const int step = static_cast<int>(tile / 4 % steps);
  const int group = static_cast<int>(tile / 4 / steps) * 4 + static_cast<int>(tile % 4);
  const int r = lane & 15, col = step * kMxStep + kMxBlock * (lane >> 4);
  int row;
  bool in;
  if (a.gate_up) {
    const int half = a.rows / 2;
    const int f = (group >> 2) * kMxBlock + 8 * (r >> 2) + 4 * ((group >> 1) & 1) + (r & 3);
    in = f < half;
    row = (group & 1) * half + f;
  } else {
    row = group * 16 + r;
    in = row < a.rows;
  }
  in = in && col < a.cols;
  uint32_t out[4] = {0u, 0u, 0u, 0u};
  int b = 0;
  if (in) {
    if constexpr (kCodes) {
      const uint8_t* p = static_cast<const uint8_t*>(a.src) + (static_cast<size_t>(row) * a.cols + col) / 2;
      const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = v[j];
      b = a.scales[static_cast<size_t>(row) * (a.cols / kMxBlock) + col / kMxBlock];
    } else {
      const T* p = static_cast<const T*>(a.src) + static_cast<size_t>(row) * a.cols + col;
      float amax = 0.f;
      bool bad = false;
      for (int j = 0; j < kMxBlock; ++j) {
        const float v = fabsf(to_f32(p[j]));
        bad |= !(v < INFINITY);
        amax = fmaxf(amax, v);
      }
      if (bad) {
        b = 255;
      } else {
        const uint32_t bits = __float_as_uint(amax);  // 6 = 1.5 * 2^2
        b = max(static_cast<int>(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0), 0);
        const float f = mx_inverse(b);
        for (int j = 0; j < kMxBlock; ++j) out[j / 8] |= mx4_code(to_f32(p[j]) * f) << (4 * (j % 8));
      }
    }
  }
  *reinterpret_cast<u32x4*>(a.codes_out + i * 16) = u32x4{out[0], out[1], out[2], out[3]};
  a.scales_out[((static_cast<size_t>(group >> 2) * steps + step) * kWave + lane) * 4 + (group & 3)] =
      static_cast<uint8_t>(b);
}

template <typename T>
hipError_t launch_pack_t(const MxPackArgs& a, hipStream_t s) {
  const size_t n = static_cast<size_t>(a.rows_p / 16) * (a.cols_p / kMxStep) * kWave;
  mx_pack_kernel<T><<<dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_quantize_t(const MxQuantArgs& a, hipStream_t s) {
  const size_t n = static_cast<size_t>(a.T) * (a.Hp / 8);
  mx_quantize_kernel<T><<<dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_prepare_t(const PermuteArgs& p, const MxQuantArgs& x, hipStream_t s) {
  const size_t n = x.x ? static_cast<size_t>(x.T) * (x.Hp / 8) : 0;
  const auto blocks = [n](int threads) { return static_cast<unsigned>((n + threads - 1) / threads); };
  if (p.R <= kWave && p.tile_rows == kRows)
    mx_prepare_kernel<T, Group::kWave><<<dim3(1 + blocks(kThreads)), dim3(kThreads), 0, s>>>(p, x);
  else if (p.n_blocks == 1)
    mx_prepare_kernel<T, Group::kOne><<<dim3(1 + blocks(kOneThreads)), dim3(kOneThreads), 0, s>>>(p, x);
  else
    mx_prepare_kernel<T, Group::kCount><<<dim3(p.n_blocks + blocks(kThreads)), dim3(kThreads), 0, s>>>(p, x);
  hipError_t err = hipGetLastError();
  return err != hipSuccess || p.n_blocks == 1 ? err : launch_permute_scatter(p, s);
}

}  // namespace

hipError_t launch_mx_prepare(const PermuteArgs& p, const MxQuantArgs& x, int dtype, hipStream_t s) {
  if (dtype == MOE355_BF16) return launch_prepare_t<bf16>(p, x, s);
  if (dtype == MOE355_F16) return launch_prepare_t<f16>(p, x, s);
  return launch_prepare_t<float>(p, x, s);
}

hipError_t launch_mx_quantize(const MxQuantArgs& a, int dtype, hipStream_t s) {
  if (a.T == 0) return hipSuccess;
  if (dtype == MOE355_BF16) return launch_quantize_t<bf16>(a, s);
  if (dtype == MOE355_F16) return launch_quantize_t<f16>(a, s);
  return launch_quantize_t<float>(a, s);
}

hipError_t launch_mx_pack(const MxPackArgs& a, int dtype, hipStream_t s) {
  if (dtype < 0) return launch_pack_t<void>(a, s);
  if (dtype == MOE355_BF16) return launch_pack_t<bf16>(a, s);
  if (dtype == MOE355_F16) return launch_pack_t<f16>(a, s);
  return launch_pack_t<float>(a, s);
}

}  // namespace moe355
