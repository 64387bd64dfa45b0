// Values to 8 bits with a scale per block of 128 (formats: fp8.h).
#include "fp8.h"

namespace moe355 {
namespace {

#include "chunk.h"

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kPer = 8;                    // values of a lane
constexpr int kLanes = kF8Block / kPer;    // lanes of a block
constexpr int kWaveBlocks = kWave / kLanes;

// kPer values from p on, of which n (may be under 1) exist; zeros for the others.
template <typename T>
__device__ __forceinline__ void load_values(const T* p, int n, float* v) {
  constexpr int N = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < kPer; i += N) {
    if (i < n) {
      Vec16<T>::unpack(load_chunk<T>(p + i, n - i), v + i);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = 0.f;
    }
  }
}

__device__ __forceinline__ float block_max16(float v) {
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}

// A wave takes 4 blocks of a row at a time, 16 lanes each. Bound by memory: a row is read once,
// its codes and scales written once.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const F8QuantArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const size_t row = static_cast<size_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
  if (row >= static_cast<size_t>(a.M)) return;
  const int blocks = f8_blocks(a.K);
  const T* x = static_cast<const T*>(a.x) + row * a.K;
  uint8_t* codes = a.codes + row * blocks * kF8Block;
  for (int b = blockIdx.y * kWaveBlocks + lane / kLanes; b < blocks; b += gridDim.y * kWaveBlocks) {
    const int e = b * kF8Block + (lane % kLanes) * kPer;
    float v[kPer], amax = 0.f;
    load_values<T>(x + e, a.K - e, v);
#pragma unroll
    for (int i = 0; i < kPer; ++i) amax = fmaxf(amax, f8_finite_abs(v[i]));
    const F8Div d = f8_div(block_max16(amax));
    *reinterpret_cast<u32x2*>(codes + e) = u32x2{f8_codes4(v, d), f8_codes4(v + 4, d)};
    if (lane % kLanes == 0) a.scales[row * blocks + b] = d.scale;
  }
}

// A workgroup takes one 128 x 128 block: 16 lanes a row, 16 rows at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_weight_kernel(const F8QuantArgs a) {
  constexpr int kRowsAtOnce = kThreads / kLanes, kRounds = kF8Block / kRowsAtOnce;
  __shared__ float most[kWaves];
  const int tid = threadIdx.x, blocks = f8_blocks(a.K);
  const int e = blockIdx.x * kF8Block + (tid % kLanes) * kPer;
  float v[kRounds][kPer], amax = 0.f;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int row = blockIdx.y * kF8Block + i * kRowsAtOnce + tid / kLanes;
    load_values<T>(static_cast<const T*>(a.x) + static_cast<size_t>(row) * a.K + e,
                   row < a.M ? a.K - e : 0, v[i]);
#pragma unroll
    for (int j = 0; j < kPer; ++j) amax = fmaxf(amax, f8_finite_abs(v[i][j]));
  }
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, kWave));
  if (tid % kWave == 0) most[tid / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) amax = fmaxf(amax, most[w]);
  const F8Div d = f8_div(amax);
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int row = blockIdx.y * kF8Block + i * kRowsAtOnce + tid / kLanes;
    if (row < a.M)
      *reinterpret_cast<u32x2*>(a.codes + static_cast<size_t>(row) * blocks * kF8Block + e) =
          u32x2{f8_codes4(v[i], d), f8_codes4(v[i] + 4, d)};
  }
  if (tid == 0) a.scales[static_cast<size_t>(blockIdx.y) * blocks + blockIdx.x] = d.scale;
}

template <typename F>
hipError_t by_type(int dtype, F f) {
  if (dtype == MOE355_F32) return f(float());
  if (dtype == MOE355_BF16) return f(bf16());
  return f(f16());
}

}  // namespace

hipError_t launch_f8_quantize(const F8QuantArgs& a, int dtype, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  // a wave walks along its row, unless the rows are too few to fill the card
  const int parts = (f8_blocks(a.K) + kWaveBlocks - 1) / kWaveBlocks;
  const int rows = (a.M + kWaves - 1) / kWaves;
  const int want = (8 * device_cu_count() + rows - 1) / rows;
  const dim3 grid(rows, parts < want ? parts : want);
  return by_type(dtype, [&](auto t) {
    quantize_kernel<decltype(t)><<<grid, dim3(kThreads), 0, s>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_f8_quantize_weight(const F8QuantArgs& a, int dtype, hipStream_t s) {
  const dim3 grid(f8_blocks(a.K), f8_blocks(a.M));
  return by_type(dtype, [&](auto t) {
    quantize_weight_kernel<decltype(t)><<<grid, dim3(kThreads), 0, s>>>(a);
    return hipGetLastError();
  });
}

}  // namespace moe355
