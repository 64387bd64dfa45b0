// Values to 8 bits with a scale per block of 128 (formats: fp8.h).
#include <climits>

#include "fp8.h"

namespace moe355 {
namespace {

#include "chunk.h"

constexpr int kThreads = 256;
constexpr int kRows = kF8StreamTile;
#include "group_slots.h"
#include "permute_body.h"

constexpr int kWaves = kThreads / kWave;
constexpr int kPer = 8;                    // values of a lane
constexpr int kLanes = kF8Block / kPer;    // lanes of a block

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

// The largest of 16 neighbouring lanes (a row of the wave's lanes, exchanged without the LDS).
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const int u = o == 8   ? __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false)
                  : o == 4 ? __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false)
                  : o == 2 ? __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, false)
                           : __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, false);
    v = fmaxf(v, __int_as_float(u));
  }
  return v;
}

// The largest finite magnitude of a lane's values; infinities cost a branch that is seldom
// taken.
__device__ __forceinline__ float finite_max(const float* v) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) amax = fmaxf(amax, fabsf(v[i]));  // ignores NaN
  if (amax == INFINITY) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) amax = fmaxf(amax, f8_finite_abs(v[i]));
  }
  return amax;
}

// Workgroup g of a launch of `threads` quantises that many times 8 values, 16 lanes to a block.
// Bound by memory: a row is read once, its codes and scales written once.
template <typename T>
__device__ __forceinline__ void quantize_group(const F8QuantArgs& a, size_t g, int threads) {
  const int blocks = f8_blocks(a.K), per = threads / kLanes;
  const size_t first = g * per, row0 = first / blocks;  // the same for the workgroup
  const int at = static_cast<int>(first - row0 * blocks) + threadIdx.x / kLanes;
  const size_t row = row0 + at / blocks;
  if (row >= static_cast<size_t>(a.M)) return;
  const int b = at % blocks, lane = threadIdx.x % kLanes, e = b * kF8Block + lane * kPer;
  float v[kPer];
  load_values<T>(static_cast<const T*>(a.x) + row * a.K + e, a.K - e, v);
  const F8Div d = f8_div(lanes_max(finite_max(v)));
  *reinterpret_cast<u32x2*>(a.codes + row * blocks * kF8Block + e) = u32x2{f8_codes4(v, d), f8_codes4(v + 4, d)};
  if (lane == 0) a.scales[row * blocks + b] = d.scale;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const F8QuantArgs a) {
  quantize_group<T>(a, blockIdx.x, kThreads);
}

// The first launch of an expert call. Its first workgroups group the slots: one wave up to 64
// slots, one workgroup of a thread per slot up to kPermuteSingleMax, above it the permute's
// counts; the others quantise x. In two launches a call of 16 tokens takes 5 us longer.
enum class Group { kWave, kOne, kCount };

template <typename T, Group kGroup>
__global__ __launch_bounds__(kGroup == Group::kOne ? kOneThreads : kThreads) void prepare_kernel(
    const PermuteArgs p, const F8QuantArgs x) {
  const int n_group = kGroup == Group::kCount ? p.n_blocks : 1, b = blockIdx.x;
  if (b >= n_group) {
    quantize_group<T>(x, b - n_group, kGroup == Group::kOne ? kOneThreads : kThreads);
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
    amax = fmaxf(amax, finite_max(v[i]));
  }
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, kWave));
  if (tid % kWave == 0) most[tid / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) amax = fmaxf(amax, most[w]);
  const F8Div d = f8_div(amax);
  uint8_t* cell = a.codes + (static_cast<size_t>(blockIdx.y) * blocks + blockIdx.x) * kF8Cell;
  const int col = tid % kLanes * kPer;
#pragma unroll
  for (int i = 0; i < kRounds; ++i)
    *reinterpret_cast<u32x2*>(cell + f8_place(i * kRowsAtOnce + tid / kLanes, col & ~15, 1) + (col & 8)) =
        u32x2{f8_codes4(v[i], d), f8_codes4(v[i] + 4, d)};
  if (tid == 0) a.scales[static_cast<size_t>(blockIdx.y) * blocks + blockIdx.x] = d.scale;
}

// A checkpoint's codes as cells: a thread per 16 codes of the result. Runs once per matrix.
__global__ __launch_bounds__(kThreads) void pack_kernel(const F8PackArgs a) {
  const int blocks = f8_blocks(a.K), rows = f8_pad(a.N), per_row = blocks * (kF8Block / 16);
  const size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= static_cast<size_t>(rows) * per_row) return;
  const int n = static_cast<int>(i / per_row), k = static_cast<int>(i % per_row) * 16;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (n < a.N && k < a.K) {
    const uint8_t* p = a.src + static_cast<size_t>(n) * a.K + k;
    typedef u32x4 u32x4_byte __attribute__((aligned(1)));
    if (k + 16 <= a.K) {
      v = *reinterpret_cast<const u32x4_byte*>(p);
    } else {
      for (int j = 0; j < a.K - k; ++j) v[j / 4] |= static_cast<uint32_t>(p[j]) << (8 * (j % 4));
    }
  }
  *reinterpret_cast<u32x4*>(a.cells + f8_place(n, k, blocks)) = v;
}

// Workgroups of `threads` that quantise a.
size_t groups_of(const F8QuantArgs& a, int threads) {
  const size_t per = threads / kLanes;
  return a.x ? (static_cast<size_t>(a.M) * f8_blocks(a.K) + per - 1) / per : 0;
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
  const size_t groups = groups_of(a, kThreads);
  if (groups > INT_MAX) return hipErrorInvalidValue;
  return by_type(dtype, [&](auto t) {
    quantize_kernel<decltype(t)><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, s>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_f8_prepare(const PermuteArgs& p, const F8QuantArgs& x, int dtype, hipStream_t s) {
  if (groups_of(x, kThreads) + p.n_blocks > INT_MAX) return hipErrorInvalidValue;
  const hipError_t err = by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    auto grid = [&](int first, int threads) { return dim3(static_cast<unsigned>(first + groups_of(x, threads))); };
    if (p.R <= kWave)
      prepare_kernel<T, Group::kWave><<<grid(1, kThreads), dim3(kThreads), 0, s>>>(p, x);
    else if (p.n_blocks == 1)
      prepare_kernel<T, Group::kOne><<<grid(1, kOneThreads), dim3(kOneThreads), 0, s>>>(p, x);
    else
      prepare_kernel<T, Group::kCount><<<grid(p.n_blocks, kThreads), dim3(kThreads), 0, s>>>(p, x);
    return hipGetLastError();
  });
  return err != hipSuccess || p.n_blocks == 1 ? err : launch_permute_scatter(p, s);
}

hipError_t launch_f8_quantize_weight(const F8QuantArgs& a, int dtype, hipStream_t s) {
  const dim3 grid(f8_blocks(a.K), f8_blocks(a.M));
  return by_type(dtype, [&](auto t) {
    quantize_weight_kernel<decltype(t)><<<grid, dim3(kThreads), 0, s>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_f8_pack(const F8PackArgs& a, hipStream_t s) {
  const size_t threads = static_cast<size_t>(f8_pad(a.N)) * f8_blocks(a.K) * (kF8Block / 16);
  const size_t groups = (threads + kThreads - 1) / kThreads;
  if (groups > INT_MAX) return hipErrorInvalidValue;
  pack_kernel<<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace moe355
