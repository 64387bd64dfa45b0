// Tokens in the order of their experts and back, with the routing weights, and the gradients.
//
//   permute   rows[row(t, k)] = x[t]                      backward: combine without weights
//   combine   out[t] = sum_k w[t, k] * rows[row(t, k)]    (k ascending, in fp32)
//   combine backward: drows[row(t, k)] = w[t, k] * dout[t],
//                     dw[t, k] = sum_h dout[t, h] * rows[row(t, k), h]
// Slots of no expert (row -1) take no part, their dw is 0; rows behind the last one that has
// a slot are zeros. Sums run in a fixed order, without atomics.
//
// Bound by memory. Every kernel goes by tokens, a wave a token: the token's row is read (or
// written) once and its K rows scattered (or gathered), so each byte moves once; by rows, the
// permute would read a token K times. The rows' numbers are the same for a wave, which reads them
// on the scalar unit.
#include "common.h"
#include "rows.h"

namespace moe355 {
namespace {

#include "chunk.h"

constexpr int kThreads = 256;
constexpr int kTokens = kThreads / kWave;  // of a workgroup

__device__ __forceinline__ int wave_of_block() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
}

// Rows outside the R there are count as none.
__device__ __forceinline__ bool has_row(int row, int R) {
  return static_cast<unsigned>(row) < static_cast<unsigned>(R);
}

// Zeros in the rows from n on, this workgroup's share of them and of their chunks.
template <typename T>
__device__ __forceinline__ void zero_tail(T* rows, int n, int R, int H, int lane, int wave) {
  constexpr int N = Vec16<T>::N;
  const int parts = gridDim.x * kTokens;
  for (int r = max(n, 0) + blockIdx.x * kTokens + wave; r < R; r += parts)
    for (int e = (blockIdx.y * kWave + lane) * N; e < H; e += gridDim.y * kWave * N)
      store_chunk<T>(rows + static_cast<size_t>(r) * H + e, u32x4{0u, 0u, 0u, 0u}, H - e);
}

template <typename T, int kCpt>
__global__ __launch_bounds__(kThreads) void permute_rows_kernel(const TokenRowsArgs a) {
  constexpr int N = Vec16<T>::N;
  const int lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const int t = blockIdx.x * kTokens + wave;
  T* dst = static_cast<T*>(a.dst);
  if (t < a.T) {
    const T* x = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.H;
    u32x4 v[kCpt];
#pragma unroll
    for (int c = 0; c < kCpt; ++c) {
      const int e = ((blockIdx.y * kCpt + c) * kWave + lane) * N;
      if (e < a.H) v[c] = load_chunk<T>(x + e, a.H - e);
    }
    const int32_t* rows = a.slot_to_row + static_cast<size_t>(t) * a.K;
    for (int k = 0; k < a.K; ++k) {
      const int row = rows[k];
      if (!has_row(row, a.R)) continue;
#pragma unroll
      for (int c = 0; c < kCpt; ++c) {
        const int e = ((blockIdx.y * kCpt + c) * kWave + lane) * N;
        if (e < a.H) store_chunk<T>(dst + static_cast<size_t>(row) * a.H + e, v[c], a.H - e);
      }
    }
  }
  zero_tail<T>(dst, *a.n_rows, a.R, a.H, lane, wave);
}

template <typename T, int kCpt, bool kWeights>
__global__ __launch_bounds__(kThreads) void combine_rows_kernel(const TokenRowsArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int kBatch = 4;  // slots whose rows are loaded before the first is used
  const int lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const int t = blockIdx.x * kTokens + wave;
  if (t >= a.T) return;
  const T* src = static_cast<const T*>(a.src);
  const int32_t* rows = a.slot_to_row + static_cast<size_t>(t) * a.K;
  const float* weights = a.topk_w + static_cast<size_t>(t) * a.K;
  float acc[kCpt][N];
#pragma unroll
  for (int c = 0; c < kCpt; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) acc[c][i] = 0.f;
  for (int k0 = 0; k0 < a.K; k0 += kBatch) {
    u32x4 v[kBatch][kCpt];
    int row[kBatch];
    float w[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      row[j] = k0 + j < a.K ? rows[k0 + j] : -1;
      if (!has_row(row[j], a.R)) row[j] = -1;
      w[j] = kWeights && k0 + j < a.K ? weights[k0 + j] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      // a slot without a row loads row 0, whose values are not used
      const T* p = src + static_cast<size_t>(row[j] < 0 ? 0 : row[j]) * a.H;
#pragma unroll
      for (int c = 0; c < kCpt; ++c) {
        const int e = ((blockIdx.y * kCpt + c) * kWave + lane) * N;
        if (e < a.H) v[j][c] = load_chunk<T>(p + e, a.H - e);
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (row[j] < 0) continue;
#pragma unroll
      for (int c = 0; c < kCpt; ++c) {
        float f[N];
        Vec16<T>::unpack(v[j][c], f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[c][i] += kWeights ? w[j] * f[i] : f[i];
      }
    }
  }
  T* out = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.H;
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = ((blockIdx.y * kCpt + c) * kWave + lane) * N;
    if (e < a.H) store_chunk<T>(out + e, pack_chunk<T>(acc[c]), a.H - e);
  }
}

// kOnce: dout's row fits the wave's registers; else it is read again for every slot, from the
// caches.
template <typename T, int kCpt, bool kOnce>
__global__ __launch_bounds__(kThreads) void combine_rows_bwd_kernel(const CombineBwdArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int kBlock = kCpt * kWave * N;  // elements of a pass
  const int lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const int t = blockIdx.x * kTokens + wave;
  T* drows = static_cast<T*>(a.drows);
  if (t < a.T) {
    const T* dout = static_cast<const T*>(a.dout) + static_cast<size_t>(t) * a.H;
    u32x4 g[kCpt];
    auto load = [&](u32x4* v, const T* p, int e0) {
#pragma unroll
      for (int c = 0; c < kCpt; ++c) {
        const int e = e0 + (c * kWave + lane) * N;
        if (e < a.H) v[c] = load_chunk<T>(p + e, a.H - e);
      }
    };
    if constexpr (kOnce) load(g, dout, 0);
    for (int k = 0; k < a.K; ++k) {
      const size_t slot = static_cast<size_t>(t) * a.K + k;
      const int row = a.slot_to_row[slot];
      if (!has_row(row, a.R)) {
        if (a.dw && lane == 0) a.dw[slot] = 0.f;
        continue;
      }
      const float w = a.topk_w[slot];
      float dot = 0.f;
      for (int e0 = 0; e0 < a.H; e0 += kBlock) {
        const size_t at = static_cast<size_t>(row) * a.H;
        u32x4 y[kCpt];
        if (a.dw) load(y, static_cast<const T*>(a.rows) + at, e0);
        if constexpr (!kOnce) load(g, dout, e0);
#pragma unroll
        for (int c = 0; c < kCpt; ++c) {
          const int e = e0 + (c * kWave + lane) * N;
          if (e >= a.H) continue;
          float gv[N], o[N];
          Vec16<T>::unpack(g[c], gv);
          if (a.dw) {
            float yv[N];
            Vec16<T>::unpack(y[c], yv);
#pragma unroll
            for (int i = 0; i < N; ++i) dot += gv[i] * yv[i];  // zeros past the row's end
          }
          if (drows) {
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = w * gv[i];
            store_chunk<T>(drows + at + e, pack_chunk<T>(o), a.H - e);
          }
        }
        if constexpr (kOnce) break;
      }
      if (a.dw) {
        dot = wave_sum(dot);
        if (lane == 0) a.dw[slot] = dot;
      }
    }
  }
  if (drows) zero_tail<T>(drows, *a.n_rows, a.R, a.H, lane, wave);
}

// Chunks of a lane: as many as a row has, up to `most`, where the tokens alone keep the CUs
// busy; one, and more workgroups a row, where they do not.
template <typename T>
int columns(int T_, int H, int most) {
  constexpr int N = Vec16<T>::N;
  const int groups = (H + N * kWave - 1) / (N * kWave);
  int c = 1;
  while (c < most && c < groups &&
         static_cast<long long>(T_) * ((groups + 2 * c - 1) / (2 * c)) >= 8ll * device_cu_count())
    c *= 2;
  return c;
}

template <typename T, int kCpt>
dim3 token_grid(int tokens, int H) {
  constexpr int per = Vec16<T>::N * kWave * kCpt;
  return dim3((tokens + kTokens - 1) / kTokens, (H + per - 1) / per);
}

template <typename T>
hipError_t permute_t(const TokenRowsArgs& a, hipStream_t s) {
  switch (columns<T>(a.T, a.H, 4)) {
    case 1: permute_rows_kernel<T, 1><<<token_grid<T, 1>(a.T, a.H), kThreads, 0, s>>>(a); break;
    case 2: permute_rows_kernel<T, 2><<<token_grid<T, 2>(a.T, a.H), kThreads, 0, s>>>(a); break;
    default: permute_rows_kernel<T, 4><<<token_grid<T, 4>(a.T, a.H), kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <typename T, bool kWeights>
hipError_t combine_t(const TokenRowsArgs& a, hipStream_t s) {
  switch (columns<T>(a.T, a.H, 4)) {
    case 1: combine_rows_kernel<T, 1, kWeights><<<token_grid<T, 1>(a.T, a.H), kThreads, 0, s>>>(a); break;
    case 2: combine_rows_kernel<T, 2, kWeights><<<token_grid<T, 2>(a.T, a.H), kThreads, 0, s>>>(a); break;
    default: combine_rows_kernel<T, 4, kWeights><<<token_grid<T, 4>(a.T, a.H), kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t combine_bwd_t(const CombineBwdArgs& a, hipStream_t s) {
  constexpr int N = Vec16<T>::N;
  const dim3 grid((a.T + kTokens - 1) / kTokens);
  const int groups = (a.H + N * kWave - 1) / (N * kWave);
  if (groups <= 2)
    combine_rows_bwd_kernel<T, 2, true><<<grid, kThreads, 0, s>>>(a);
  else if (groups <= 4)
    combine_rows_bwd_kernel<T, 4, true><<<grid, kThreads, 0, s>>>(a);
  else if (groups <= 8)
    combine_rows_bwd_kernel<T, 8, true><<<grid, kThreads, 0, s>>>(a);
  else
    combine_rows_bwd_kernel<T, 4, false><<<grid, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <typename F>
hipError_t by_type(int dtype, F f) {
  if (dtype == MOE355_F32) return f(float());
  if (dtype == MOE355_BF16) return f(bf16());
  return f(f16());
}

}  // namespace

hipError_t launch_permute_rows(const TokenRowsArgs& a, int dtype, hipStream_t s) {
  return by_type(dtype, [&](auto t) { return permute_t<decltype(t)>(a, s); });
}

hipError_t launch_combine_rows(const TokenRowsArgs& a, int dtype, hipStream_t s) {
  return by_type(dtype, [&](auto t) {
    return a.topk_w ? combine_t<decltype(t), true>(a, s) : combine_t<decltype(t), false>(a, s);
  });
}

hipError_t launch_combine_rows_bwd(const CombineBwdArgs& a, int dtype, hipStream_t s) {
  return by_type(dtype, [&](auto t) { return combine_bwd_t<decltype(t)>(a, s); });
}

}  // namespace moe355
