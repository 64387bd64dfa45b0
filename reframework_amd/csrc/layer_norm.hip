// Residual add + LayerNorm and its gradient.
//
//   r    = x + residual                (in the storage type; r = x without a residual)
//   xhat = (r - mean(r)) * rstd,  rstd = 1 / sqrt(mean((r - mean(r))^2) + eps)
//   out  = xhat * w + b
// and backwards, with dy the gradient of out and dres that of r as it goes on:
//   g  = dy * w
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dres
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
// All in fp32, rounded once. Bound by memory: the forward pass reads x and the residual
// and writes r and out, the backward pass reads dy, dres and r and writes dx.
//
// A row lies in the registers of kWaves waves (kCpt 16-byte chunks a lane), so it is
// read once. Its variance is summed around the mean of each wave's part, and the waves' parts
// are joined by (n, mean, sum of squares around it): one exchange between the waves
// instead of two, and no difference of large sums.
#include "common.h"
#include "rows.h"

namespace moe355 {
namespace {

#include "chunk.h"

constexpr int kFwdThreads = 256;

template <typename T, typename W, int kWaves, int kCpt>
__global__ __launch_bounds__(kFwdThreads) void layer_norm_kernel(const LayerNormArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int kRows = kFwdThreads / (kWaves * kWave);  // rows of a workgroup
  constexpr int kLanes = kWaves * kWave;
  __shared__ float part[kRows][kWaves][2];
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, wave = lane / kWave;
  const int t = blockIdx.x * kRows + group;
  const bool live = t < a.T;
  const size_t row = static_cast<size_t>(live ? t : a.T - 1) * a.H;
  const T* x = static_cast<const T*>(a.x) + row;
  const T* res = static_cast<const T*>(a.residual) + row;

  u32x4 raw[kCpt], add[kCpt];
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
    if (e >= a.H) continue;
    raw[c] = load_chunk<T>(x + e, a.H - e);
    if (a.residual) add[c] = load_chunk<T>(res + e, a.H - e);
  }
  float wv[kCpt][N], bv[kCpt][N];
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
    if (e >= a.H) continue;
    load_params<W, N>(static_cast<const W*>(a.weight) + e, a.H - e, wv[c]);
    if (a.bias) load_params<W, N>(static_cast<const W*>(a.bias) + e, a.H - e, bv[c]);
  }

  float r[kCpt][N];
  float sum = 0.f;
  int mine = 0;  // elements of this lane
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
    if (e >= a.H) continue;
    Vec16<T>::unpack(raw[c], r[c]);
    if (a.residual) {
      float s[N];
      Vec16<T>::unpack(add[c], s);
#pragma unroll
      for (int i = 0; i < N; ++i) r[c][i] += s[i];
      raw[c] = pack_chunk<T>(r[c]);
      Vec16<T>::unpack(raw[c], r[c]);
      if (live) store_chunk<T>(static_cast<T*>(a.residual_out) + row + e, raw[c], a.H - e);
    }
    const int n = min(N, a.H - e);
    mine += n;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += i < n ? r[c][i] : 0.f;
  }
  // elements of this wave: its lanes hold neighbouring chunks
  const int n_wave = static_cast<int>(wave_sum(static_cast<float>(mine)));
  const float m_wave = n_wave ? wave_sum(sum) / static_cast<float>(n_wave) : 0.f;
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
    if (e >= a.H) continue;
    const int n = min(N, a.H - e);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = r[c][i] - m_wave;
      sq += i < n ? d * d : 0.f;
    }
  }
  sq = wave_sum(sq);
  float mean = m_wave, m2 = sq;
  if constexpr (kWaves > 1) {
    __shared__ int count[kRows][kWaves];
    if (lane % kWave == 0) {
      part[group][wave][0] = m_wave;
      part[group][wave][1] = sq;
      count[group][wave] = n_wave;
    }
    __syncthreads();
    mean = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mean += part[group][w][0] * static_cast<float>(count[group][w]);
    mean /= static_cast<float>(a.H);
    m2 = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float d = part[group][w][0] - mean;
      m2 += part[group][w][1] + static_cast<float>(count[group][w]) * d * d;
    }
  }
  const float rstd = 1.0f / sqrtf(m2 / static_cast<float>(a.H) + a.eps);
  if (!live) return;
  if (a.mean && lane == 0) {
    a.mean[t] = mean;
    a.rstd[t] = rstd;
  }
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
    if (e >= a.H) continue;
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i] = (r[c][i] - mean) * rstd * wv[c][i];
      if (a.bias) o[i] += bv[c][i];
    }
    store_chunk<T>(static_cast<T*>(a.out) + row + e, pack_chunk<T>(o), a.H - e);
  }
}

// Backward. A workgroup of 8 waves walks over rows, kRows at a time, and keeps its share
// of dw and db in registers; what the row groups of a workgroup hold is added in LDS at the
// end and left as one row of `part`, which a second launch adds up: no atomics, so
// equal calls give equal sums.
constexpr int kBwdThreads = 512;

template <typename T, typename W, int kWaves, int kCpt>
__global__ __launch_bounds__(kBwdThreads) void layer_norm_bwd_kernel(const LayerNormBwdArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int kLanes = kWaves * kWave;
  constexpr int kRows = kBwdThreads / kLanes;
  static_assert(kRows == 1 || kCpt <= 2, "LDS of the sums over row groups");
  __shared__ float exch[2][kRows][kWaves][2];
  __shared__ float sums[kRows > 1 ? kRows * kLanes * kCpt * N : 1];
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, wave = lane / kWave;

  float wv[kCpt][N], dw[kCpt][N], db[kCpt][N];
#pragma unroll
  for (int c = 0; c < kCpt; ++c) {
    const int e = (lane + c * kLanes) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) wv[c][i] = dw[c][i] = db[c][i] = 0.f;
    if (e < a.H) load_params<W, N>(static_cast<const W*>(a.weight) + e, a.H - e, wv[c]);
  }
  u32x4 dy[kCpt], rr[kCpt], dr[kCpt];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int t) {
    if (t >= a.T) return;
    const size_t row = static_cast<size_t>(t) * a.H;
#pragma unroll
    for (int c = 0; c < kCpt; ++c) {
      const int e = (lane + c * kLanes) * N;
      if (e >= a.H) continue;
      dy[c] = load_chunk<T>(static_cast<const T*>(a.dy) + row + e, a.H - e);
      rr[c] = load_chunk<T>(static_cast<const T*>(a.r) + row + e, a.H - e);
      if (a.dres) dr[c] = load_chunk<T>(static_cast<const T*>(a.dres) + row + e, a.H - e);
    }
    mean = a.mean[t];
    rstd = a.rstd[t];
  };
  const int stride = gridDim.x * kRows;
  const int rounds = (a.T + stride - 1) / stride;
  int t = blockIdx.x * kRows + group;
  load(t);
  for (int it = 0; it < rounds; ++it, t += stride) {
    const bool live = t < a.T;
    float g[kCpt][N], xh[kCpt][N], res[kCpt][N];
    float s1 = 0.f, s2 = 0.f;
    const float rs = rstd;
#pragma unroll
    for (int c = 0; c < kCpt; ++c) {
      const int e = (lane + c * kLanes) * N;
      if (!live || e >= a.H) continue;
      Vec16<T>::unpack(dy[c], g[c]);
      Vec16<T>::unpack(rr[c], xh[c]);
      if (a.dres) Vec16<T>::unpack(dr[c], res[c]);
      const int n = min(N, a.H - e);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        xh[c][i] = i < n ? (xh[c][i] - mean) * rstd : 0.f;  // g is 0 there: load_chunk
        dw[c][i] += g[c][i] * xh[c][i];
        db[c][i] += g[c][i];
        g[c][i] *= wv[c][i];
        s1 += g[c][i];
        s2 += g[c][i] * xh[c][i];
      }
    }
    load(t + stride);  // on its way while this row is reduced and stored
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if constexpr (kWaves > 1) {
      // two sets of slots in turn: one barrier a row
      auto& ex = exch[it & 1][group];
      if (lane % kWave == 0) {
        ex[wave][0] = s1;
        ex[wave][1] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        s1 += ex[w][0];
        s2 += ex[w][1];
      }
    }
    if (!live || !a.dx) continue;
    s1 /= static_cast<float>(a.H);
    s2 /= static_cast<float>(a.H);
    const size_t row = static_cast<size_t>(t) * a.H;
#pragma unroll
    for (int c = 0; c < kCpt; ++c) {
      const int e = (lane + c * kLanes) * N;
      if (e >= a.H) continue;
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        o[i] = rs * (g[c][i] - s1 - xh[c][i] * s2);
        if (a.dres) o[i] += res[c][i];
      }
      store_chunk<T>(static_cast<T*>(a.dx) + row + e, pack_chunk<T>(o), a.H - e);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = a.part + (static_cast<size_t>(blockIdx.x) * 2 + which) * a.H;
    float (&v)[kCpt][N] = which ? db : dw;
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kCpt; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i)
          sums[((group * kCpt + c) * N + i) * kLanes + lane] = v[c][i];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int c = 0; c < kCpt; ++c)
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int q = 1; q < kRows; ++q) v[c][i] += sums[((q * kCpt + c) * N + i) * kLanes + lane];
      }
    }
    if (group == 0) {
#pragma unroll
      for (int c = 0; c < kCpt; ++c) {
        const int e = (lane + c * kLanes) * N;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (e + i < a.H) out[e + i] = v[c][i];
      }
    }
  }
}

// dw, db = sums over the n rows of part; 64 columns a workgroup, its 16 waves' rows
// joined in LDS in their order.
constexpr int kSumWaves = 16;

template <typename W>
__global__ __launch_bounds__(kSumWaves* kWave) void layer_norm_sum_kernel(const float* part, int n,
                                                                           int H, W* dw, W* db) {
  __shared__ float s[kSumWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int which = blockIdx.y, col = blockIdx.x * kWave + lane;
  float v = 0.f;
  if (col < H) {
    const float* p = part + static_cast<size_t>(which) * H + col;
#pragma unroll 8
    for (int i = wave; i < n; i += kSumWaves) v += p[static_cast<size_t>(i) * 2 * H];
  }
  s[wave][lane] = v;
  __syncthreads();
  W* out = which ? db : dw;
  if (wave == 0 && col < H && out) {
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kSumWaves; ++w) v += s[w][lane];
    out[col] = from_f32<W>(v);
  }
}

template <typename T, typename W>
hipError_t launch_fwd(const LayerNormArgs& a, hipStream_t s) {
  constexpr int N = Vec16<T>::N;
  const int chunks = (a.H + N - 1) / N;
  if (chunks <= kWave)
    layer_norm_kernel<T, W, 1, 1><<<dim3((a.T + 3) / 4), dim3(kFwdThreads), 0, s>>>(a);
  else if (chunks <= 2 * kWave)
    layer_norm_kernel<T, W, 1, 2><<<dim3((a.T + 3) / 4), dim3(kFwdThreads), 0, s>>>(a);
  else if (chunks <= kFwdThreads)
    layer_norm_kernel<T, W, 4, 1><<<dim3(a.T), dim3(kFwdThreads), 0, s>>>(a);
  else if (chunks <= 2 * kFwdThreads)
    layer_norm_kernel<T, W, 4, 2><<<dim3(a.T), dim3(kFwdThreads), 0, s>>>(a);
  else if (chunks <= 4 * kFwdThreads)
    layer_norm_kernel<T, W, 4, 4><<<dim3(a.T), dim3(kFwdThreads), 0, s>>>(a);
  else if (chunks <= 8 * kFwdThreads)
    layer_norm_kernel<T, W, 4, 8><<<dim3(a.T), dim3(kFwdThreads), 0, s>>>(a);
  else
    return hipErrorInvalidValue;
  return hipGetLastError();
}

template <typename T, typename W>
hipError_t launch_bwd(const LayerNormBwdArgs& a, hipStream_t s) {
  constexpr int N = Vec16<T>::N;
  const int chunks = (a.H + N - 1) / N;
  const dim3 grid(layer_norm_bwd_parts(a.T, a.H, sizeof(T) == 4 ? MOE355_F32 : MOE355_BF16));
  const dim3 block(kBwdThreads);
  if (chunks <= kWave)
    layer_norm_bwd_kernel<T, W, 1, 1><<<grid, block, 0, s>>>(a);
  else if (chunks <= 2 * kWave)
    layer_norm_bwd_kernel<T, W, 1, 2><<<grid, block, 0, s>>>(a);
  else if (chunks <= 4 * kWave)
    layer_norm_bwd_kernel<T, W, 2, 2><<<grid, block, 0, s>>>(a);
  else if (chunks <= 8 * kWave)
    layer_norm_bwd_kernel<T, W, 4, 2><<<grid, block, 0, s>>>(a);
  else if (chunks <= 16 * kWave)
    layer_norm_bwd_kernel<T, W, 8, 2><<<grid, block, 0, s>>>(a);
  else if (chunks <= 32 * kWave)
    layer_norm_bwd_kernel<T, W, 8, 4><<<grid, block, 0, s>>>(a);
  else
    return hipErrorInvalidValue;
  if (a.part) {
    const dim3 cols((a.H + kWave - 1) / kWave, 2);
    layer_norm_sum_kernel<W><<<cols, dim3(kSumWaves * kWave), 0, s>>>(
        a.part, static_cast<int>(grid.x), a.H, static_cast<W*>(a.dw), static_cast<W*>(a.db));
  }
  return hipGetLastError();
}

template <typename F>
hipError_t by_types(int dtype, int weight_dtype, F f) {
  auto w = [&](auto t) {
    if (weight_dtype == MOE355_F32) return f(t, float());
    if (weight_dtype == MOE355_BF16) return f(t, bf16());
    return f(t, f16());
  };
  if (dtype == MOE355_F32) return w(float());
  if (dtype == MOE355_BF16) return w(bf16());
  return w(f16());
}

}  // namespace

int layer_norm_bwd_parts(int T, int H, int dtype) {
  const int chunks = dtype == MOE355_F32 ? (H + 3) / 4 : (H + 7) / 8;
  int waves = 1;
  while (waves < 8 && chunks > 2 * kWave * waves) waves *= 2;
  const int rows = kBwdThreads / (kWave * waves);
  const int groups = (T + rows - 1) / rows;
  return groups < device_cu_count() ? groups : device_cu_count();
}

hipError_t launch_layer_norm(const LayerNormArgs& a, int dtype, hipStream_t s) {
  return by_types(dtype, a.weight_dtype, [&](auto t, auto w) {
    return launch_fwd<decltype(t), decltype(w)>(a, s);
  });
}

hipError_t launch_layer_norm_bwd(const LayerNormBwdArgs& a, int dtype, hipStream_t s) {
  return by_types(dtype, a.weight_dtype, [&](auto t, auto w) {
    return launch_bwd<decltype(t), decltype(w)>(a, s);
  });
}

}  // namespace moe355
