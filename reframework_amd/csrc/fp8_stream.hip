// Grouped product of 8-bit rows and 8-bit weights (formats: fp8.h) for few rows per matrix:
// the weights stream from memory past 16 token rows at a time.
//
// A wave multiplies two 16-row weight tiles, straight from memory in the layout of the
// matrix instruction; kSplit waves share the columns of a tile and add their sums in
// LDS. gate_up: the two tiles are gate and up of the same 16 features and 8 such pairs make a
// workgroup, so that it holds whole blocks of 128 features and can leave them in 8 bits.
#include "fp8.h"

namespace moe355 {
namespace {

#include "fp8_mma.h"

template <bool kGateUp, int kPairs, int kSplit, bool kExact, typename OutT>
__global__ __launch_bounds__(kPairs* kSplit* kWave, 4) void stream_kernel(const F8MatmulArgs a) {
  constexpr int kThreads = kPairs * kSplit * kWave;
  constexpr int kUnroll = kGateUp ? 3 : 4;  // steps whose operands are loaded at once
  __shared__ f32x4 part[kSplit > 1 ? kSplit - 1 : 1][kPairs][2][kWave];
  __shared__ float most[kPairs][16];
  const int lane = threadIdx.x & (kWave - 1), q = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int pair = wave % kPairs, split = wave / kPairs;
  if constexpr (!kGateUp) zero_rest<OutT, kThreads>(a);

  const int I = a.N / 2;
  const int groups = kGateUp ? f8_blocks(I) : (a.N + 32 * kPairs - 1) / (32 * kPairs);
  const int group = blockIdx.x % groups;
  const RowTile t = find_tile(a, kF8StreamTile, blockIdx.x / groups);
  if (t.e < 0) return;

  const int steps = a.Kp / kF8Block;
  // this wave's two tiles: their first rows and, of the scales, their blocks of rows
  const int first = (group * kPairs + pair) * (kGateUp ? 16 : 32);
  const int cell_rows = f8_cell_rows(a.N, kGateUp);
  const uint8_t* wp[2];
  const float* ws[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    // Rows past the matrix's last: cells are padded; tiles past the last cell read it again. Those
    // results are not stored.
    const int n = first + (kGateUp ? 0 : 16 * j);
    const int block = min(n / kF8Block + (kGateUp && j ? cell_rows / 2 : 0), cell_rows - 1);
    const size_t cells = (static_cast<size_t>(t.e) * cell_rows + block) * steps;
    wp[j] = a.w + cells * kF8Cell + n % kF8Block / 16 * kF8Tile + lane * 16;
    ws[j] = a.w_scales + cells;
  }
  const int row = min(t.row0 + r, t.row_end - 1);  // tokens past the last: it again
  const size_t src = a.row_src ? a.row_src[row] : row;
  const uint8_t* xp = a.x + src * a.Kp + q * 16;
  const float* xs = a.x_scales + src * steps;

  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  // kCount steps from k0 on, straight-line (mma_f8), all their operands loaded at once.
  auto run = [&](int k0, auto count) {
    constexpr int kCount = decltype(count)::value;
    u32x4 w[kCount][2][2], x[kCount][2];
    float sx[kCount], sw[kCount][2];
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      const int k = k0 + u * kSplit;
      const size_t at = static_cast<size_t>(k) * kF8Block;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        w[u][j][0] = *reinterpret_cast<const u32x4*>(wp[j] + at * kF8Block);
        w[u][j][1] = *reinterpret_cast<const u32x4*>(wp[j] + at * kF8Block + kF8Tile / 2);
        sw[u][j] = ws[j][k];
      }
      x[u][0] = *reinterpret_cast<const u32x4*>(xp + at);
      x[u][1] = *reinterpret_cast<const u32x4*>(xp + at + 64);
      sx[u] = xs[k];
    }
#pragma unroll
    for (int u = 0; u < kCount; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 p = kExact ? mma_f8_exact(to_bf16(w[u][j]), to_bf16(x[u])) : mma_f8(w[u][j], x[u]);
        const float s = sx[u] * sw[u][j];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(p[i], s, acc[j][i]);
      }
  };
  int k0 = split, left = (steps - split + kSplit - 1) / kSplit;  // this wave's steps
  for (; left >= kUnroll; left -= kUnroll, k0 += kUnroll * kSplit)
    run(k0, std::integral_constant<int, kUnroll>());
  static_assert(kUnroll <= 4, "what may be left");
  if (kUnroll > 3 && left == 3) run(k0, std::integral_constant<int, 3>());
  if (left == 2) run(k0, std::integral_constant<int, 2>());
  if (left == 1) run(k0, std::integral_constant<int, 1>());
  if constexpr (kSplit > 1) {
    if (split > 0) {
#pragma unroll
      for (int j = 0; j < 2; ++j) part[split - 1][pair][j][lane] = acc[j];
    }
    __syncthreads();
    if (split == 0) {
#pragma unroll
      for (int s = 0; s < kSplit - 1; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[j] += part[s][pair][j][lane];
    }
  }
  const bool live = t.row0 + r < t.row_end;
  if constexpr (!kGateUp) {
    if (split == 0 && live) {
#pragma unroll
      for (int j = 0; j < 2; ++j) store_results<OutT>(a, row, first + 16 * j + 4 * q, acc[j]);
    }
  } else {
    float h[4], amax = 0.f;
    if (split == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = first + 4 * q + i < I ? gate_act(a.act, acc[0][i]) * acc[1][i] : 0.f;
        amax = fmaxf(amax, f8_finite_abs(h[i]));
      }
      amax = fmaxf(amax, __shfl_xor(amax, 16, kWave));
      amax = fmaxf(amax, __shfl_xor(amax, 32, kWave));
      if (q == 0) most[pair][r] = amax;
    }
    __syncthreads();
    if (split == 0 && live) {
#pragma unroll
      for (int p = 0; p < kPairs; ++p) amax = fmaxf(amax, most[p][r]);
      const F8Div d = f8_div(amax);
      const size_t Ip = f8_pad(I);
      *reinterpret_cast<uint32_t*>(a.out_codes + row * Ip + first + 4 * q) = f8_codes4(h, d);
      if (pair == 0 && q == 0) a.out_scales[row * (Ip / kF8Block) + group] = d.scale;
    }
  }
}

// Workgroups at most: every matrix that has rows has a tile that is not full.
long long stream_groups(const F8MatmulArgs& a, bool gate_up) {
  const long long groups = gate_up ? f8_blocks(a.N / 2) : (a.N + 31) / 32;
  return groups * (a.offsets ? a.M / kF8StreamTile + (a.E < a.M ? a.E : a.M)
                             : (a.M + kF8StreamTile - 1) / kF8StreamTile);
}

template <bool kGateUp, int kPairs, int kSplit, bool kExact, typename OutT>
hipError_t launch(const F8MatmulArgs& a, hipStream_t s) {
  const long long groups = stream_groups(a, kGateUp);
  if (groups > 0x7fffffffll) return hipErrorInvalidValue;
  stream_kernel<kGateUp, kPairs, kSplit, kExact, OutT>
      <<<dim3(static_cast<unsigned>(groups)), dim3(kPairs * kSplit * kWave), 0, s>>>(a);
  return hipGetLastError();
}

// More waves share a tile's columns where there are few tiles. us with 4 / 8 waves: 256 workgroups
// (2 rows of 2 matrices, 4096 x 14336) 26.6 / 23.6, 128 (1 row, 4096 x 4096) 8.0 / 7.3, 896
// (2 rows of 2, 14336 x 4096) 23.1 / 25.3, 5632 (96 rows of 64, 2816 x 2048) 62 / 73.
template <bool kExact, typename OutT>
hipError_t launch_product(const F8MatmulArgs& a, hipStream_t s) {
  return stream_groups(a, false) <= 2ll * device_cu_count() ? launch<false, 1, 8, kExact, OutT>(a, s)
                                                            : launch<false, 1, 4, kExact, OutT>(a, s);
}

}  // namespace

hipError_t launch_f8_stream(const F8MatmulArgs& a, bool gate_up, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  // Two waves a pair of tiles, as above, gain nothing here: whole calls, us with 1 / 2, 1 token
  // of 8 experts of H 4096, I 14336 88 / 87, of H 1024, I 1024 18.6 / 18.2; 16 tokens of 64 of H
  // 2048, I 1408 100 / 103.
  if (gate_up) return a.exact ? launch<true, 8, 1, true, float>(a, s) : hipErrorInvalidValue;
  if (a.exact) return launch_product<true, float>(a, s);
  if (a.out_dtype == MOE355_F32) return launch_product<false, float>(a, s);
  if (a.out_dtype == MOE355_BF16) return launch_product<false, bf16>(a, s);
  return launch_product<false, f16>(a, s);
}

}  // namespace moe355
