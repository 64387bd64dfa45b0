// Grouped expert FFN on 4-bit weights and 8-bit tokens (formats: mx.h) for few tokens
// per expert:
//   g, u = deq(x) . deq(w1)^T;  h = act(g) * u in 8 bits;  y = deq(h) . deq(w2)^T
// Then the weights, read once, bound it. A workgroup owns one supergroup (64 packed
// rows) of one expert and a tile of up to 16 of its tokens; its four waves split the
// columns, two steps of 4 KB each in flight, and add their sums in LDS in a fixed
// order. Weights sit on the M side of the product, tokens on the N side, so a lane
// ends with 4 consecutive features of one token per group. The products are exact
// (mx_mma.h) whatever the result's type is: the weights' stream hides them but for 2 to
// 5 % (us with scaled products / with these: 8 experts of H 4096, I 14336, one token 39.0 /
// 40.7, 8 rows each 79 + 53 / 82 + 56; 64 of H 2048, I 1408, 16 tokens of 6 slots 50.1 / 50.9).
// Weights of 8 experts of H 4096, I 14336 stream at 6.1 and 4.5 TB/s (gate|up and down, 8 rows
// each: 82 and 56 us), of the 51 of 64 experts of H 2048, I 1408 that 16 tokens reach at 5.3
// and 4.8 (29 and 16 us), of two experts of the former for one token at 5.0 and 4.9 (25 and
// 13 us).
#include "dma_pipe.h"
#include "mx.h"

namespace moe355 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
#include "mx_mma.h"

template <bool kGateUp>
__global__ __launch_bounds__(kThreads) void mx_ffn_kernel(const MxFfnArgs a) {
  constexpr int D = 2;  // steps in flight per wave (4 need more registers and gain nothing)
  __shared__ f32x4 red[kWaves][4][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int ttile = blockIdx.x, sg = blockIdx.y, split = blockIdx.z;
  if (ttile >= a.tile_map[0]) return;
  const int e = a.tile_map[2 + 2 * ttile];
  const int row0 = a.tile_map[3 + 2 * ttile];
  const int row_end = min(row0 + kMxStreamTile, a.offsets[e + 1]);

  const int steps = a.Kp / kMxStep;
  const int sbeg = min(split * a.steps_per_split, steps);
  const int send = min(sbeg + a.steps_per_split, steps);
  const int per = (send - sbeg + kWaves - 1) / kWaves;
  const int s0 = min(sbeg + wave * per, send), n = min(s0 + per, send) - s0;

  const uint8_t* w = a.w + e * a.w_stride + (static_cast<size_t>(sg) * steps + s0) * 4 * kMxTileBytes +
                     lane * 16;
  const uint32_t* ws = a.w_scales + e * a.ws_stride + (static_cast<size_t>(sg) * steps + s0) * kWave + lane;
  const int q = lane >> 4, row = row0 + (lane & 15);
  // rows past the tile's last read its first; their results are not stored
  const int p = row < row_end ? row : row0;
  const size_t src = kGateUp ? a.row_src[p] : p;
  const uint8_t* xp = a.x + src * a.Kp + s0 * kMxStep + 32 * q;
  const uint8_t* xsp = a.x_scales + src * (a.Kp / kMxBlock) + s0 * (kMxStep / kMxBlock);

  u32x4 wr[D][4], xr[D][2];
  uint32_t wsr[D], xsr[D];
  auto issue = [&](int slot, int st) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      wr[slot][g] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(w + static_cast<size_t>(st) * 4 * kMxTileBytes + g * kMxTileBytes));
    wsr[slot] = ws[st * kWave];
    const u32x4* x = reinterpret_cast<const u32x4*>(xp + st * kMxStep);
    xr[slot][0] = x[0];
    xr[slot][1] = x[1];
    xsr[slot] = *reinterpret_cast<const uint32_t*>(xsp + st * (kMxStep / kMxBlock));
  };
  f32x4 acc[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto consume = [&](int slot) {
    const uint32_t s = wsr[slot], xs = xsr[slot] >> (8 * q);
    const u32x4* x = xr[slot];
    const float xf = scale_of(xs & 0xffu);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 t = tokens_bf16(x[j / 2][2 * (j % 2)], x[j / 2][2 * (j % 2) + 1], xf);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            weights_bf16(wr[slot][g][j], scale_of((s >> (8 * g)) & 0xffu)), t, acc[g], 0, 0, 0);
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < n) issue(d, d);
  for (int st = 0; st < n; st += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (st + d < n) {
        consume(d);
        if (st + d + D < n) issue(d, st + d + D);
      }
    }
  }

#pragma unroll
  for (int g = 0; g < 4; ++g) red[wave][g][lane] = acc[g];
  __syncthreads();
  if constexpr (kGateUp) {
    if (wave != 0) return;
    f32x4 v[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      v[g] = red[0][g][lane];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) v[g] += red[k][g][lane];
    }
    by_activation(a.act, [&](auto act) {
      float h[8];
      uint32_t amax = gated_block<act.value, true>(v, h);
      if (amax == kInfBits) amax = finite_max(h);
      const int scale = mx8_scale(__uint_as_float(block_max(amax)));
      if (row >= row_end) return;
      *reinterpret_cast<u32x2*>(a.out_codes + static_cast<size_t>(row) * a.Ip + sg * kMxBlock + 8 * q) =
          mx8_codes(h, scale);
      if (q == 0)
        a.out_scales[static_cast<size_t>(row) * (a.Ip / kMxBlock) + sg] = static_cast<uint8_t>(scale);
    });
  } else {
    // Group g by wave g.
    const int g = wave, col = sg * kMxSuper + 16 * g + 4 * q;
    f32x4 v = red[0][g][lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) v += red[k][g][lane];
    if (row < row_end && col < a.H)
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + (static_cast<size_t>(split) * a.R + row) * a.H +
                                col) = v;
  }
}

template <bool kGateUp>
hipError_t launch_t(const MxFfnArgs& a, hipStream_t s) {
  if (a.max_tiles == 0) return hipSuccess;
  const dim3 grid(a.max_tiles, a.n_super, a.splits), block(kThreads);
  mx_ffn_kernel<kGateUp><<<grid, block, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_gate_up(const MxFfnArgs& a, hipStream_t s) { return launch_t<true>(a, s); }

hipError_t launch_mx_down(const MxFfnArgs& a, hipStream_t s) { return launch_t<false>(a, s); }

}  // namespace moe355
