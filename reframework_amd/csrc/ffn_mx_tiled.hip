// Grouped expert FFN on 4-bit weights and 8-bit tokens (formats: mx.h) for many tokens
// per expert: a workgroup multiplies BM token rows of one expert by 256 packed weight
// rows (4 supergroups: 128 features of gate and up), 128 columns a step.
//
// Tokens (128 bytes a row and step), weights (64) and both scales go straight to
// LDS, kStages steps deep. Token rows are stored with their 16-byte chunks XORed by
// half the row number, which leaves the fragment reads without bank conflicts;
// weight tiles lie in fragment order already. A wave owns 64 tokens x 128 weight
// rows: per step it reads 8 KB of each operand for 32 instructions of 32 cycles, so
// that LDS is read at half of its rate while the matrix cores are busy.
#include <climits>

#include "dma_pipe.h"
#include "mx.h"

namespace moe355 {
namespace {

#include "mx_mma.h"

constexpr int kBN = 256;
constexpr int kWaveM = 64, kWaveN = 128;
constexpr int kMT = kWaveM / 16, kNT = kWaveN / 16;

template <int BM>
struct Shape {
  static constexpr int kWaves = BM / kWaveM * (kBN / kWaveN);
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kTokBytes = BM * kMxStep;          // codes of the tokens
  static constexpr int kWgtBytes = kBN * kMxStep / 2;     // codes of the weights
  static constexpr int kTokScale = BM * 4;                // a dword per row
  static constexpr int kWgtScale = kBN / kMxSuper * kWave * 4;
  static constexpr int kStage = kTokBytes + kWgtBytes + kTokScale + kWgtScale;
  static constexpr int kStages = 160 * 1024 / kStage;
  // direct-to-LDS loads of a wave per step: 1 KB of codes, 256 bytes of scales each
  static constexpr int kTokLoads = kTokBytes / 1024 / kWaves;
  static constexpr int kWgtLoads = kWgtBytes / 1024 / kWaves;
  static constexpr int kScaleLoads = BM == 256 ? 1 : 2;
  static constexpr int kLoads = kTokLoads + kWgtLoads + kScaleLoads;
};

__device__ __forceinline__ void dma4_rsrc(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff,
                                          uint8_t* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (pipe::lds_void*)(dst), 4, off, soff, 0, 0);
}

template <bool kGateUp, int BM, bool kExact>
__global__ __launch_bounds__(Shape<BM>::kThreads) void mx_tiled_kernel(const MxFfnArgs a) {
  typedef Shape<BM> S;
  static_assert(S::kStages >= 3 && (S::kStages - 1) * S::kLoads < 64, "pipeline");
  __shared__ __attribute__((aligned(1024))) uint8_t stage[S::kStages][S::kStage];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int q = lane >> 4, r = lane & 15;

  // Item: weight tile wt of token tile tt, the token tiles of an expert varying
  // fastest, so that neighbours (on one XCD) share their weights.
  const int nw = (a.n_super * kMxSuper + kBN - 1) / kBN;
  const int n_tiles = a.tile_map[0];
  const int per_split = n_tiles * nw, total = per_split * a.splits;
  if (static_cast<int>(blockIdx.x) >= total) return;
  const int item = xcd_remap(blockIdx.x, total);
  const int split = item / per_split, rem = item - split * per_split;
  const int t0 = rem / nw;
  const int e = a.tile_map[2 + 2 * t0];
  const int eb = a.offsets[e], ee = a.offsets[e + 1];
  const int height = tile_height(ee - eb, a.tile_rows);
  const int b = t0 - (a.tile_map[3 + 2 * t0] - eb) / height;
  const int ne = (ee - eb + a.tile_rows - 1) / a.tile_rows;
  const int r2 = rem - b * nw;
  const int wt = r2 / ne;
  const int row0 = a.tile_map[3 + 2 * (b + r2 - wt * ne)];
  const int row_end = min(row0 + height, ee);

  const int steps = a.Kp / kMxStep;
  const int sbeg = min(split * a.steps_per_split, steps);
  const int n = min(sbeg + a.steps_per_split, steps) - sbeg;

  // Sources. Rows past the tile's last load zeros (an offset that is out of range).
  const size_t first = kGateUp ? 0 : row0;
  const __amdgpu_buffer_rsrc_t xsrc = pipe::lds_rsrc(a.x + first * a.Kp);
  const __amdgpu_buffer_rsrc_t xssrc = pipe::lds_rsrc(a.x_scales + first * (a.Kp / kMxBlock));
  const int sg0 = wt * (kBN / kMxSuper);
  const __amdgpu_buffer_rsrc_t wsrc =
      pipe::lds_rsrc(a.w + e * a.w_stride + static_cast<size_t>(sg0) * steps * 4 * kMxTileBytes);
  const __amdgpu_buffer_rsrc_t wssrc =
      pipe::lds_rsrc(a.w_scales + e * a.ws_stride + static_cast<size_t>(sg0) * steps * kWave);
  auto token = [&](int row) {  // row of x of tile row `row`, or -1
    const int p = row0 + row;
    return p >= row_end ? -1 : kGateUp ? a.row_src[p] : row;
  };
  // The last weight tile of a matrix of an odd number of 128 rows reads its last
  // supergroup twice; those results are not stored.
  auto super = [&](int s) { return min(s, a.n_super - 1 - sg0); };
  uint32_t xoff[S::kTokLoads], woff[S::kWgtLoads], soff[S::kScaleLoads];
#pragma unroll
  for (int i = 0; i < S::kTokLoads; ++i) {
    const int row = 8 * (wave * S::kTokLoads + i) + (lane >> 3);
    const int src = token(row);
    xoff[i] = src < 0 ? pipe::kPadOffset
                      : static_cast<uint32_t>(src) * a.Kp + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < S::kWgtLoads; ++i) {
    const int c = wave * S::kWgtLoads + i;  // tile c % 4 of supergroup c / 4
    woff[i] = static_cast<uint32_t>(super(c >> 2)) * steps * 4 * kMxTileBytes +
              (c & 3) * kMxTileBytes + lane * 16;
  }
  // Scale loads: the weights' four, then the tokens' (64 rows each). With 8 waves
  // one each; with 4 waves one of each kind, the tokens' two loaded twice.
  const bool first_is_token = S::kScaleLoads == 1 && wave >= 4;
  const int tok64 = S::kScaleLoads == 1 ? wave & 3 : wave & 1;
  const int ssrc = token(64 * tok64 + lane);
  const uint32_t tok_scale = ssrc < 0 ? pipe::kPadOffset : static_cast<uint32_t>(ssrc) * (a.Kp / kMxBlock);
  const uint32_t wgt_scale = (static_cast<uint32_t>(super(wave & 3)) * steps * kWave + lane) * 4;
  soff[0] = first_is_token ? tok_scale : wgt_scale;
  if (S::kScaleLoads == 2) soff[S::kScaleLoads - 1] = tok_scale;

  auto issue = [&](int st) {
    uint8_t* s = stage[st % S::kStages];
    const int k = sbeg + st;
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i)
      pipe::dma16_rsrc(xsrc, xoff[i], k * kMxStep, s + (wave * S::kTokLoads + i) * 1024);
#pragma unroll
    for (int i = 0; i < S::kWgtLoads; ++i)
      pipe::dma16_rsrc(wsrc, woff[i], k * 4 * kMxTileBytes,
                       s + S::kTokBytes + (wave * S::kWgtLoads + i) * 1024);
    uint8_t* ts = s + S::kTokBytes + S::kWgtBytes;
    uint8_t* ws = ts + S::kTokScale;
    if (first_is_token)
      dma4_rsrc(xssrc, soff[0], k * (kMxStep / kMxBlock), ts + tok64 * 256);
    else
      dma4_rsrc(wssrc, soff[0], k * kWave * 4, ws + (wave & 3) * 256);
    if (S::kScaleLoads == 2)
      dma4_rsrc(xssrc, soff[S::kScaleLoads - 1], k * (kMxStep / kMxBlock), ts + tok64 * 256);
  };

  const int wm = wave >> 1, wn = wave & 1;  // this wave's 64 tokens and 128 weight rows
  f32x4 acc[kMT][kNT];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int g = 0; g < kNT; ++g) acc[m][g] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int st = 0; st < S::kStages - 1; ++st)
    if (st < n) issue(st);
  for (int st = 0; st < n; ++st) {
    // All but the newest kStages - 2 steps have landed, for every wave; and every wave
    // has read step st - 1, whose buffer the next load overwrites.
    pipe::wait_lgkm0();
    if (st + S::kStages - 1 <= n)
      pipe::dma_barrier<(S::kStages - 2) * S::kLoads>();
    else
      pipe::dma_barrier<0>();
    if (st + S::kStages - 1 < n) issue(st + S::kStages - 1);
    const uint8_t* s = stage[st % S::kStages];
    const uint8_t* wtile = s + S::kTokBytes + wn * (kNT * kMxTileBytes) + lane * 16;
    const uint8_t* ts = s + S::kTokBytes + S::kWgtBytes + (wm * kWaveM + r) * 4;
    const uint8_t* ws = s + S::kTokBytes + S::kWgtBytes + S::kTokScale + wn * 512 + lane * 4;
    u32x4 w[kNT];
#pragma unroll
    for (int g = 0; g < kNT; ++g) w[g] = *reinterpret_cast<const u32x4*>(wtile + g * kMxTileBytes);
    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(ws);
    const uint32_t w1 = *reinterpret_cast<const uint32_t*>(ws + 256);
    u32x4 x[kMT][2];
    uint32_t xs[kMT];
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      const int row = wm * kWaveM + 16 * m + r, sw = (row >> 1) & 7;
      const uint8_t* p = s + row * kMxStep;
      x[m][0] = *reinterpret_cast<const u32x4*>(p + (((kExact ? 2 * q : q) ^ sw) << 4));
      x[m][1] = *reinterpret_cast<const u32x4*>(p + (((kExact ? 2 * q + 1 : 4 + q) ^ sw) << 4));
      xs[m] = *reinterpret_cast<const uint32_t*>(ts + 64 * m) >> (8 * q);
    }
    if constexpr (kExact) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 wb[kNT];
#pragma unroll
        for (int g = 0; g < kNT; ++g)
          wb[g] = weights_bf16(w[g][j], scale_of(((g < 4 ? w0 : w1) >> (8 * (g & 3))) & 0xffu));
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          const bf16x8 t = tokens_bf16(x[m][j / 2][2 * (j % 2)], x[m][j / 2][2 * (j % 2) + 1],
                                       scale_of(xs[m] & 0xffu));
#pragma unroll
          for (int g = 0; g < kNT; ++g)
            acc[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[g], t, acc[m][g], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        acc[m][0] = mma_scaled<0>(w[0], w0, x[m], xs[m], acc[m][0]);
        acc[m][1] = mma_scaled<1>(w[1], w0, x[m], xs[m], acc[m][1]);
        acc[m][2] = mma_scaled<2>(w[2], w0, x[m], xs[m], acc[m][2]);
        acc[m][3] = mma_scaled<3>(w[3], w0, x[m], xs[m], acc[m][3]);
        acc[m][4] = mma_scaled<0>(w[4], w1, x[m], xs[m], acc[m][4]);
        acc[m][5] = mma_scaled<1>(w[5], w1, x[m], xs[m], acc[m][5]);
        acc[m][6] = mma_scaled<2>(w[6], w1, x[m], xs[m], acc[m][6]);
        acc[m][7] = mma_scaled<3>(w[7], w1, x[m], xs[m], acc[m][7]);
      }
    }
  }

#pragma unroll
  for (int m = 0; m < kMT; ++m) {
    const int row = row0 + wm * kWaveM + 16 * m + r;
    if constexpr (kGateUp) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        store_block<kExact>(a, &acc[m][4 * h], sg0 + 2 * wn + h, row, row_end, q);
    } else {
      float* y = a.y + (static_cast<size_t>(split) * a.R + row) * a.H;
#pragma unroll
      for (int g = 0; g < kNT; ++g) {
        const int col = wt * kBN + wn * kWaveN + 16 * g + 4 * q;
        if (row < row_end && col < a.H) *reinterpret_cast<f32x4*>(y + col) = acc[m][g];
      }
    }
  }
}

template <bool kGateUp, int BM>
hipError_t launch_t(const MxFfnArgs& a, hipStream_t s) {
  if (a.max_tiles == 0) return hipSuccess;
  const int nw = (a.n_super * kMxSuper + kBN - 1) / kBN;
  const long long grid = static_cast<long long>(a.max_tiles) * nw * a.splits;
  if (grid > INT_MAX) return hipErrorInvalidValue;
  const dim3 g(static_cast<unsigned>(grid)), block(Shape<BM>::kThreads);
  if (a.exact)
    mx_tiled_kernel<kGateUp, BM, true><<<g, block, 0, s>>>(a);
  else
    mx_tiled_kernel<kGateUp, BM, false><<<g, block, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_gate_up_tiled(const MxFfnArgs& a, hipStream_t s) {
  return a.tile_rows == 256 ? launch_t<true, 256>(a, s) : launch_t<true, 128>(a, s);
}

hipError_t launch_mx_down_tiled(const MxFfnArgs& a, hipStream_t s) {
  return a.tile_rows == 256 ? launch_t<false, 256>(a, s) : launch_t<false, 128>(a, s);
}

}  // namespace moe355
