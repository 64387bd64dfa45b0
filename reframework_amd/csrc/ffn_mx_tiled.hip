// Grouped expert FFN on 4-bit weights and 8-bit tokens (formats: mx.h) for many tokens
// per expert: an item multiplies BM token rows of one expert by 256 packed weight rows
// (4 supergroups: 128 features of gate and up), 128 columns a step.
//
// Tokens (128 bytes a row and step), weights (64) and both scales go straight to
// LDS, several steps deep. Token rows are stored with their 16-byte chunks XORed by
// half the row number, which leaves the fragment reads without bank conflicts;
// weight tiles lie in fragment order already.
//
// Eight waves, two per SIMD, work in turns: while the first four multiply a step, the
// others read theirs from LDS, and a barrier swaps them, so that the matrix cores
// always have a wave with its operands in registers. Only gate_up's 64-row tiles, of
// which two workgroups share a CU, do without turns: all waves read and multiply a step
// between two barriers, and the other workgroup fills the gaps.
//
// Rates (random codes): 8 experts of 1024 rows, 4096 x 14336, 256-row tiles, gate|up 740 us
// (2.60 PFLOP/s), down 342 (2.81), matrix cores 73 to 76 % busy at 1.73 to 1.98 GHz, so bound
// by power (a long run of one launch after the other falls to 805 and 350); 64 experts of
// 384 rows, 2048 x 1408: 152 and 85 us, bound by the epilogues and load latency of items of
// 16 and 11 steps; 8 of 49 rows, exact, 64-row tiles: 123 and 68 us, 4.0 TB/s of weights. One
// barrier a step instead of two, with the groups half a step apart, takes 865 and 387 us in
// a long run of the first of these.
//
// A workgroup runs several items, whose steps follow each other in one stream of
// loads: the first steps of an item are on their way while the item before it is
// multiplied and stored.
#include <climits>

#include "dma_pipe.h"
#include "mx.h"

namespace moe355 {
namespace {

#include "mx_mma.h"

constexpr int kBN = 256;
constexpr int kWaves = 8, kThreads = kWaves * kWave;
constexpr int kMaxItems = 32;  // items of a workgroup

// BM token rows, WM waves over them and 8 / WM over the weight rows; kPerCu workgroups
// share a CU.
template <int BM, int WM, int kPerCu>
struct Shape {
  static constexpr int kMT = BM / WM / 16, kNT = kBN / (kWaves / WM) / 16;  // 16 x 16 tiles of a wave
  static constexpr int kTokBytes = BM * kMxStep;          // codes of the tokens
  static constexpr int kWgtBytes = kBN * kMxStep / 2;     // codes of the weights
  static constexpr int kTokScale = BM * 4;                // a dword per row
  static constexpr int kWgtScale = kBN / kMxSuper * kWave * 4;
  static constexpr int kStage = kTokBytes + kWgtBytes + kTokScale + kWgtScale;
  static constexpr int kStages = (160 * 1024 / kPerCu - kMaxItems * 16) / kStage;
  // direct-to-LDS loads of a wave per step: 1 KB of codes each, and 256 bytes of
  // scales (the weights' four by waves 0-3, the tokens' by the others, some twice)
  static constexpr int kTokLoads = kTokBytes / 1024 / kWaves;
  static constexpr int kWgtLoads = kWgtBytes / 1024 / kWaves;
  static constexpr int kLoads = kTokLoads + kWgtLoads + 1;
  static_assert(kNT % 4 == 0 && kMT >= 1 && kTokLoads >= 1 && kWgtLoads >= 1, "whole supergroups");
  static_assert(kStages >= 3 && (kStages - 1) * kLoads < 64, "pipeline");
};

__device__ __forceinline__ void dma4_rsrc(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff,
                                          uint8_t* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (pipe::lds_void*)(dst), 4, off, soff, 0, 0);
}

// Item L: weight tile `wt` of the token rows [row0, row_end) of expert e, split z of
// the columns. The token tiles of an expert vary fastest, so that neighbours (on one
// XCD) share their weights.
struct Item {
  int e_split, row0, row_end, wt;  // e_split: expert + 256 * split
};

template <int BM>
__device__ __forceinline__ Item decode_item(const MxFfnArgs& a, int L, int nw, int per_split) {
  const int split = L / per_split, rem = L - split * per_split;
  const int t0 = rem / nw;
  const int e = a.tile_map[2 + 2 * t0];
  const int eb = a.offsets[e], ee = a.offsets[e + 1];
  const int b = t0 - (a.tile_map[3 + 2 * t0] - eb) / BM;  // the expert's first tile
  const int ne = (ee - eb + BM - 1) / BM;
  const int r2 = rem - b * nw, wt = r2 / ne;
  const int row0 = eb + (r2 - wt * ne) * BM;
  return Item{e + 256 * split, row0, min(row0 + BM, ee), wt};
}

__device__ __forceinline__ u32x2 pack_f16(f32x4 v) {
  typedef f16 f16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, f16x4{from_f32<f16>(v[0]), from_f32<f16>(v[1]),
                                         from_f32<f16>(v[2]), from_f32<f16>(v[3])});
}

template <bool kGateUp, int BM, int WM, int kPerCu, bool kExact>
__global__ __launch_bounds__(kThreads, 2 * kPerCu) void mx_tiled_kernel(const MxFfnArgs a) {
  typedef Shape<BM, WM, kPerCu> S;
  // gate_up of 64-row tiles without turns, with: 13.1 / 15.4 us (8 x 128 rows,
  // 2048 x 1408), 42 / 46 us (32 x 128, 1280 x 3328); 137 / 146 us (8 x 49, 4096 x 14336,
  // exact). down, whose items are fewer and longer: 34 / 30, 170 / 112 us (scaled).
  constexpr bool kTurns = !(kGateUp && kPerCu == 2);
  constexpr int kMT = S::kMT, kNT = S::kNT;
  __shared__ __attribute__((aligned(1024))) uint8_t stage[S::kStages][S::kStage];
  __shared__ Item items[kMaxItems];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int q = lane >> 4, r = lane & 15;

  // This workgroup's items: one of every gridDim.x, the workgroups of an XCD taking
  // neighbouring ones, each time some further: otherwise experts of two tiles would
  // give one workgroup all full tiles and the next all partial ones (64 experts of 350
  // rows, 2048 x 1408: 153 us, so 141). Grids of 256 or 512 and kShift more share no
  // factor up to 16 with the number of tiles.
  constexpr int kShift = 15;
  const int nw = (a.n_super * kMxSuper + kBN - 1) / kBN;
  const int per_split = a.tile_map[0] * nw, total = per_split * a.splits;
  const int G = gridDim.x, pid = blockIdx.x;
  const int rounds = total / G, tail = total - rounds * G;
  const int n_items = rounds + (pid < tail ? 1 : 0);
  if (n_items == 0) return;
  if (wave == 0 && lane < n_items) {
    const int n = lane < rounds ? G : tail;
    items[lane] = decode_item<BM>(a, lane * G + (xcd_remap(pid, n) + kShift * lane) % n, nw, per_split);
  }
  __syncthreads();
  auto item_at = [&](int j) {
    const Item* p = &items[j];
    return Item{__builtin_amdgcn_readfirstlane(p->e_split), __builtin_amdgcn_readfirstlane(p->row0),
                __builtin_amdgcn_readfirstlane(p->row_end), __builtin_amdgcn_readfirstlane(p->wt)};
  };
  const int steps = a.Kp / kMxStep;
  auto first_step = [&](const Item& it) { return (it.e_split >> 8) * a.steps_per_split; };
  auto n_steps = [&](const Item& it) {
    return min(first_step(it) + a.steps_per_split, steps) - first_step(it);
  };

  // Token rows whose codes (kTokLoads of them) and scales this lane loads, as rows of
  // x; -1 past the tile's last row.
  const int tok64 = (wave & 3) % (BM / 64);  // 64 tokens whose scales waves 4-7 load
  int src[S::kTokLoads + 1];
  auto load_rows = [&](const Item& it) {
#pragma unroll
    for (int i = 0; i <= S::kTokLoads; ++i) {
      const int row = i < S::kTokLoads ? 8 * (wave * S::kTokLoads + i) + (lane >> 3) : 64 * tok64 + lane;
      const int p = it.row0 + row;
      src[i] = p >= it.row_end ? -1 : kGateUp ? a.row_src[p] : row;
    }
  };

  // The item whose steps are being loaded: sources, and this lane's offsets.
  __amdgpu_buffer_rsrc_t xsrc, xssrc, wsrc, wssrc;
  uint32_t xoff[S::kTokLoads], woff[S::kWgtLoads], soff;
  int load_item = 0, load_step, load_end, loaded = 0;  // loaded: steps of all items
  auto begin_loads = [&](const Item& it) {
    const int e = it.e_split & 255;
    const int sg0 = it.wt * (kBN / kMxSuper);
    // down: rows are counted from the tile's first, so that offsets stay small
    const size_t first = kGateUp ? 0 : it.row0;
    xsrc = pipe::lds_rsrc(a.x + first * a.Kp);
    xssrc = pipe::lds_rsrc(a.x_scales + first * (a.Kp / kMxBlock));
    wsrc = pipe::lds_rsrc(a.w + e * a.w_stride + static_cast<size_t>(sg0) * steps * 4 * kMxTileBytes);
    wssrc = pipe::lds_rsrc(a.w_scales + e * a.ws_stride + static_cast<size_t>(sg0) * steps * kWave);
    // The last weight tile of a matrix of an odd number of 128 rows reads its last
    // supergroup again; those results are not stored.
    const int last = a.n_super - 1 - sg0;
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i) {
      const int row = 8 * (wave * S::kTokLoads + i) + (lane >> 3);
      xoff[i] = src[i] < 0 ? pipe::kPadOffset  // out of range: zeros
                           : static_cast<uint32_t>(src[i]) * a.Kp + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < S::kWgtLoads; ++i) {
      const int c = wave * S::kWgtLoads + i;  // tile c % 4 of supergroup c / 4
      woff[i] = static_cast<uint32_t>(min(c >> 2, last)) * steps * 4 * kMxTileBytes +
                (c & 3) * kMxTileBytes + lane * 16;
    }
    soff = wave < 4 ? (static_cast<uint32_t>(min(wave, last)) * steps * kWave + lane) * 4
           : src[S::kTokLoads] < 0 ? pipe::kPadOffset
                                   : static_cast<uint32_t>(src[S::kTokLoads]) * (a.Kp / kMxBlock);
    load_step = first_step(it);
    load_end = load_step + n_steps(it);
    if (load_item + 1 < n_items) load_rows(item_at(load_item + 1));
  };
  // Loads the next step of the stream, if there is one.
  auto load = [&]() {
    if (load_item >= n_items) return;
    uint8_t* s = stage[loaded % S::kStages];
    const int k = load_step;
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i)
      pipe::dma16_rsrc(xsrc, xoff[i], k * kMxStep, s + (wave * S::kTokLoads + i) * 1024);
#pragma unroll
    for (int i = 0; i < S::kWgtLoads; ++i)
      pipe::dma16_rsrc(wsrc, woff[i], k * 4 * kMxTileBytes,
                       s + S::kTokBytes + (wave * S::kWgtLoads + i) * 1024);
    uint8_t* ts = s + S::kTokBytes + S::kWgtBytes;
    if (wave < 4)
      dma4_rsrc(wssrc, soff, k * kWave * 4, ts + S::kTokScale + wave * 256);
    else
      dma4_rsrc(xssrc, soff, k * (kMxStep / kMxBlock), ts + tok64 * 256);
    ++loaded;
    if (++load_step == load_end && ++load_item < n_items) begin_loads(item_at(load_item));
  };
  // Waits until this wave's loads of step `step` of the stream have landed; of the
  // steps after it kStages - 2 may be in flight (fewer at the end of the stream, where
  // it waits for all).
  auto landed = [&](int step) {
    if (loaded >= step + S::kStages - 1)
      pipe::wait_vmcnt<(S::kStages - 2) * S::kLoads>();
    else
      pipe::wait_vmcnt<0>();
  };
  // All waves; nothing moves across it.
  auto turn = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_sched_barrier(0);
  };

  load_rows(item_at(0));
  begin_loads(item_at(0));
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) load();
  // Half-step 2 s: the first waves read step s of the stream, the second multiply step
  // s - 1; the next half-step the other way round. Before half-step 2 s every wave
  // has seen its loads of step s land; the buffer of step s - 1 was last read in
  // half-step 2 s - 1 and is filled again from half-step 2 s on.
  const bool second = wave >= 4;
  if constexpr (kTurns) {
    landed(0);
    turn();
    if (second) turn();
  }
  int done = 0;  // steps of the stream
  const int wm = wave % WM, wn = wave / WM;  // this wave's tokens and weight rows
  for (int j = 0; j < n_items; ++j) {
    const Item it = item_at(j);
    const int n = n_steps(it);
    f32x4 acc[kMT][kNT];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int g = 0; g < kNT; ++g) acc[m][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    // A wave has every WM-th 16 rows of the tile, so that the waves share the rows of
    // one that is not full; mt of its kMT hold any.
    const int mt = min((it.row_end - it.row0 + 16 * (WM - 1 - wm) + 15) / (16 * WM), kMT);
    auto run_steps = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      for (int st = 0; st < n; ++st, ++done) {
        if constexpr (!kTurns) {
          // Every wave has read step `done` - 1, whose buffer is filled again, and has
          // seen its loads of step `done` land.
          landed(done);
          pipe::wait_lgkm0();
          turn();
          load();
        }
        const uint8_t* s = stage[done % S::kStages];
        const uint8_t* wtile = s + S::kTokBytes + wn * (kNT * kMxTileBytes) + lane * 16;
        const uint8_t* ts = s + S::kTokBytes + S::kWgtBytes + (16 * wm + r) * 4;
        const uint8_t* ws = s + S::kTokBytes + S::kWgtBytes + S::kTokScale + wn * (kNT / 4 * 256) + lane * 4;
        u32x4 w[kNT];
        uint32_t wsc[kNT / 4];
#pragma unroll
        for (int g = 0; g < kNT; ++g) w[g] = *reinterpret_cast<const u32x4*>(wtile + g * kMxTileBytes);
#pragma unroll
        for (int h = 0; h < kNT / 4; ++h) wsc[h] = *reinterpret_cast<const uint32_t*>(ws + 256 * h);
        u32x4 x[kMT][2];
        uint32_t xs[kMT];
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          if (!kFull && m >= mt) continue;
          const int row = 16 * (wm + WM * m) + r, sw = (row >> 1) & 7;
          const uint8_t* p = s + row * kMxStep;
          x[m][0] = *reinterpret_cast<const u32x4*>(p + (((kExact ? 2 * q : q) ^ sw) << 4));
          x[m][1] = *reinterpret_cast<const u32x4*>(p + (((kExact ? 2 * q + 1 : 4 + q) ^ sw) << 4));
          xs[m] = *reinterpret_cast<const uint32_t*>(ts + 64 * WM * m) >> (8 * q);
        }
        if constexpr (kTurns) {
          load();
          if (second) landed(done + 1);
          pipe::wait_lgkm0();
          turn();
        }
        // Conversions and products go before other waves' reads (8 experts of 49 rows,
        // 4096 x 14336: gate|up 126 us, without 136; the scaled products do not care).
        if constexpr (kExact) __builtin_amdgcn_s_setprio(1);
        if constexpr (kExact) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bf16x8 wb[kNT];
#pragma unroll
            for (int g = 0; g < kNT; ++g)
              wb[g] = weights_bf16(w[g][i], scale_of((wsc[g / 4] >> (8 * (g & 3))) & 0xffu));
#pragma unroll
            for (int m = 0; m < kMT; ++m) {
              if (!kFull && m >= mt) continue;
              const bf16x8 t = tokens_bf16(x[m][i / 2][2 * (i % 2)], x[m][i / 2][2 * (i % 2) + 1],
                                           scale_of(xs[m] & 0xffu));
#pragma unroll
              for (int g = 0; g < kNT; ++g)
                acc[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[g], t, acc[m][g], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            if (!kFull && m >= mt) continue;
#pragma unroll
            for (int h = 0; h < kNT / 4; ++h) {
              acc[m][4 * h + 0] = mma_scaled<0>(w[4 * h + 0], wsc[h], x[m], xs[m], acc[m][4 * h + 0]);
              acc[m][4 * h + 1] = mma_scaled<1>(w[4 * h + 1], wsc[h], x[m], xs[m], acc[m][4 * h + 1]);
              acc[m][4 * h + 2] = mma_scaled<2>(w[4 * h + 2], wsc[h], x[m], xs[m], acc[m][4 * h + 2]);
              acc[m][4 * h + 3] = mma_scaled<3>(w[4 * h + 3], wsc[h], x[m], xs[m], acc[m][4 * h + 3]);
            }
          }
        }
        if constexpr (kExact) __builtin_amdgcn_s_setprio(0);
        if constexpr (kTurns) {
          __builtin_amdgcn_sched_barrier(0);
          if (!second) landed(done + 1);
          turn();
        }
      }
    };
    if (it.row_end - it.row0 > BM - 16 * WM)
      run_steps(std::true_type());
    else
      run_steps(std::false_type());

    const int n_rows = it.row_end - it.row0, row1 = 16 * wm + r;
    if constexpr (kGateUp) {
      // Stored relative to the tile's first row; an offset out of range stores nothing.
      const auto codes = pipe::lds_rsrc(a.out_codes + static_cast<size_t>(it.row0) * a.Ip);
      const auto scales = pipe::lds_rsrc(a.out_scales + static_cast<size_t>(it.row0) * (a.Ip / kMxBlock));
      by_activation(a.act, [&](auto act) {
        // Two rows of blocks at once, which cover each other's latency (all at once
        // do not fit the registers).
        constexpr int kGroup = 2;
        static_assert(kMT % kGroup == 0, "rows of blocks");
#pragma unroll
        for (int m0 = 0; m0 < kMT; m0 += kGroup) {
          if (m0 >= mt) continue;
          float h[kGroup][kNT / 4][8];
          uint32_t amax[kGroup][kNT / 4], largest = 0;
#pragma unroll
          for (int m = 0; m < kGroup; ++m)
#pragma unroll
            for (int b = 0; b < kNT / 4; ++b) {
              amax[m][b] = gated_block<act.value, kExact>(&acc[m0 + m][4 * b], h[m][b]);
              largest = max(largest, amax[m][b]);
            }
          if (largest == kInfBits) {
#pragma unroll
            for (int m = 0; m < kGroup; ++m)
#pragma unroll
              for (int b = 0; b < kNT / 4; ++b) amax[m][b] = finite_max(h[m][b]);
          }
#pragma unroll
          for (int m = 0; m < kGroup; ++m)
#pragma unroll
            for (int b = 0; b < kNT / 4; ++b) amax[m][b] = block_max(amax[m][b]);
#pragma unroll
          for (int m = 0; m < kGroup; ++m) {
            const int row = row1 + 16 * WM * (m0 + m);
#pragma unroll
            for (int b = 0; b < kNT / 4; ++b) {
              const int sg = it.wt * (kBN / kMxSuper) + wn * (kNT / 4) + b;
              const int scale = mx8_scale(__uint_as_float(amax[m][b]));
              __builtin_amdgcn_raw_buffer_store_b64(
                  mx8_codes(h[m][b], scale), codes,
                  row < n_rows ? row * a.Ip + sg * kMxBlock + 8 * q : pipe::kPadOffset, 0, 0);
              __builtin_amdgcn_raw_buffer_store_b8(
                  static_cast<uint8_t>(scale), scales,
                  row < n_rows && q == 0 ? row * (a.Ip / kMxBlock) + sg : pipe::kPadOffset, 0, 0);
            }
          }
        }
      });
    } else {
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        if (m >= mt) continue;
        const int row = row1 + 16 * WM * m;
        const size_t at = (static_cast<size_t>(it.e_split >> 8) * a.R + it.row0 + row) * a.H;
        if (!kExact && a.y16) {
          // 16 bits with a scale per 64 columns (Scaled16). Two column groups are exchanged
          // between the lanes of a row so that each stores 16 bytes: 64 consecutive ones
          // of a row instead of 32 (97 us to 87 for 64 experts of 384 rows, 2048 x 1408).
          int byte[kNT / 4];
          float amax[kNT / 4], largest = 0.f;
#pragma unroll
          for (int b = 0; b < kNT / 4; ++b) {
            amax[b] = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) amax[b] = fmaxf(amax[b], fabsf(acc[m][4 * b + i / 4][i % 4]));
            largest = fmaxf(largest, amax[b]);
          }
          if (largest == INFINITY) {
#pragma unroll
            for (int b = 0; b < kNT / 4; ++b) {
              amax[b] = 0.f;
#pragma unroll
              for (int i = 0; i < 16; ++i)
                amax[b] = fmaxf(amax[b], mx_finite_abs(acc[m][4 * b + i / 4][i % 4]));
            }
          }
#pragma unroll
          for (int b = 0; b < kNT / 4; ++b) {
            const f32x4* v = &acc[m][4 * b];
            byte[b] = scaled16_byte(block_max(__float_as_uint(amax[b])));
            const float f = scaled16_factor(byte[b]);
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
              const u32x2 u = pack_f16(v[g] * f), w = pack_f16(v[g + 1] * f);
              const auto lo = __builtin_amdgcn_permlane16_swap(u[0], w[0], false, false);
              const auto hi = __builtin_amdgcn_permlane16_swap(u[1], w[1], false, false);
              const int col = it.wt * kBN + (wn * kNT + 4 * b + g + (q & 1)) * 16 + 8 * (q >> 1);
              if (row < n_rows && col < a.H)
                *reinterpret_cast<u32x4*>(static_cast<f16*>(a.y) + at + col) =
                    u32x4{lo[0], hi[0], lo[1], hi[1]};
            }
          }
          const int block = it.wt * (kBN / kMxSuper) + wn * (kNT / 4) + q;
          if (q < kNT / 4 && row < n_rows && block < a.n_super)
            a.y_scales[static_cast<size_t>(it.row0 + row) * a.n_super + block] =
                static_cast<uint8_t>(q ? byte[kNT / 4 - 1] : byte[0]);
        } else {
#pragma unroll
          for (int g = 0; g < kNT; ++g) {
            const int col = it.wt * kBN + (wn * kNT + g) * 16 + 4 * q;
            if (row < n_rows && col < a.H)
              *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at + col) = acc[m][g];
          }
        }
      }
    }
  }
  if (kTurns && !second) turn();
}

template <bool kGateUp, int BM, int WM, int kPerCu, bool kExact>
hipError_t launch_t(const MxFfnArgs& a, hipStream_t s) {
  if (a.max_tiles == 0) return hipSuccess;
  // every part of the columns has steps: the stream of loads has no empty items
  if ((a.splits - 1) * a.steps_per_split >= a.Kp / kMxStep) return hipErrorInvalidValue;
  const int nw = (a.n_super * kMxSuper + kBN - 1) / kBN;
  const long long total = static_cast<long long>(a.max_tiles) * nw * a.splits;
  if (total > INT_MAX) return hipErrorInvalidValue;
  long long grid = static_cast<long long>(device_cu_count()) * kPerCu;
  grid = total < grid ? total : grid * ((total + grid * kMaxItems - 1) / (grid * kMaxItems));
  mx_tiled_kernel<kGateUp, BM, WM, kPerCu, kExact>
      <<<dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

// Exact products (four instructions and their conversions instead of one) leave no
// registers for a 256-row tile.
template <bool kGateUp>
hipError_t launch(const MxFfnArgs& a, hipStream_t s) {
  if (a.exact)
    return a.tile_rows == 128 ? launch_t<kGateUp, 128, 2, 1, true>(a, s)
                              : launch_t<kGateUp, 64, 2, 2, true>(a, s);
  return a.tile_rows == 256 ? launch_t<kGateUp, 256, 4, 1, false>(a, s)
                            : launch_t<kGateUp, 64, 2, 2, false>(a, s);
}

}  // namespace

hipError_t launch_mx_gate_up_tiled(const MxFfnArgs& a, hipStream_t s) { return launch<true>(a, s); }

hipError_t launch_mx_down_tiled(const MxFfnArgs& a, hipStream_t s) { return launch<false>(a, s); }

}  // namespace moe355
