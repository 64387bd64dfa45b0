// Grouped product of 8-bit rows and 8-bit weights (formats: fp8.h) for many rows per matrix:
// an item multiplies BM token rows by 256 weight rows (gate_up: gate and up of 128
// features, a block of the result's scales), a step of 128 columns at a time.
//
// Rows of both operands go straight to LDS, 128 bytes a row and step, with their 16-byte chunks
// XORed by half the row number, which leaves the fragment reads without bank
// conflicts. A step is one block of both operands' scales, so the matrix core sums it from
// zero and the sum is scaled and added in fp32 by the vector unit, whose instructions run beside
// the next products. Token scales go to LDS with the rows; the weights' one (gate_up: two) of a
// wave and step is a scalar load.
//
// A workgroup runs several items, whose steps follow each other in one stream of loads:
// the first steps of an item are on their way while the item before it is multiplied and
// stored.
#include <climits>

#include "dma_pipe.h"
#include "fp8.h"

namespace moe355 {
namespace {

#include "fp8_mma.h"
#include "permute_body.h"

constexpr int kBN = 256;
constexpr int kWaves = 8, kThreads = kWaves * kWave;
constexpr int kMaxItems = 32;  // items of a workgroup

typedef __attribute__((address_space(4))) float const_f32;

// BM token rows, WM waves over them and 8 / WM over the weight rows.
template <int BM, int WM>
struct Shape {
  static constexpr int kWN = kWaves / WM;
  static constexpr int kMT = BM / WM / 16, kNT = kBN / kWN / 16;  // 16 x 16 tiles of a wave
  static constexpr int kTokBytes = BM * kF8Block;
  static constexpr int kWgtBytes = kBN * kF8Block;
  static constexpr int kStage = kTokBytes + kWgtBytes + BM * 4;
  static constexpr int kSpare = kMaxItems * 16 + (kMaxExperts + 1) * 8 + kWN * BM * 4 + 64;
  static constexpr int kStages = (160 * 1024 - kSpare) / kStage;
  // direct-to-LDS loads of a wave per step: 1 KB of codes each, and 256 bytes of scales
  // (some waves' a second time)
  static constexpr int kTokLoads = kTokBytes / 1024 / kWaves;
  static constexpr int kWgtLoads = kWgtBytes / 1024 / kWaves;
  static constexpr int kLoads = kTokLoads + kWgtLoads + 1;
  static_assert(kMT >= 1 && kNT >= 2 && kTokLoads >= 1, "tiles of a wave");
  static_assert(kStages >= 2 && (kStages - 1) * kLoads < 64, "pipeline");
};

// Weight tile `wt` of the token rows [row0, row_end) of matrix e.
struct Item {
  int e, row0, row_end, wt;
};

template <bool kGateUp, int BM, int WM>
__global__ __launch_bounds__(kThreads, 2) void tiled_kernel(const F8MatmulArgs a) {
  typedef Shape<BM, WM> S;
  constexpr int kMT = S::kMT, kNT = S::kNT;
  __shared__ __attribute__((aligned(1024))) uint8_t stage[S::kStages][S::kStage];
  __shared__ Item items[kMaxItems];
  __shared__ int first_row[kMaxExperts + 1], first_tile[kMaxExperts + 1];
  __shared__ float most[S::kWN][BM];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int q = lane >> 4, r = lane & 15;
  const int I = a.N / 2;

  if constexpr (!kGateUp) {
    if (a.out_dtype == MOE355_F32)
      zero_rest<float, kThreads>(a);
    else
      zero_rest<f16, kThreads>(a);  // zeros of both 16-bit types
  }
  for (int e = threadIdx.x; e <= a.E; e += kThreads) first_row[e] = group_start(a, e);
  __syncthreads();
  if (wave == 0)
    wave_scan(a.E, lane, [&](int e) { return (max(first_row[e + 1] - first_row[e], 0) + BM - 1) / BM; },
              first_tile);
  __syncthreads();

  // This workgroup's items: one of every gridDim.x, the workgroups of an XCD taking
  // neighbouring ones, each time some further, so that a matrix of one full and one partial
  // tile does not give one workgroup all full ones. The token tiles of a matrix vary
  // fastest, so that neighbours share its weights.
  constexpr int kShift = 15;
  const int nw = kGateUp ? f8_blocks(I) : (a.N + kBN - 1) / kBN;
  const int total = first_tile[a.E] * nw;
  const int G = gridDim.x, pid = blockIdx.x;
  const int rounds = min(total / G, kMaxItems - 1), tail = min(total - rounds * G, G);
  const int n_items = rounds + (pid < tail ? 1 : 0);
  if (n_items == 0) return;
  if (wave == 0 && lane < n_items) {
    const int n = lane < rounds ? G : tail;
    const int L = lane * G + (xcd_remap(pid, n) + kShift * lane) % n;
    int lo = 0, hi = a.E - 1;  // the last matrix whose items start at or before L
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_tile[mid] * nw <= L) lo = mid; else hi = mid - 1;
    }
    const int begin = first_row[lo], rows = first_row[lo + 1] - begin;
    const int tiles = first_tile[lo + 1] - first_tile[lo];
    // the matrix's rows are shared evenly by its tiles
    const int height = ((rows + tiles - 1) / tiles + 16 * WM - 1) / (16 * WM) * (16 * WM);
    const int at = L - first_tile[lo] * nw, wt = at / tiles;
    const int row0 = begin + (at - wt * tiles) * height;
    items[lane] = Item{lo, row0, min(row0 + height, begin + rows), wt};
  }
  __syncthreads();
  auto item_at = [&](int j) {
    const Item* p = &items[j];
    return Item{__builtin_amdgcn_readfirstlane(p->e), __builtin_amdgcn_readfirstlane(p->row0),
                __builtin_amdgcn_readfirstlane(p->row_end), __builtin_amdgcn_readfirstlane(p->wt)};
  };
  const int steps = a.Kp / kF8Block;

  // Token rows whose codes (kTokLoads of them) and scales this lane loads, as rows of x; -1
  // past the tile's last row.
  const int tok64 = wave % (BM / 64);  // 64 tokens whose scales this wave loads
  int src[S::kTokLoads + 1];
  auto load_rows = [&](const Item& it) {
#pragma unroll
    for (int i = 0; i <= S::kTokLoads; ++i) {
      const int row = i < S::kTokLoads ? 8 * (wave * S::kTokLoads + i) + (lane >> 3) : 64 * tok64 + lane;
      const int p = it.row0 + row;
      src[i] = p >= it.row_end ? -1 : a.row_src ? a.row_src[p] : row;
    }
  };

  // The item whose steps are being loaded: sources, and this lane's offsets. Where rows are not
  // gathered they are counted from the tile's first, so that offsets stay small.
  __amdgpu_buffer_rsrc_t xsrc, xssrc, wsrc;
  uint32_t xoff[S::kTokLoads], woff[S::kWgtLoads], soff;
  int load_item = 0, load_step = 0, loaded = 0;  // loaded: steps of all items
  auto begin_loads = [&](const Item& it) {
    const size_t first = a.row_src ? 0 : it.row0;
    xsrc = pipe::lds_rsrc(a.x + first * a.Kp);
    xssrc = pipe::lds_rsrc(a.x_scales + first * steps);
    wsrc = pipe::lds_rsrc(a.w + static_cast<size_t>(it.e) * a.N * a.Kp);
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i) {
      const int row = 8 * (wave * S::kTokLoads + i) + (lane >> 3);
      xoff[i] = src[i] < 0 ? pipe::kPadOffset  // out of range: zeros
                           : static_cast<uint32_t>(src[i]) * a.Kp + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < S::kWgtLoads; ++i) {
      const int row = 8 * (wave * S::kWgtLoads + i) + (lane >> 3);  // of the tile
      int n;
      bool in;
      if constexpr (kGateUp) {
        const int wn = row / (16 * kNT), g = row / 16 % kNT;
        const int f = it.wt * kF8Block + wn * 8 * kNT + g % (kNT / 2) * 16 + row % 16;
        in = f < I;
        n = f + (g < kNT / 2 ? 0 : I);
      } else {
        n = it.wt * kBN + row;
        in = n < a.N;
      }
      woff[i] = in ? static_cast<uint32_t>(n) * a.Kp + (((lane & 7) ^ ((row >> 1) & 7)) << 4)
                   : pipe::kPadOffset;
    }
    soff = src[S::kTokLoads] < 0 ? pipe::kPadOffset : static_cast<uint32_t>(src[S::kTokLoads]) * steps * 4;
    load_step = 0;
    if (load_item + 1 < n_items) load_rows(item_at(load_item + 1));
  };
  // Loads the next step of the stream, if there is one.
  auto load = [&]() {
    if (load_item >= n_items) return;
    uint8_t* s = stage[loaded % S::kStages];
    const int k = load_step;
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i)
      pipe::dma16_rsrc(xsrc, xoff[i], k * kF8Block, s + (wave * S::kTokLoads + i) * 1024);
#pragma unroll
    for (int i = 0; i < S::kWgtLoads; ++i)
      pipe::dma16_rsrc(wsrc, woff[i], k * kF8Block, s + S::kTokBytes + (wave * S::kWgtLoads + i) * 1024);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        xssrc, (pipe::lds_void*)(s + S::kTokBytes + S::kWgtBytes + tok64 * 256), 4, soff, k * 4, 0, 0);
    ++loaded;
    if (++load_step == steps && ++load_item < n_items) begin_loads(item_at(load_item));
  };
  // Waits until this wave's loads of step `step` of the stream have landed; of the steps after
  // it kStages - 2 may be in flight (fewer at the end of the stream, where it waits for
  // all).
  auto landed = [&](int step) {
    if (loaded >= step + S::kStages - 1)
      pipe::wait_vmcnt<(S::kStages - 2) * S::kLoads>();
    else
      pipe::wait_vmcnt<0>();
  };
  auto barrier = [&]() {
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
  int done = 0;  // steps of the stream
  const int wm = wave % WM, wn = wave / WM;  // this wave's tokens and weight rows
  for (int j = 0; j < n_items; ++j) {
    const Item it = item_at(j);
    // scales of this wave's weight rows: of gate (all of a product) and of up
    const int n_blocks = kGateUp ? 2 * f8_blocks(I) : f8_blocks(a.N);
    const int block = kGateUp ? it.wt : min((it.wt * kBN + wn * 16 * kNT) / kF8Block, n_blocks - 1);
    const const_f32* ws0 = (const const_f32*)(a.w_scales + (static_cast<size_t>(it.e) * n_blocks + block) * steps);
    const const_f32* ws1 = ws0 + (kGateUp ? static_cast<size_t>(f8_blocks(I)) * steps : 0);
    f32x4 acc[kMT][kNT];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int g = 0; g < kNT; ++g) acc[m][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    // A wave has every WM-th 16 rows of the tile, so that the waves share the rows of one that
    // is not full; mt of its kMT hold any.
    const int mt = min((it.row_end - it.row0 + 16 * (WM - 1 - wm) + 15) / (16 * WM), kMT);
    // One instance per count: mma_f8 needs straight-line code.
    auto run_steps = [&](auto count) {
      constexpr int kM = decltype(count)::value;
      for (int st = 0; st < steps; ++st, ++done) {
        // Every wave has read step `done` - 1, whose buffer is filled again, and has seen its
        // loads of step `done` land.
        landed(done);
        pipe::wait_lgkm0();
        barrier();
        load();
        const float s0 = ws0[st], s1 = kGateUp ? ws1[st] : 0.f;
        const uint8_t* s = stage[done % S::kStages];
        const uint8_t* wtile = s + S::kTokBytes + (wn * kNT * 16 + r) * kF8Block;
        const uint8_t* ts = s + S::kTokBytes + S::kWgtBytes + (16 * wm + r) * 4;
        const int sw = (r >> 1) & 7;  // rows of a tile start at multiples of 16
        u32x4 x[kM + 1][2];
        float sg[kM + 1], su[kM + 1];
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          const uint8_t* p = s + (16 * (wm + WM * m) + r) * kF8Block;
          x[m][0] = *reinterpret_cast<const u32x4*>(p + ((q ^ sw) << 4));
          x[m][1] = *reinterpret_cast<const u32x4*>(p + (((4 + q) ^ sw) << 4));
          const float xs = *reinterpret_cast<const float*>(ts + 64 * WM * m);
          sg[m] = xs * s0;
          su[m] = xs * s1;
        }
#pragma unroll
        for (int g = 0; g < (kM ? kNT : 0); ++g) {
          u32x4 w[2];
          const uint8_t* p = wtile + g * 16 * kF8Block;
          w[0] = *reinterpret_cast<const u32x4*>(p + ((q ^ sw) << 4));
          w[1] = *reinterpret_cast<const u32x4*>(p + (((4 + q) ^ sw) << 4));
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            const f32x4 v = mma_f8(w, x[m]);
            const float f = kGateUp && g >= kNT / 2 ? su[m] : sg[m];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][g][i] = fmaf(v[i], f, acc[m][g][i]);
          }
        }
      }
    };
    switch (mt) {
      case 0: run_steps(std::integral_constant<int, 0>()); break;
      case 1: run_steps(std::integral_constant<int, 1>()); break;
      case 2: run_steps(std::integral_constant<int, (kMT < 2 ? kMT : 2)>()); break;
      case 3: run_steps(std::integral_constant<int, (kMT < 3 ? kMT : 3)>()); break;
      default: run_steps(std::integral_constant<int, kMT>()); break;
    }

    const int n_rows = it.row_end - it.row0, row1 = 16 * wm + r;
    if constexpr (kGateUp) {
      constexpr int kHalf = kNT / 2;
      const int f0 = it.wt * kF8Block + wn * 16 * kHalf + 4 * q;  // this lane's first feature
      const size_t Ip = f8_pad(I);
      // gate's place takes the activation
      float amax[kMT];
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        amax[m] = 0.f;
#pragma unroll
        for (int g = 0; g < kHalf; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float h =
                f0 + 16 * g + i < I ? gate_act_fast(a.act, acc[m][g][i]) * acc[m][g + kHalf][i] : 0.f;
            acc[m][g][i] = h;
            amax[m] = fmaxf(amax[m], f8_finite_abs(h));
          }
        amax[m] = fmaxf(amax[m], __shfl_xor(amax[m], 16, kWave));
        amax[m] = fmaxf(amax[m], __shfl_xor(amax[m], 32, kWave));
        if (q == 0) most[wn][row1 + 16 * WM * m] = amax[m];
      }
      pipe::wait_lgkm0();
      barrier();
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        const int row = row1 + 16 * WM * m;
        if (row >= n_rows) continue;
#pragma unroll
        for (int w = 0; w < S::kWN; ++w) amax[m] = fmaxf(amax[m], most[w][row]);
        const F8Div d = f8_div(amax[m]);
        uint8_t* out = a.out_codes + static_cast<size_t>(it.row0 + row) * Ip + f0;
#pragma unroll
        for (int g = 0; g < kHalf; ++g) {
          const float h[4] = {acc[m][g][0], acc[m][g][1], acc[m][g][2], acc[m][g][3]};
          *reinterpret_cast<uint32_t*>(out + 16 * g) = f8_codes4(h, d);
        }
        if (wn == 0 && q == 0)
          a.out_scales[static_cast<size_t>(it.row0 + row) * (Ip / kF8Block) + it.wt] = d.scale;
      }
      // `most` is written again by the next item's epilogue, behind a barrier of its steps
    } else {
      auto store = [&](auto type) {
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          const int row = row1 + 16 * WM * m;
          if (row >= n_rows) continue;
#pragma unroll
          for (int g = 0; g < kNT; ++g)
            store_results<decltype(type)>(a, it.row0 + row, it.wt * kBN + (wn * kNT + g) * 16 + 4 * q,
                                          acc[m][g]);
        }
      };
      if (a.out_dtype == MOE355_F32) store(float());
      else if (a.out_dtype == MOE355_BF16) store(bf16());
      else store(f16());
    }
  }
}

template <bool kGateUp, int BM, int WM>
hipError_t launch(const F8MatmulArgs& a, hipStream_t s) {
  const long long nw = kGateUp ? f8_blocks(a.N / 2) : (a.N + kBN - 1) / kBN;
  // at most: every matrix that has rows has a tile that is not full
  const long long tiles = a.offsets ? a.M / BM + (a.E < a.M ? a.E : a.M) : (a.M + BM - 1) / BM;
  const long long total = tiles * nw;
  if (total > INT_MAX) return hipErrorInvalidValue;
  long long grid = device_cu_count();
  // the items of a workgroup have kMaxItems - 1 full rounds at most
  const long long most = grid * (kMaxItems - 1);
  grid = total < grid ? total : grid * ((total + most - 1) / most);
  tiled_kernel<kGateUp, BM, WM><<<dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_f8_tiled(const F8MatmulArgs& a, bool gate_up, int tile_rows, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  if (tile_rows == 256) return gate_up ? launch<true, 256, 4>(a, s) : launch<false, 256, 4>(a, s);
  return gate_up ? launch<true, 64, 2>(a, s) : launch<false, 64, 2>(a, s);
}

}  // namespace moe355
