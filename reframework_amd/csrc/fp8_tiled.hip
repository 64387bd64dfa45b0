// Grouped product of 8-bit rows and 8-bit weights (formats: fp8.h) for many rows per matrix:
// an item multiplies BM token rows by 256 weight rows (gate_up: gate and up of 128
// features, a block of the result's scales), a step of 128 columns at a time.
//
// Tokens go straight to LDS, rows by 128 bytes a step, with their 16-byte chunks XORed by half
// the row number, which leaves the fragment reads without bank conflicts. Weight tiles go to LDS
// as they are laid out where 256 rows share them (turns_kernel, bound by the matrix cores), and
// to the registers of the one wave that needs them up to 128 rows (rows_kernel, bound by the
// weights' stream). A step is one block of both operands' scales, so the matrix core sums it from
// zero and the sum is scaled and added in fp32 by the vector unit, whose instructions run beside
// the next products. Token scales go to LDS with the rows; the weights' one (gate_up: two) of a
// wave and step is a scalar load.
//
// A workgroup of turns_kernel runs several items, whose steps follow each other in one stream of
// loads: the first steps of an item are on their way while the item before it is multiplied and
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
  static constexpr int kStage = kTokBytes + kWgtBytes + (BM < 64 ? 64 : BM) * 4;
  static constexpr int kPartTile = kMT * kNT * kThreads * 4;  // floats of a part's sums
  static constexpr int kSpare = kMaxItems * 32 + (kMaxExperts + 1) * 8 + kWN * BM * 4 + 64;
  static constexpr int kStages = (160 * 1024 - kSpare) / kStage;
  // direct-to-LDS loads of a wave per step: 1 KB of codes each, and 256 bytes of scales
  // (some waves' a second time)
  static constexpr int kTokPieces = BM / 8;  // of 8 rows, 1 KB
  static constexpr int kTokLoads = (kTokPieces + kWaves - 1) / kWaves;
  static constexpr int kWgtLoads = kWgtBytes / 1024 / kWaves;
  static constexpr int kLoads = kTokLoads + kWgtLoads + 1;
  static_assert(kMT >= 1 && kNT >= 2 && kTokLoads >= 1, "tiles of a wave");
  static_assert(kStages >= 2 && (kStages - 1) * kLoads < 64, "pipeline");
};

// Weight tile `wt` of the token rows [row0, row_end) of matrix e, steps [k0, k1). part: where its
// sums go where they are only some of the steps, else -1.
struct Item {
  int e, row0, row_end, wt, k0, k1, part;
};

__device__ __forceinline__ Item uniform(const Item* p) {
  return Item{__builtin_amdgcn_readfirstlane(p->e),  __builtin_amdgcn_readfirstlane(p->row0),
              __builtin_amdgcn_readfirstlane(p->row_end), __builtin_amdgcn_readfirstlane(p->wt),
              __builtin_amdgcn_readfirstlane(p->k0), __builtin_amdgcn_readfirstlane(p->k1),
              __builtin_amdgcn_readfirstlane(p->part)};
}

// The items of a launch of G workgroups: `rounds` of one per workgroup, and `tail` more. Run as
// they are those would take a whole item's time on some of the CUs; cut into `split` parts of
// the steps each they take a part of it on all, and a second launch adds the parts and stores.
struct Rounds {
  int rounds, tail, split;
};

// What a cut saves and costs, in steps of an item: a part's sums go to memory and back, all
// workgroups' at once (256 rows: 0.5 MB per unit at 5 TB/s, against 2 us a step), and the
// second launch takes 4 us.
template <int BM>
__device__ __forceinline__ Rounds plan_rounds(int total, int G, int steps, int max_parts) {
  Rounds p{min(total / G, kMaxItems - 1), 0, 1};
  p.tail = min(total - p.rounds * G, G);
  const int cap = min(max_parts, G);
  int best = 40 * steps;
  for (int s = 2; s <= 16 && s * p.tail <= cap && steps >= 4 * s; s *= 2) {
    const int cost = (40 * steps + s - 1) / s + 80 + 2 * s * p.tail;
    if (cost < best) {
      best = cost;
      p.split = s;
    }
  }
  return p;
}

// The matrices' first rows and tiles (the last entries: the ends).
template <int BM>
__device__ __forceinline__ void list_tiles(const F8MatmulArgs& a, int* first_row, int* first_tile) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int e = threadIdx.x; e <= a.E; e += kThreads) first_row[e] = group_start(a, e);
  __syncthreads();
  if (threadIdx.x < kWave)
    wave_scan(a.E, lane, [&](int e) { return (max(first_row[e + 1] - first_row[e], 0) + BM - 1) / BM; },
              first_tile);
  __syncthreads();
}

// Item L of all. The token tiles of a matrix vary fastest, so that neighbours share its
// weights.
template <int BM, int WM>
__device__ __forceinline__ Item decode_item(const F8MatmulArgs& a, int nw, const int* first_row,
                                            const int* first_tile, int L) {
  int lo = 0, hi = a.E - 1;  // the last matrix whose items start at or before L
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_tile[mid] * nw <= L) lo = mid; else hi = mid - 1;
  }
  const int begin = first_row[lo], rows = first_row[lo + 1] - begin;
  const int tiles = first_tile[lo + 1] - first_tile[lo];
  // the matrix's rows are shared evenly by its tiles, in whole 16 rows of the waves of a turn
  constexpr int kStep = 16 * WM / 2;
  const int height = ((rows + tiles - 1) / tiles + kStep - 1) / kStep * kStep;
  const int at = L - first_tile[lo] * nw, wt = at / tiles;
  const int row0 = begin + (at - wt * tiles) * height;
  return Item{lo, row0, min(row0 + height, begin + rows), wt, 0, a.Kp / kF8Block, -1};
}

// Writes this workgroup's items and returns how many there are: one of every gridDim.x, the
// workgroups of an XCD taking neighbouring ones, each time some further, so that a matrix of
// one full and one partial tile does not give one workgroup all full ones.
template <int BM, int WM>
__device__ __forceinline__ int list_items(const F8MatmulArgs& a, int nw, Item* items) {
  constexpr int kShift = 15;
  __shared__ int first_row[kMaxExperts + 1], first_tile[kMaxExperts + 1];
  list_tiles<BM>(a, first_row, first_tile);
  const int G = gridDim.x, pid = blockIdx.x, lane = threadIdx.x, steps = a.Kp / kF8Block;
  const Rounds p = plan_rounds<BM>(first_tile[a.E] * nw, G, steps, a.max_parts);
  const int units = p.tail * p.split;
  const int n_items = p.rounds + (pid < units ? 1 : 0);
  if (lane < n_items) {
    const bool full = lane < p.rounds;
    const int n = full ? G : units;
    const int u = (xcd_remap(pid, n) + kShift * lane) % n;
    Item it = decode_item<BM, WM>(a, nw, first_row, first_tile, lane * G + (full ? u : u / p.split));
    if (!full && p.split > 1) {
      const int part = u % p.split;
      it.k0 = part * steps / p.split;
      it.k1 = (part + 1) * steps / p.split;
      it.part = u;
    }
    items[lane] = it;
  }
  __syncthreads();
  return n_items;
}

// What a wave loads of the stream of its workgroup's steps.
template <bool kGateUp, int BM, int WM>
struct Loader {
  typedef Shape<BM, WM> S;
  const F8MatmulArgs& a;
  const Item* items;
  const int n_items, steps, wave;
  // The item whose steps are being loaded: sources, and this lane's offsets.
  __amdgpu_buffer_rsrc_t xsrc, xssrc, wsrc;
  uint32_t xoff[S::kTokLoads], cell[2], soff;
  // Token rows of the next item whose codes and scales this lane loads, as rows of x; -1 past
  // the tile's last row. (gate_up reads them under branches, where the compiler waits for all
  // loads in flight: once an item.)
  int src[S::kTokLoads + 1];
  int item = 0, step = 0, end = 0, loaded = 0;  // loaded: steps of all items

  __device__ __forceinline__ Loader(const F8MatmulArgs& args, const Item* list, int n, int w)
      : a(args), items(list), n_items(n), steps(args.Kp / kF8Block), wave(w) {
    load_rows(uniform(items));
    begin(uniform(items));
  }
  // 64 tokens whose scales this wave loads
  __device__ __forceinline__ int tok64() const { return BM <= 64 ? 0 : wave % (BM / 64); }
  // Piece of the tokens that load i brings (some waves' a second time where there are few).
  __device__ __forceinline__ int piece(int i) const { return wave * S::kTokLoads + i; }
  // The lane, opaque: what follows from it is computed where an item begins, not kept.
  static __device__ __forceinline__ int lane_id() { return pipe::opaque(threadIdx.x & (kWave - 1)); }
  static __device__ __forceinline__ uint32_t lane16() { return (threadIdx.x & (kWave - 1)) * 16; }
  __device__ __forceinline__ void load_rows(const Item& it) {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i <= S::kTokLoads; ++i) {
      const int row = i < S::kTokLoads ? 8 * piece(i) + (lane >> 3) : 64 * tok64() + lane;
      const int p = it.row0 + row;
      src[i] = p >= it.row_end ? -1 : a.row_src ? a.row_src[p] : row;
    }
  }
  // Chunk of a row (modulo 8) that a lane loads.
  static __device__ __forceinline__ int chunk(int lane, int row) { return ((lane & 7) ^ ((row >> 1) & 7)) << 4; }
  __device__ __forceinline__ void begin(const Item& it) {
    const int lane = lane_id();
    // Rows that are not gathered are counted from the tile's first, so that offsets stay small.
    const size_t first = a.row_src ? 0 : it.row0;
    xsrc = pipe::lds_rsrc(a.x + first * a.Kp);
    xssrc = pipe::lds_rsrc(a.x_scales + first * steps);
    wsrc = pipe::lds_rsrc(a.w + static_cast<size_t>(it.e) * f8_cell_rows(a.N, kGateUp) * steps * kF8Cell);
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i) {
      const int row = 8 * piece(i) + (lane >> 3);
      xoff[i] = src[i] < 0 ? pipe::kPadOffset  // out of range: zeros
                           : static_cast<uint32_t>(src[i]) * a.Kp + chunk(lane, row);
    }
    // Cells past the last of a matrix are out of range: zeros.
    const int cell_rows = f8_cell_rows(a.N, kGateUp);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int block = kGateUp ? it.wt + i * (cell_rows / 2) : it.wt * 2 + i;
      cell[i] = block < cell_rows ? static_cast<uint32_t>(block) * steps * kF8Cell : pipe::kPadOffset;
    }
    soff = src[S::kTokLoads] < 0 ? pipe::kPadOffset : static_cast<uint32_t>(src[S::kTokLoads]) * steps * 4;
    step = it.k0;
    end = it.k1;
    if (item + 1 < n_items) load_rows(uniform(items + item + 1));
  }
  // The 2 KB tile of its cell that loads i, i ^ 1 bring, and its place in LDS, where a wave's
  // tiles follow each other: loads of the first half bring the first half of every wave's
  // (gate_up: gate's; up's are the second).
  struct Piece {
    int cell, tile, at;
  };
  __device__ __forceinline__ Piece piece_of(int wave, int i) const {
    constexpr int kHalf = S::kWgtLoads / 4;  // tiles of this wave and half
    const int half = i / (2 * kHalf), n = wave * kHalf + i / 2 % kHalf;  // of 8
    const int wn = n / (S::kNT / 2), g = n % (S::kNT / 2);
    const int at = wn * S::kNT + half * (S::kNT / 2) + g;
    return kGateUp ? Piece{half, n, at} : Piece{at / 8, at % 8, at};
  }
  __device__ __forceinline__ bool more() const { return item < n_items; }
  // The wave's number, opaque like the lane: places in LDS are computed again rather than kept
  // in scalar registers, which are few (kept, they were moved to vector lanes and back every
  // step).
  __device__ __forceinline__ int wave_id() const {
    int w = wave;
    asm volatile("" : "+s"(w));
    return w;
  }
  __device__ __forceinline__ void load_tokens(uint8_t* s) const {
    uint8_t* to = s + wave_id() * S::kTokLoads * 1024;
#pragma unroll
    for (int i = 0; i < S::kTokLoads; ++i)
      pipe::dma16_rsrc(xsrc, xoff[i], step * kF8Block, to + i * 1024);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        xssrc, (pipe::lds_void*)(s + S::kTokBytes + S::kWgtBytes + tok64() * 256), 4, soff, step * 4, 0, 0);
  }
  template <int kHalf>
  __device__ __forceinline__ void load_weights(uint8_t* s) const {
    const int w = wave_id();
#pragma unroll
    for (int i = kHalf * (S::kWgtLoads / 2); i < (kHalf + 1) * (S::kWgtLoads / 2); ++i) {
      const Piece p = piece_of(w, i);
      const int part = i % 2 * (kF8Tile / 2);
      pipe::dma16_rsrc(wsrc, (p.cell ? cell[1] : cell[0]) + lane16(), step * kF8Cell + p.tile * kF8Tile + part,
                       s + S::kTokBytes + p.at * kF8Tile + part);
    }
  }
  __device__ __forceinline__ void next() {
    ++loaded;
    if (++step == end && ++item < n_items) begin(uniform(items + item));
  }
};

// All waves; nothing moves across it.
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_sched_barrier(0);
}

// n products and the scaled sums of their results, product(i) and add(i, its result), each result
// added behind the third product after it (kMostAhead): it is there by then (12 wait states),
// without waits between the products. Left to itself the compiler waits for every result: 10 % slower.
template <int n, int kMostAhead, typename P, typename A>
__device__ __forceinline__ void interleaved(P product, A add) {
  constexpr int kAhead = n < kMostAhead ? n : kMostAhead;
  f32x4 v[kAhead + 1];
#pragma unroll
  for (int i = 0; i < n + kAhead; ++i) {
    if (i < n) v[i % (kAhead + 1)] = product(i);
    __builtin_amdgcn_sched_barrier(0);
    if (i >= kAhead) add(i - kAhead, v[(i - kAhead) % (kAhead + 1)]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// f(mt as a compile-time constant, 1 rounded up to kLeast and those above 4 to even ones), mt in
// [0, kMost].
template <int kMost, int kLeast = 1, typename F>
__device__ __forceinline__ void by_count(int mt, F f) {
  if constexpr (kMost > 4) {
    if (mt > kMost - 2)
      f(std::integral_constant<int, kMost>());
    else
      by_count<kMost - 2, kLeast>(mt, f);
  } else {
    switch (mt) {
      case 0: f(std::integral_constant<int, 0>()); break;
      case 1: f(std::integral_constant<int, kLeast>()); break;
      case 2: f(std::integral_constant<int, (kMost < 2 ? kMost : 2)>()); break;
      case 3: f(std::integral_constant<int, (kMost < 3 ? kMost : 3)>()); break;
      default: f(std::integral_constant<int, kMost>()); break;
    }
  }
}

// Scales of the weight rows of a wave in an item, by step: of gate (all of a product), of up.
template <bool kGateUp, typename S>
__device__ __forceinline__ void weight_scales(const F8MatmulArgs& a, const Item& it, int wn,
                                              const const_f32** gate, const const_f32** up) {
  const int I = a.N / 2, steps = a.Kp / kF8Block;
  const int n_blocks = kGateUp ? 2 * f8_blocks(I) : f8_blocks(a.N);
  const int block = kGateUp ? it.wt : min((it.wt * kBN + wn * 16 * S::kNT) / kF8Block, n_blocks - 1);
  *gate = (const const_f32*)(a.w_scales + (static_cast<size_t>(it.e) * n_blocks + block) * steps);
  *up = *gate + (kGateUp ? static_cast<size_t>(f8_blocks(I)) * steps : 0);
}

// The epilogues take kM of a wave's kMT tile rows, from m0 on.
// gate_up's, first part: gate's place takes act(gate) * up; the largest of each token's
// features in this wave goes to `most` [waves over weights][BM]. The result goes to 8 bits, so the
// hardware's sigmoid (off by 3e-7) does in every type.
template <typename S, int BM, int WM, int kM>
__device__ __forceinline__ void activate(const F8MatmulArgs& a, const Item& it, f32x4 (&acc)[kM][S::kNT],
                                         int wm, int wn, int m0, float (*most)[BM]) {
  constexpr int kHalf = S::kNT / 2;
  const int lane = pipe::opaque(threadIdx.x & (kWave - 1)), q = lane >> 4, r = lane & 15;
  const int f0 = it.wt * kF8Block + wn * 16 * kHalf + 4 * q, I = a.N / 2;
  by_activation(a.act, [&](auto act) {
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      float amax = 0.f;
#pragma unroll
      for (int g = 0; g < kHalf; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float h =
              f0 + 16 * g + i < I ? gate_act_fast(act.value, acc[m][g][i]) * acc[m][g + kHalf][i] : 0.f;
          acc[m][g][i] = h;
          amax = fmaxf(amax, f8_finite_abs(h));
        }
      amax = row_max(amax);
      if (q == 0) most[wn][16 * (wm + WM * (m0 + m)) + r] = amax;
    }
  });
}

// The second part, behind a barrier: the codes and scales.
template <typename S, int BM, int WM, int kM>
__device__ __forceinline__ void store_codes(const F8MatmulArgs& a, const Item& it,
                                            const f32x4 (&acc)[kM][S::kNT], int wm, int wn, int m0,
                                            const float (*most)[BM]) {
  constexpr int kHalf = S::kNT / 2;
  const int lane = pipe::opaque(threadIdx.x & (kWave - 1)), q = lane >> 4, r = lane & 15;
  const int f0 = it.wt * kF8Block + wn * 16 * kHalf + 4 * q;
  const size_t Ip = f8_pad(a.N / 2);
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    const int row = 16 * (wm + WM * (m0 + m)) + r;
    if (row >= it.row_end - it.row0) continue;
    float amax = most[0][row];
#pragma unroll
    for (int w = 1; w < S::kWN; ++w) amax = fmaxf(amax, most[w][row]);
    const F8Div d = f8_div(amax);
    uint8_t* out = a.out_codes + static_cast<size_t>(it.row0 + row) * Ip + f0;
#pragma unroll
    for (int g = 0; g < kHalf; ++g) {
      const float h[4] = {acc[m][g][0], acc[m][g][1], acc[m][g][2], acc[m][g][3]};
      *reinterpret_cast<uint32_t*>(out + 16 * g) = f8_codes4(h, d);
    }
    if (wn == 0 && q == 0)
      a.out_scales[static_cast<size_t>(it.row0 + row) * (Ip / kF8Block) + it.wt] = d.scale;
  }
}

typedef unsigned short u16;

// Four results rounded to a 16-bit type.
template <typename T>
__device__ __forceinline__ u32x2 pack4(f32x4 v) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, T4{from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])});
}

// Two tiles' values of 16 bits, from column n on. They are exchanged between the lanes of a row,
// so that each stores 16 bytes and a row gets 64 consecutive ones.
template <typename T>
__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t out, uint32_t at, int n, int N, int q, f32x4 v0,
                                        f32x4 v1) {
  const u32x2 u = pack4<T>(v0), w = pack4<T>(v1);
  const auto lo = __builtin_amdgcn_permlane16_swap(u[0], w[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(u[1], w[1], false, false);
  n += 16 * (q & 1) + 8 * (q >> 1);
  __builtin_amdgcn_raw_buffer_store_b128(u32x4{lo[0], hi[0], lo[1], hi[1]}, out,
                                         n < N ? at + n * 2 : pipe::kPadOffset, 0, 0);
}

// A product's epilogue. Stored relative to the tile's first row; an offset out of range stores
// nothing, so that there are no branches per element.
template <typename S, int WM, typename OutT, int kM>
__device__ __forceinline__ void store_rows(const F8MatmulArgs& a, const Item& it,
                                           const f32x4 (&acc)[kM][S::kNT], int wm, int wn, int m0) {
  const int lane = pipe::opaque(threadIdx.x & (kWave - 1)), q = lane >> 4, r = lane & 15;
  constexpr int kSize = sizeof(OutT);
  const auto out = pipe::lds_rsrc(static_cast<OutT*>(a.out) + static_cast<size_t>(it.row0) * a.N);
  const int n_rows = it.row_end - it.row0;
  const int n0 = it.wt * kBN + wn * S::kNT * 16;  // this wave's first column
  if constexpr (std::is_same<OutT, Scaled16>::value) {  // N is a multiple of 16
    static_assert(S::kNT % 4 == 0 && kScaled16Block == 64, "four tiles a scale");
    const int blocks = (a.N + kScaled16Block - 1) / kScaled16Block;
    const auto scales = pipe::lds_rsrc(a.slot_scales + static_cast<size_t>(it.row0) * blocks);
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const int row = 16 * (wm + WM * (m0 + m)) + r;
      const uint32_t at = row < n_rows ? row * a.N * kSize : pipe::kPadOffset;
#pragma unroll
      for (int b = 0; b < S::kNT; b += 4) {
        float amax = 0.f;
#pragma unroll
        for (int g = b; g < b + 4; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = fmaxf(amax, f8_finite_abs(acc[m][g][i]));
        amax = fmaxf(amax, __shfl_xor(amax, 16, kWave));
        amax = fmaxf(amax, __shfl_xor(amax, 32, kWave));
        const int byte = scaled16_byte(__float_as_uint(amax));
        const float f = scaled16_factor(byte);
#pragma unroll
        for (int g = b; g < b + 4; g += 2) store16<f16>(out, at, n0 + 16 * g, a.N, q, acc[m][g] * f, acc[m][g + 1] * f);
        const int n = n0 + 16 * b;
        __builtin_amdgcn_raw_buffer_store_b8(
            static_cast<uint8_t>(byte), scales,
            q == 0 && row < n_rows && n < a.N ? row * blocks + n / kScaled16Block : pipe::kPadOffset, 0, 0);
      }
    }
    return;
  } else if (a.N % 8 == 0) {
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const int row = 16 * (wm + WM * (m0 + m)) + r;
      const uint32_t at = row < n_rows ? row * a.N * kSize : pipe::kPadOffset;
#pragma unroll
      for (int g = 0; g < S::kNT; g += kSize == 4 ? 1 : 2) {
        if constexpr (kSize == 4) {
          const int n = n0 + 16 * g + 4 * q;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[m][g]), out,
                                                 n < a.N ? at + n * kSize : pipe::kPadOffset, 0, 0);
        } else {
          store16<OutT>(out, at, n0 + 16 * g, a.N, q, acc[m][g], acc[m][g + 1]);
        }
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const int row = 16 * (wm + WM * (m0 + m)) + r;
      const uint32_t at = row < n_rows ? row * a.N * kSize : pipe::kPadOffset;
#pragma unroll
      for (int g = 0; g < S::kNT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + 16 * g + 4 * q + i;
          const uint32_t off = n < a.N ? at + n * kSize : pipe::kPadOffset;
          const OutT v = from_f32<OutT>(acc[m][g][i]);
          if constexpr (kSize == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), out, off, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(u16, v), out, off, 0, 0);
        }
    }
  }
}

// Sums of some of an item's steps, as they lie in the lanes.
template <typename S>
__device__ __forceinline__ f32x4* part_at(const F8MatmulArgs& a, int part, int m) {
  return reinterpret_cast<f32x4*>(a.parts + static_cast<size_t>(part) * S::kPartTile) +
         m * S::kNT * kThreads + threadIdx.x;
}

template <typename S>
__device__ __forceinline__ void store_part(const F8MatmulArgs& a, const Item& it,
                                           const f32x4 (&acc)[S::kMT][S::kNT]) {
#pragma unroll
  for (int m = 0; m < S::kMT; ++m)
#pragma unroll
    for (int g = 0; g < S::kNT; ++g) part_at<S>(a, it.part, m)[g * kThreads] = acc[m][g];
}

// Adds the parts of the items of the last round, in their order, and stores: a workgroup takes
// one tile row of every wave.
template <bool kGateUp, int BM, int WM, typename OutT>
__global__ __launch_bounds__(kThreads) void parts_kernel(const F8MatmulArgs a, int G) {
  typedef Shape<BM, WM> S;
  __shared__ int first_row[kMaxExperts + 1], first_tile[kMaxExperts + 1];
  __shared__ float most[S::kWN][BM];
  list_tiles<BM>(a, first_row, first_tile);
  const int nw = kGateUp ? f8_blocks(a.N / 2) : (a.N + kBN - 1) / kBN;
  const Rounds p = plan_rounds<BM>(first_tile[a.E] * nw, G, a.Kp / kF8Block, a.max_parts);
  const int i = blockIdx.x / S::kMT, m = blockIdx.x % S::kMT;
  if (p.split == 1 || i >= p.tail) return;
  const Item it = decode_item<BM, WM>(a, nw, first_row, first_tile, p.rounds * G + i);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / S::kWN, wn = wave % S::kWN;
  f32x4 acc[1][S::kNT];
#pragma unroll
  for (int g = 0; g < S::kNT; ++g) acc[0][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.split; ++s) {
    const f32x4* part = part_at<S>(a, i * p.split + s, m);
#pragma unroll
    for (int g = 0; g < S::kNT; ++g) acc[0][g] += part[g * kThreads];
  }
  if constexpr (kGateUp) {
    activate<S, BM, WM>(a, it, acc, wm, wn, m, most);
    __syncthreads();
    store_codes<S, BM, WM>(a, it, acc, wm, wn, m, most);
  } else {
    store_rows<S, WM, OutT>(a, it, acc, wm, wn, m);
  }
}

// A row's operand as it lies in LDS, or in bf16.
struct Codes {
  u32x4 v[2];
};
template <typename Row>
__device__ __forceinline__ Row row_of(const u32x4* c) {
  if constexpr (std::is_same<Row, Codes>::value)
    return Codes{{c[0], c[1]}};
  else
    return to_bf16(c);
}
template <typename Row>
__device__ __forceinline__ Row row_of(const uint8_t* lo, const uint8_t* hi) {
  const u32x4 c[2] = {*reinterpret_cast<const u32x4*>(lo), *reinterpret_cast<const u32x4*>(hi)};
  return row_of<Row>(c);
}
__device__ __forceinline__ f32x4 product(const Codes& w, const Codes& x) { return mma_f8(w.v, x.v); }
__device__ __forceinline__ f32x4 product(const Bf16Row& w, const Bf16Row& x) { return mma_f8_exact(w, x); }

// Up to 128 token rows, where the weights' stream counts: a workgroup multiplies BM rows by 256
// weight rows, a wave by 32 of them, whose tiles it alone needs: they go straight to its
// registers, 1 KB a load, asked for while the group of kAhead steps before is multiplied. The
// tokens, which all waves need, go through LDS, a group at a time, so that the waves meet once in
// as many steps. (With the weights in LDS every step waits for all waves: 394 rows of 16 matrices
// of 12800 x 4096 179 us, so 157, 5.35 TB/s of weights. Of 4096 x 6400 93 us, 4.5 TB/s.)
// A group does not overlap the next one's tokens: the compiler, which cannot tell the two buffers
// apart, takes its LDS reads to depend on the loads just asked for and waits for them, and so for
// all weights before them, behind each barrier. Two workgroups share a CU where 128 registers
// do; scaled products of 64 rows do not quite fit there (19 registers spilled, 48 bytes).
// tests/test_token_loads.py holds that enough loads stay behind the tokens' for the wait below.
template <bool kGateUp, int BM, bool kExact, typename OutT>
__global__ __launch_bounds__(kThreads, kExact || BM > 64 ? 2 : 4) void rows_kernel(const F8MatmulArgs a) {
  constexpr int WM = 1, kAhead = kExact || BM > 64 ? 3 : 2;
  typedef Shape<BM, WM> S;
  constexpr int kMT = S::kMT, kNT = S::kNT;
  static_assert(kNT == 2, "a wave's tiles");
  static_assert((BM + 63) / 64 * kAhead <= kWaves, "a wave a piece of the scales");
  constexpr int kPieces = BM / 8;  // of a step's tokens, 8 rows each
  constexpr int kTokLoads = (kPieces * kAhead + kWaves - 1) / kWaves;
  constexpr int kWgtLoads = 2 * kNT;  // of a step
  __shared__ __attribute__((aligned(1024))) uint8_t tokens[2][kAhead][BM * kF8Block];
  constexpr int kScales = (BM + 63) / 64;  // pieces of 64
  __shared__ float scales[2][kAhead][kScales * 64];
  __shared__ float most[S::kWN][BM];
  const int lane = threadIdx.x & (kWave - 1), q = lane >> 4, r = lane & 15, sw = (r >> 1) & 7;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if constexpr (!kGateUp) zero_rest<OutT, kThreads>(a);

  const int cell_rows = f8_cell_rows(a.N, kGateUp), steps = a.Kp / kF8Block;
  const int nw = kGateUp ? cell_rows / 2 : (cell_rows + 1) / 2;
  // The token tiles of a matrix vary fastest and neighbours run on one XCD: they share its weights.
  const int id = xcd_remap(blockIdx.x, gridDim.x), tiles = gridDim.x / nw;
  const RowTile t = find_tile(a, BM, id % tiles);
  if (t.e < 0) return;
  const Item it{t.e, t.row0, t.row_end, id / tiles, 0, steps, -1};
  const int n_rows = it.row_end - it.row0;

  // tokens: rows of a piece, offsets as in Loader
  const size_t first = a.row_src ? 0 : it.row0;
  const auto xsrc = pipe::lds_rsrc(a.x + first * a.Kp);
  const auto xssrc = pipe::lds_rsrc(a.x_scales + first * steps);
  auto source = [&](int row) {
    return row >= n_rows ? -1 : a.row_src ? a.row_src[it.row0 + row] : row;
  };
  // this wave's pieces: of every step where there are as many as waves or more
  constexpr int kRows8 = kPieces > kWaves ? kPieces / kWaves : 1;
  uint32_t xoff[kRows8];
#pragma unroll
  for (int i = 0; i < kRows8; ++i) {
    const int row = (wave + i * kWaves) % kPieces * 8 + (lane >> 3), src = source(row);
    xoff[i] = src < 0 ? pipe::kPadOffset
                      : static_cast<uint32_t>(src) * a.Kp + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  const int s64 = wave % kScales, src64 = source(s64 * 64 + lane);
  const uint32_t soff = src64 < 0 ? pipe::kPadOffset : static_cast<uint32_t>(src64) * steps * 4;
  auto load_tokens = [&](int k0, int buffer) {
#pragma unroll
    for (int i = 0; i < kTokLoads; ++i) {
      // some waves load a step's a second time
      const int u = min((wave + i * kWaves) / kPieces, kAhead - 1), k = min(k0 + u, steps - 1);
      const int piece = (wave + i * kWaves) % kPieces;
      pipe::dma16_rsrc(xsrc, xoff[i % kRows8], k * kF8Block, &tokens[buffer][u][piece * 1024]);
    }
    const int u = wave / kScales % kAhead, k = min(k0 + u, steps - 1);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xssrc, (pipe::lds_void*)(&scales[buffer][u][s64 * 64]), 4, soff, k * 4, 0, 0);
  };

  // this wave's two tiles (gate_up: gate and up of the same features)
  const uint8_t* wp[kNT];
  const const_f32* ws[kNT];
#pragma unroll
  for (int g = 0; g < kNT; ++g) {
    const int block = min(kGateUp ? it.wt + g * (cell_rows / 2) : it.wt * 2 + wave / 4, cell_rows - 1);
    const int tile = kGateUp ? wave : wave % 4 * 2 + g;
    const size_t cells = (static_cast<size_t>(it.e) * cell_rows + block) * steps;
    wp[g] = a.w + cells * kF8Cell + tile * kF8Tile + lane * 16;
    ws[g] = (const const_f32*)(a.w_scales + cells);
  }
  u32x4 w[kAhead][kNT][2];
  // always as many loads, the last step again past it: the waits for the tokens count them
  auto load_weights = [&](int k, u32x4 (*to)[2]) {
    const size_t at = static_cast<size_t>(min(k, steps - 1)) * kF8Cell;
#pragma unroll
    for (int g = 0; g < kNT; ++g) {
      to[g][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[g] + at));
      to[g][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[g] + at + kF8Tile / 2));
    }
  };

  load_tokens(0, 0);
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load_weights(u, w[u]);
  f32x4 acc[kMT][kNT];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int g = 0; g < kNT; ++g) acc[m][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  by_count<kMT>((n_rows + 15) / 16, [&](auto count) {
    constexpr int kM = decltype(count)::value > 0 ? decltype(count)::value : 1;  // a tile has rows
    // n steps from k0 on, straight-line (mma_f8)
    auto run = [&](int k0, int buffer, auto n) {
#pragma unroll
      for (int u = 0; u < decltype(n)::value; ++u) {
        const int k = k0 + u;
        const float s0 = ws[0][k], s1 = ws[1][k];
        typedef typename std::conditional<kExact, Bf16Row, Codes>::type Row;
        const Row w0 = row_of<Row>(w[u][0]), w1 = row_of<Row>(w[u][1]);
        auto read = [&](int m) {
          const uint8_t* p = tokens[buffer][u] + (16 * m + r) * kF8Block;
          return row_of<Row>(p + ((q ^ sw) << 4), p + (((4 + q) ^ sw) << 4));
        };
        // A tile row at a time: its products, the sums of the one before, and the reads of the
        // next.
        f32x4 v[2][kNT];
        Row x = read(0);
#pragma unroll
        for (int m = 0; m <= kM; ++m) {
          if (m < kM) {
            v[m & 1][0] = product(w0, x);
            v[m & 1][1] = product(w1, x);
            if (m + 1 < kM)
              x = read(m + 1);
            else
              load_weights(k + kAhead, w[u]);  // into the registers that are free now
          }
          if (m > 0) {
            const float xs = scales[buffer][u][16 * (m - 1) + r];
#pragma unroll
            for (int g = 0; g < kNT; ++g) {
              const float f = xs * (g ? s1 : s0);
              f32x4& sum = acc[m - 1][g];
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[i] = fmaf(v[(m - 1) & 1][g][i], f, sum[i]);
              asm volatile("" : "+v"(sum));  // added here (mma_f8)
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    auto next_tokens = [&](int k0, int buffer) {
      // Of this wave's loads of these tokens: behind them those of kAhead steps' weights
      pipe::wait_vmcnt<kWgtLoads * kAhead>();
      pipe::wait_lgkm0();
      barrier();  // all have read the tokens before
      load_tokens(k0 + kAhead, buffer ^ 1);
      __builtin_amdgcn_sched_barrier(0);
    };
    int buffer = 0, k0 = 0;
    for (; k0 + kAhead <= steps; k0 += kAhead, buffer ^= 1) {
      next_tokens(k0, buffer);
      run(k0, buffer, std::integral_constant<int, kAhead>());
    }
    if (k0 < steps) {
      next_tokens(k0, buffer);
      static_assert(kAhead <= 4, "what may be left");
      if (kAhead > 3 && steps - k0 == 3)
        run(k0, buffer, std::integral_constant<int, (kAhead > 3 ? 3 : 1)>());
      else if (kAhead > 2 && steps - k0 == 2)
        run(k0, buffer, std::integral_constant<int, 2>());
      else
        run(k0, buffer, std::integral_constant<int, 1>());
    }
  });
  if constexpr (kGateUp) {
    activate<S, BM, WM>(a, it, acc, 0, wave, 0, most);
    __syncthreads();
    store_codes<S, BM, WM>(a, it, acc, 0, wave, 0, most);
  } else {
    store_rows<S, WM, OutT>(a, it, acc, 0, wave, 0);
  }
}

// 256 token rows. Two waves share a SIMD and work in turns, half a step each: while the first
// four waves multiply four of their eight tile columns, the others read the operands of
// theirs from LDS, and a barrier swaps them, so that the matrix cores always have a wave with
// its operands in registers. Reading and multiplying a step between two barriers, all waves read at once
// while the matrix cores wait: 730 us instead of 515 for 8192 rows of 8 matrices of 14336 x
// 4096.
//
// There is room for two steps in LDS. A step's tokens and the first half of its weight tiles
// are read in the first of a step's two reading phases only, so their place is loaded again half a
// step before that of the other half: each load has one and a half steps until it is
// read.
//   phase        4s          4s + 1      4s + 2      4s + 3
//   waves 0-3    read s, 1   mul s, 1    read s, 2   mul s, 2
//   waves 4-7    (mul s-1,2) read s, 1   mul s, 1    read s, 2
// A wave asks for the second half of step s + 1 when it reads the first half of s, and for the
// tokens and first half of s + 2 when it reads the second half of s: both places were read for the
// last time in the phase before. Before a phase that reads a part, every wave has seen its
// own loads of it land: those of at most the two parts asked for after it are in flight.
template <bool kGateUp, typename OutT>
__global__ __launch_bounds__(kThreads, 2) void turns_kernel(const F8MatmulArgs a) {
  constexpr int BM = 256, WM = 4;
  typedef Shape<BM, WM> S;
  constexpr int kMT = S::kMT, kNT = S::kNT, kHalf = kNT / 2;
  static_assert(S::kStages == 2, "room for two steps");
  __shared__ __attribute__((aligned(1024))) uint8_t stage[S::kStages][S::kStage];
  __shared__ Item items[kMaxItems];
  __shared__ float most[S::kWN][BM];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int q = lane >> 4, r = lane & 15, sw = (r >> 1) & 7;

  if constexpr (!kGateUp && !std::is_same<OutT, Scaled16>::value) zero_rest<OutT, kThreads>(a);
  const int nw = kGateUp ? f8_blocks(a.N / 2) : (a.N + kBN - 1) / kBN;
  const int n_items = list_items<BM, WM>(a, nw, items);
  if (n_items == 0) return;
  Loader<kGateUp, BM, WM> ld(a, items, n_items, wave);
  auto load_first = [&]() {
    if (!ld.more()) return;
    uint8_t* s = stage[ld.loaded & 1];
    ld.load_tokens(s);
    ld.template load_weights<0>(s);
  };
  auto load_second = [&]() {
    if (!ld.more()) return;
    ld.template load_weights<1>(stage[ld.loaded & 1]);
    ld.next();
  };
  // Waits for this wave's loads of a part of step `step`; `after`: steps whose loads have been
  // asked for in full and lie behind it in the pipeline when that is full.
  auto landed = [&](int full) {
    if (ld.loaded >= full && ld.more())
      pipe::wait_vmcnt<S::kLoads>();
    else
      pipe::wait_vmcnt<0>();
  };
  load_first();
  load_second();
  load_first();
  const bool second = wave >= 4;
  landed(1);
  barrier();
  if (second) barrier();

  int done = 0;  // steps of the stream
  // The four waves of a turn hold both halves of the weight rows of their tokens.
  const int wm = wave / S::kWN, wn = wave % S::kWN;
  for (int j = 0; j < n_items; ++j) {
    const Item it = uniform(items + j);
    const const_f32 *ws0, *ws1;
    weight_scales<kGateUp, S>(a, it, wn, &ws0, &ws1);
    f32x4 acc[kMT][kNT];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int g = 0; g < kNT; ++g) acc[m][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int mt = min((it.row_end - it.row0 + 16 * (WM - 1 - wm) + 15) / (16 * WM), kMT);
    // Of one tile row the compiler waits for all loads in flight before it reads LDS: 16 matrices
    // of 8192 x 8192 on 64 rows each 420 us, on 128 rows 235.
    by_count<kMT, 2>(mt, [&](auto count) {
      constexpr int kM = decltype(count)::value;
      for (int st = it.k0; st < it.k1; ++st, ++done) {
        const uint8_t* s = stage[done & 1];
        const uint8_t* wtile = s + S::kTokBytes + wn * kNT * kF8Tile + lane * 16;
        const uint8_t* ts = s + S::kTokBytes + S::kWgtBytes + (16 * wm + r) * 4;
        const float s0 = ws0[st], s1 = kGateUp ? ws1[st] : 0.f;
        u32x4 x[kM + 1][2], w[kHalf][2];
        float sg[kM + 1], su[kM + 1], xs[kM + 1];
        auto read_weights = [&](int half) {
#pragma unroll
          for (int g = 0; g < (kM ? kHalf : 0); ++g) {
            const uint8_t* p = wtile + (half * kHalf + g) * kF8Tile;
            w[g][0] = *reinterpret_cast<const u32x4*>(p);
            w[g][1] = *reinterpret_cast<const u32x4*>(p + kF8Tile / 2);
          }
        };
        auto multiply = [&](int half) {
          if constexpr (kM > 0) {
            // gate_up's second scales leave registers for two results on their way
            interleaved<kM * kHalf, kGateUp ? 2 : 3>(
                [&](int i) { return mma_f8(w[i / kM], x[i % kM]); },
                [&](int i, f32x4 v) {
                  const int m = i % kM;
                  const float f = kGateUp && half ? su[m] : sg[m];
                  f32x4& sum = acc[m][half * kHalf + i / kM];
#pragma unroll
                  for (int j = 0; j < 4; ++j) sum[j] = fmaf(v[j], f, sum[j]);
                  // added here, not where the sum is used next
                  asm volatile("" : "+v"(sum));
                });
          }
        };
        // read the first half
        read_weights(0);
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          const uint8_t* p = s + (16 * (wm + WM * m) + r) * kF8Block;
          x[m][0] = *reinterpret_cast<const u32x4*>(p + ((q ^ sw) << 4));
          x[m][1] = *reinterpret_cast<const u32x4*>(p + (((4 + q) ^ sw) << 4));
          xs[m] = *reinterpret_cast<const float*>(ts + 64 * WM * m);
        }
        // Asked for behind the reads, while they are on their way (before them: 8192 rows of 8
        // matrices of 14336 x 4096 522 us, so 497).
        __builtin_amdgcn_sched_barrier(0);
        load_second();  // of step done + 1
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          sg[m] = xs[m] * s0;
          su[m] = xs[m] * s1;
        }
        if (second) landed(done + 2);  // the second half of step done
        pipe::wait_lgkm0();
        barrier();
        multiply(0);
        if (!second) landed(done + 2);
        barrier();
        // read the second half
        load_first();  // of step done + 2
        read_weights(1);
        if (second) landed(done + 2);  // the first half of step done + 1
        pipe::wait_lgkm0();
        barrier();
        multiply(1);
        if (!second) landed(done + 2);
        barrier();
      }
    });
    if (it.part >= 0) {
      store_part<S>(a, it, acc);
    } else if constexpr (kGateUp) {
      activate<S, BM, WM>(a, it, acc, wm, wn, 0, most);
      pipe::wait_lgkm0();
      barrier();  // one turn more, for both groups of waves
      store_codes<S, BM, WM>(a, it, acc, wm, wn, 0, most);
    } else {
      store_rows<S, WM, OutT>(a, it, acc, wm, wn, 0);
    }
  }
  if (!second) barrier();
}

// Tiles of rows at most: every matrix that has rows has a tile that is not full.
long long row_tiles(const F8MatmulArgs& a, int rows) {
  return a.offsets ? a.M / rows + (a.E < a.M ? a.E : a.M) : (a.M + rows - 1) / rows;
}

template <bool kGateUp, typename OutT>
hipError_t launch_turns(const F8MatmulArgs& a, hipStream_t s) {
  constexpr int BM = 256, WM = 4;
  static_assert(Shape<BM, WM>::kPartTile == kF8PartFloats, "room of a part");
  const int cell_rows = f8_cell_rows(a.N, kGateUp);
  const long long nw = kGateUp ? cell_rows / 2 : (cell_rows + 1) / 2;
  const long long total = row_tiles(a, BM) * nw;
  if (total > INT_MAX) return hipErrorInvalidValue;
  long long grid = device_cu_count();
  // the items of a workgroup have kMaxItems - 1 full rounds at most
  const long long most = grid * (kMaxItems - 1);
  grid = total < grid ? total : grid * ((total + most - 1) / most);
  turns_kernel<kGateUp, OutT><<<dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s>>>(a);
  if (a.max_parts > 0 && hipPeekAtLastError() == hipSuccess) {
    // at least two parts an item
    const long long tails = total < a.max_parts / 2 ? total : a.max_parts / 2;
    parts_kernel<kGateUp, BM, WM, OutT>
        <<<dim3(static_cast<unsigned>(tails * Shape<BM, WM>::kMT)), dim3(kThreads), 0, s>>>(a, static_cast<int>(grid));
  }
  return hipGetLastError();
}

template <bool kGateUp, int BM, bool kExact, typename OutT>
hipError_t launch_rows(const F8MatmulArgs& a, hipStream_t s) {
  const int cell_rows = f8_cell_rows(a.N, kGateUp);
  const long long nw = kGateUp ? cell_rows / 2 : (cell_rows + 1) / 2;
  const long long groups = row_tiles(a, BM) * nw;
  if (groups * kThreads > UINT_MAX) return hipErrorInvalidValue;
  rows_kernel<kGateUp, BM, kExact, OutT><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

template <int BM>
hipError_t launch_rows_of(const F8MatmulArgs& a, bool gate_up, hipStream_t s) {
  if (gate_up && a.exact) return launch_rows<true, BM, true, float>(a, s);
  if (gate_up)  // not where exact products cost next to nothing (f8_experts)
    return BM == 128 ? launch_rows<true, 128, false, float>(a, s) : hipErrorInvalidValue;
  if (a.exact) return launch_rows<false, BM, true, float>(a, s);
  if (a.out_dtype == MOE355_F32) return launch_rows<false, BM, false, float>(a, s);
  if (a.out_dtype == MOE355_BF16) return launch_rows<false, BM, false, bf16>(a, s);
  return launch_rows<false, BM, false, f16>(a, s);
}

}  // namespace

hipError_t launch_f8_tiled(const F8MatmulArgs& a, bool gate_up, int tile_rows, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  if (tile_rows == 32) return launch_rows_of<32>(a, gate_up, s);
  if (tile_rows == 64) return launch_rows_of<64>(a, gate_up, s);
  if (tile_rows == 128) return launch_rows_of<128>(a, gate_up, s);
  if (tile_rows != 256 || a.exact) return hipErrorInvalidValue;
  if (gate_up) return launch_turns<true, float>(a, s);
  if (a.slot_scales) return a.zero_rest ? hipErrorInvalidValue : launch_turns<false, Scaled16>(a, s);
  if (a.out_dtype == MOE355_F32) return launch_turns<false, float>(a, s);
  if (a.out_dtype == MOE355_BF16) return launch_turns<false, bf16>(a, s);
  return launch_turns<false, f16>(a, s);
}

}  // namespace moe355
