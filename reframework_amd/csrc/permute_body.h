// Device code of the permute (permute.hip) that the quantised experts' first launch
// (mx_format.hip) runs too. Included inside their anonymous namespaces.
#pragma once

constexpr int kPermuteThreads = 256;
constexpr int kRounds = kPermuteChunk / kPermuteThreads;  // count + scatter launches
constexpr int kOneThreads = kPermuteSingleMax;      // the one-block permute: a thread per slot
constexpr int kOneWaves = kOneThreads / kWave;
static_assert(kMaxExperts <= 256, "the scatter ranks slots by the 8 bits of the expert id");

// Counts of block b's slots by expert (kPermuteThreads threads).
__device__ __forceinline__ void permute_count(const PermuteArgs& a, int b) {
  __shared__ int hist[kMaxExperts];
  const int tid = threadIdx.x;
  for (int e = tid; e < a.E; e += kPermuteThreads) hist[e] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int slot = b * kPermuteChunk + r * kPermuteThreads + tid;
    if (slot < a.R) {
      const int e = routed_expert(a, slot);
      if (e >= 0) atomicAdd(&hist[e], 1);
    }
  }
  __syncthreads();
  for (int e = tid; e < a.E; e += kPermuteThreads) a.block_counts[b * a.E + e] = hist[e];
}

// Rank of this lane's slot among the wave's slots of the same expert (e < 0: not
// routed): the routed lanes that agree with this lane on each of the 8 bits of
// the expert id (E <= 256), one ballot per bit instead of one per distinct
// expert. `same` gets those lanes.
__device__ __forceinline__ int rank_in_wave(int e, int lane, unsigned long long* same) {
  unsigned long long m = __ballot(e >= 0);
#pragma unroll
  for (int bit = 0; bit < 8; ++bit) {
    const bool set = (e >> bit) & 1;
    const unsigned long long b = __ballot(set);
    m &= set ? b : ~b;
  }
  *same = m;
  return __popcll(m & ((1ull << lane) - 1ull));
}

// Exclusive scan by one wave of E values, lane l owning l*per .. l*per+per-1
// (per <= 4 for E <= 256): out[i] for i <= E, out[E] the sum.
template <typename F>
__device__ __forceinline__ void wave_scan(int E, int lane, F value, int* out) {
  constexpr int kPer = kMaxExperts / kWave;
  const int per = (E + kWave - 1) / kWave;
  int v[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int x = lane * per + i;
    v[i] = i < per && x < E ? value(x) : 0;
    sum += v[i];
  }
  int inc = sum;  // inclusive across lanes
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int up = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += up;
  }
  int ex = inc - sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int x = lane * per + i;
    if (i < per && x < E) out[x] = ex;
    ex += v[i];
  }
  if (lane == kWave - 1) out[E] = inc;
}

// The tile map lists the experts' tiles in an interleaved order of their
// sizes (largest, smallest, second largest, second smallest, ..; ties by
// expert id), so the GEMMs' rounds mix weight-stream-bound items of small
// experts with MFMA-bound items of large ones: fine-grained 4096 tokens
// gate_up -2 %, Phi-3.5 2048 tokens -2 %, Mixtral 4096 tokens down -2 %
// against expert-id order. Rank r of the size order goes to place 2 r in
// the first half, 2 (E - 1 - r) + 1 in the second.
__device__ __forceinline__ int size_place(const int* total, int E, int e) {
  const int n = total[e];
  int r = 0;
  for (int f = 0; f < E; ++f) r += (total[f] > n || (total[f] == n && f < e)) ? 1 : 0;
  return 2 * r < E ? 2 * r : 2 * (E - 1 - r) + 1;
}

// Tile j of the map (place_start: first tile of each place of `order`).
__device__ __forceinline__ void write_tile(const PermuteArgs& a, const int* start, const int* order,
                                           const int* place_start, int j) {
  int lo = 0, hi = a.E - 1;  // last place with place_start[p] <= j
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (place_start[mid] <= j) lo = mid; else hi = mid - 1;
  }
  const int e = order[lo];
  a.tile_map[2 + 2 * j] = e;
  a.tile_map[3 + 2 * j] =
      start[e] + (j - place_start[lo]) *
                     (a.full_tiles ? a.tile_rows : tile_height(start[e + 1] - start[e], a.tile_rows));
}

// All slots fit one block (up to kPermuteSingleMax), one thread each: a chain of
// dependent steps, so the fewest of them decide. Each wave ranks its 64 slots
// and counts them per expert; a thread per expert turns the waves' counts into
// bases; then one wave scans the experts while the others rank them by size, and
// rows and tile map are written. With 256 threads in four rounds, each with its
// own barriers, and a counting pass before them this took 10.9 us at 1024 slots
// of 8 experts and 12.5 at 999 of 12; now 5.7 and 5.6.
__device__ __forceinline__ void permute_one(const PermuteArgs& a) {
  __shared__ int wave_cnt[kOneWaves][kMaxExperts];  // slots of expert e in a wave, then before it
  __shared__ int total[kMaxExperts], start[kMaxExperts + 1];
  __shared__ int order[kMaxExperts], place_start[kMaxExperts + 1];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;

  const int e = tid < a.R ? routed_expert(a, tid) : -1;
  for (int x = lane; x < a.E; x += kWave) wave_cnt[wave][x] = 0;  // this wave's own row
  unsigned long long same;
  const int rank = rank_in_wave(e, lane, &same);
  if (e >= 0 && rank == 0) wave_cnt[wave][e] = __popcll(same);
  __syncthreads();
  if (tid < a.E) {
    int c[kOneWaves], sum = 0;
#pragma unroll
    for (int w = 0; w < kOneWaves; ++w) c[w] = wave_cnt[w][tid];
#pragma unroll
    for (int w = 0; w < kOneWaves; ++w) {
      wave_cnt[w][tid] = sum;
      sum += c[w];
    }
    total[tid] = sum;
  }
  __syncthreads();
  if (wave == 0) wave_scan(a.E, lane, [&](int x) { return total[x]; }, start);
  for (int x = tid - kWave; x >= 0 && x < a.E; x += kOneThreads) order[size_place(total, a.E, x)] = x;
  __syncthreads();
  if (wave == 1)
    wave_scan(a.E, lane, [&](int x) { return (total[order[x]] + a.tile_rows - 1) / a.tile_rows; },
              place_start);
  if (tid < a.R) {
    const int row = e >= 0 ? start[e] + wave_cnt[wave][e] + rank : -1;
    a.slot_to_row[tid] = row;
    if (row >= 0) a.row_src[row] = tid / a.K;
  }
  for (int x = tid; x <= a.E; x += kOneThreads) a.offsets[x] = start[x];
  __syncthreads();
  const int ntiles = min(place_start[a.E], a.max_tiles);
  if (tid == 0) {
    a.tile_map[0] = ntiles;
    a.tile_map[1] = a.tile_rows;
  }
  for (int j = tid; j < ntiles; j += kOneThreads) write_tile(a, start, order, place_start, j);
}
