// Stable counting sort of routed slots by expert.
//
// Replaces the grouping of fused_experts (reframework/moe/fused.py:70-80),
// which visits experts in ascending id and, inside an expert, slots in
// ascending flat (t,k) order. Two launches, no host round trip:
//   1. count:   each block histograms kPermuteChunk slots into LDS and writes
//               its per-expert counts (256 slots a block, one per thread: at
//               1024 a block ranked its slots in four dependent rounds, and
//               the scatter of 8192 slots ran on 8 CUs);
//   2. scatter: each block rebuilds the global expert starts and its own
//               prefix from the count table, ranks its slots stably with
//               wavefront ballots, and writes slot_to_row / row_src. Block 0
//               also writes expert_offsets and the tile map the expert-FFN
//               kernels are launched over.
// Up to kPermuteSingleMax slots one block of that many threads does both.
// Only indices move here (4*T*K bytes each way); token rows are gathered later
// by the gate_up kernel straight from x, so no permuted copy of x is written.
#include "common.h"

namespace moe355 {
namespace {

#include "permute_body.h"

constexpr int kThreads = kPermuteThreads;
constexpr int kWaves = kThreads / kWave;

__global__ __launch_bounds__(kThreads) void count_kernel(const PermuteArgs a) {
  permute_count(a, blockIdx.x);
}

__global__ __launch_bounds__(kOneThreads) void permute_one_kernel(const PermuteArgs a) {
  permute_one(a);
}

__global__ __launch_bounds__(kThreads) void scatter_kernel(const PermuteArgs a) {
  __shared__ int base[kMaxExperts];       // first row of this block's slots of expert e
  __shared__ int start[kMaxExperts + 1];  // expert_offsets
  __shared__ int total[kMaxExperts];
  __shared__ int wave_cnt[kWaves][kMaxExperts];

  const int b = blockIdx.x, tid = threadIdx.x;
  const int lane = tid & (kWave - 1), wave = tid / kWave;

  {
    // Slots of expert e in all blocks (total) and in the blocks before this
    // one (base), from the count table. Thread tid sums expert tid % E over
    // part tid / E of the blocks (P = min(256 / E, 8) parts; one part when
    // E > 128) with its loads unrolled, so they are in flight together; the
    // parts are added in LDS, at most 8 per expert. One thread per expert
    // walking every block paid one L2 round trip per block (32 for 64 experts
    // at 4096 tokens).
    __shared__ int ptot[kThreads], ppre[kThreads];
    const int P = min(kThreads / a.E, 8);
    const int e = tid % a.E, p = tid / a.E;
    int tot = 0, pre = 0;
    if (p < P) {
      const int per = (a.n_blocks + P - 1) / P;
      const int b1 = min(a.n_blocks, (p + 1) * per);
#pragma unroll 8
      for (int bb = p * per; bb < b1; ++bb) {
        const int c = a.block_counts[bb * a.E + e];
        tot += c;
        pre += bb < b ? c : 0;
      }
    }
    ptot[tid] = tot;
    ppre[tid] = pre;
    __syncthreads();
    for (int x = tid; x < a.E; x += kThreads) {
      int t2 = 0, p2 = 0;
      for (int q = 0; q < P; ++q) {
        t2 += ptot[q * a.E + x];
        p2 += ppre[q * a.E + x];
      }
      total[x] = t2;
      base[x] = p2;
    }
  }
  __syncthreads();
  if (wave == 0) wave_scan(a.E, lane, [&](int x) { return total[x]; }, start);
  __syncthreads();
  for (int e = tid; e < a.E; e += kThreads) base[e] += start[e];

  if (b == 0) {
    __shared__ int order[kMaxExperts];            // expert at place p
    __shared__ int place_start[kMaxExperts + 1];  // first tile of place p
    for (int e = tid; e <= a.E; e += kThreads) a.offsets[e] = start[e];
    for (int e = tid; e < a.E; e += kThreads) order[size_place(total, a.E, e)] = e;
    __syncthreads();
    if (wave == 0)
      wave_scan(a.E, lane, [&](int x) { return (total[order[x]] + a.tile_rows - 1) / a.tile_rows; },
                place_start);
    __syncthreads();
    const int ntiles = min(place_start[a.E], a.max_tiles);
    if (tid == 0) {
      a.tile_map[0] = ntiles;
      a.tile_map[1] = a.tile_rows;
    }
    for (int j = tid; j < ntiles; j += kThreads) write_tile(a, start, order, place_start, j);
  }

  for (int r = 0; r < kRounds; ++r) {
    for (int i = tid; i < kWaves * a.E; i += kThreads) wave_cnt[i / a.E][i % a.E] = 0;
    __syncthreads();
    const int slot = b * kPermuteChunk + r * kThreads + tid;
    const int e = slot < a.R ? routed_expert(a, slot) : -1;
    unsigned long long same;
    const int rank = rank_in_wave(e, lane, &same);
    if (e >= 0 && rank == 0) wave_cnt[wave][e] = __popcll(same);
    __syncthreads();
    if (slot < a.R) {
      if (e >= 0) {
        int row = base[e] + rank;
        for (int w = 0; w < wave; ++w) row += wave_cnt[w][e];
        a.slot_to_row[slot] = row;
        a.row_src[row] = slot / a.K;
      } else {
        a.slot_to_row[slot] = -1;
      }
    }
    __syncthreads();
    for (int ee = tid; ee < a.E; ee += kThreads) {
      int add = 0;
      for (int w = 0; w < kWaves; ++w) add += wave_cnt[w][ee];
      base[ee] += add;
    }
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_permute_scatter(const PermuteArgs& a, hipStream_t s) {
  scatter_kernel<<<dim3(a.n_blocks), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_permute(const PermuteArgs& a, hipStream_t s) {
  if (a.R == 0) return hipSuccess;
  if (a.n_blocks == 1) {
    permute_one_kernel<<<dim3(1), dim3(kOneThreads), 0, s>>>(a);
    return hipGetLastError();
  }
  count_kernel<<<dim3(a.n_blocks), dim3(kThreads), 0, s>>>(a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  return launch_permute_scatter(a, s);
}

}  // namespace moe355
