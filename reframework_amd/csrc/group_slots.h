// Grouping of a decode step's routed slots by one wave, for the first launch of the
// weight-streaming kernels (ffn_skinny.hip, mx_format.hip). Included inside their
// anonymous namespaces, after kRows, the rows of a token tile.
#pragma once

// Grouping of <= 64 routed slots by one wave, the same stable counting sort
// as the permute kernels (experts ascending, slots ascending within an
// expert): lane s holds slot s. Each slot ORs its bit into its expert's 64-bit
// mask in LDS; an expert's row count is its mask's popcount and a slot's rank
// among its expert's slots the popcount of the mask bits below it, so no step
// depends on how many distinct experts there are. Lane l owns experts 4 l ..
// 4 l + 3 (E <= 256); one wave scan gives every expert's first row and first
// tile. Returns, for token tile ttile, its expert, first row and row end in
// meta[1..3] and the tile count in meta[0]; rowsrc[row] = source token of each
// permuted row. With write_global the wave also writes the permute's outputs
// (offsets, slot_to_row, row_src, tile_map with kRows-row tiles in expert
// order) for the later stages.
constexpr int kGroupExpertsPerLane = 4;
static_assert(kGroupExpertsPerLane * kWave >= kMaxExperts, "experts per lane");

__device__ void group_slots(const PermuteArgs& pa, int ttile, bool write_global, int* meta,
                            int* rowsrc, unsigned long long* emask, int* estart) {
  const int lane = threadIdx.x & (kWave - 1);
  constexpr int P = kGroupExpertsPerLane;
#pragma unroll
  for (int i = 0; i < P; ++i) emask[P * lane + i] = 0ull;
  const int e = lane < pa.R ? routed_expert(pa, lane) : -1;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  if (e >= 0) atomicOr(&emask[e], 1ull << lane);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  // this lane's experts: row counts and tile counts, then exclusive scans
  int cnt[P], nt[P], rows = 0, tiles = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int x = P * lane + i;
    cnt[i] = x < pa.E ? __popcll(emask[x]) : 0;
    nt[i] = (cnt[i] + kRows - 1) / kRows;
    rows += cnt[i];
    tiles += nt[i];
  }
  int rscan = rows, tscan = tiles;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int rv = __shfl_up(rscan, o, kWave), tv = __shfl_up(tscan, o, kWave);
    if (lane >= o) {
      rscan += rv;
      tscan += tv;
    }
  }
  const int total_rows = __shfl(rscan, kWave - 1, kWave);
  const int total_tiles = __shfl(tscan, kWave - 1, kWave);
  int rstart = rscan - rows, tstart = tscan - tiles;
  if (lane == 0) {
    meta[0] = total_tiles;
    meta[1] = -1;
    meta[2] = 0;
    meta[3] = 0;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int x = P * lane + i;
    if (x < pa.E) {
      estart[x] = rstart;
      if (ttile >= tstart && ttile < tstart + nt[i]) {
        const int r0 = rstart + (ttile - tstart) * kRows;
        meta[1] = x;
        meta[2] = r0;
        meta[3] = min(r0 + kRows, rstart + cnt[i]);
      }
      if (write_global) {
        pa.offsets[x] = rstart;
        for (int j = 0; j < nt[i]; ++j) {
          pa.tile_map[2 + 2 * (tstart + j)] = x;
          pa.tile_map[3 + 2 * (tstart + j)] = rstart + j * kRows;
        }
      }
    }
    rstart += cnt[i];
    tstart += nt[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const unsigned long long lt_mask = (1ull << lane) - 1ull;
  const int row = e >= 0 ? estart[e] + __popcll(emask[e] & lt_mask) : -1;
  if (row >= 0) rowsrc[row] = lane / pa.K;
  if (!write_global) return;
  if (lane < pa.R) pa.slot_to_row[lane] = row;
  if (row >= 0) pa.row_src[row] = lane / pa.K;
  if (lane == 0) {
    pa.offsets[pa.E] = total_rows;
    pa.tile_map[0] = total_tiles;
    pa.tile_map[1] = kRows;
  }
}
