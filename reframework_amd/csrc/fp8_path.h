// Which kernels run an 8-bit product or expert call (formats: fp8.h). Plain C++, without a device:
// tests/test_fp8_paths.py asks it which kernels the tests' sizes reach.
#pragma once

#include <algorithm>
#include <cstddef>

#include "../../include/moe355.h"

namespace moe355 {

constexpr int kF8Block = 128;
constexpr int kF8StreamTile = 16;  // token rows of a tile of the weight-streaming kernel
constexpr int kF8PartFloats = 256 * 256;  // sums of a part of an item of 256 rows

constexpr int f8_blocks(int n) { return (n + kF8Block - 1) / kF8Block; }
constexpr int f8_pad(int n) { return f8_blocks(n) * kF8Block; }

// Which kernels run a product of M rows of E matrices of N x Kp (gate_up: N of both): tile_rows
// 0 streams the weights past 16-row tiles; max_parts: parts of items that the 256-row tiles may
// leave in memory.
struct F8Path {
  int tile_rows, max_parts;
  size_t part_bytes;
};

// By rows per matrix that has any, on average; random routing gives some matrices a tile more.
// Skewed routing is on one matrix's wrong side: experts in proportion to 1 / rank, us, even / skewed
// (most rows), B at 12 rows 112 / 124 (100), 36 rows 161 / 175 (303), 96 rows 196 / 217 (796); A at 12 rows
// 254 / 267 (34), 64 rows 321 / 370 (173), 125 rows 420 / 376 (314).
// Whole expert calls in us, A: 8 experts of H 4096, I 14336 (2 slots), B: 64 of H 2048, I 1408
// (6), C: 32 of H 1280, I 3328 (4), D: 16 of H 4096, I 6400 (2).
// Streaming / 32-row tiles: A at 1 row 112 / 165, 3 rows 228 / 247; B at 1 row 80 / 91, 2 rows 103 /
// 96, 6 rows 118 / 106; C at 4 rows 88 / 96, 12 rows 95 / 100; D at 4 rows 214 / 232. Where the tiles of
// 256 weight rows are fewer than would keep the CUs busy, or have few steps, streaming pays longer;
// products, streaming / 64 rows: one matrix of 28672 x 4096 at 8 rows 24 / 33, of 4096 x 4096
// at 12 rows 7.5 / 26; 8 of 4096 x 14336 at 8 rows 83 / 106, 12 rows to fp32 89 / 102; 32 of 6656 x 1280 at
// 8 rows 43 / 53; but 8 of 14336 x 4096 (448 such tiles) at 8 rows 83 / 75.
// 32 / 64: A at 12 rows 267 / 273; B at 12 rows 123 / 116; D at 25 rows 254 / 276; A at 64 rows
// 479 / 417.
// 64 / 128: A at 32 rows 302 / 290, 64 rows 398 / 320; B at 36 rows 157 / 157, 65 rows 212 / 178;
// C at 64 rows 167 / 135.
// 128 / 256: A at 120 rows 390 / 523, 140 rows 492 / 461; B at 96 rows 195 / 219, 122 rows 221 /
// 224; C at 106 rows 151 / 186, 128 rows 204 / 195, 150 rows 234 / 184; 4 experts of H 1024, I
// 1024 at 1000 rows, 128 items, 59 / 77. Exact products of f16 (8 of H 2048, I 4096; 256: the
// weights through LDS, a kernel since removed) at 512 rows 298 / 360, 1024 rows 560 / 561
// (now 463, fp32 545; bf16 on 256 rows 310).
constexpr int kF8StreamRows = 5, kF8StreamRowsFew = 12;

inline F8Path f8_path(int M, int N, int Kp, int E, bool exact, int cus) {
  F8Path p{};
  const int active = std::max(1, std::min(M, E)), rows = M / active;
  const long long wide = static_cast<long long>(active) * ((N + 255) / 256);
  const bool few = 2 * wide < 3 * cus || Kp / kF8Block < 16;
  if (rows <= (few ? kF8StreamRowsFew : kF8StreamRows)) return p;
  // Very few wide tiles leave most CUs idle. One matrix, streaming / tiled, of 4096 x 4096 at 16 rows
  // 7.9 / 24, 100 rows 16 / 34, of 8192 x 8192 at 64 rows 41 / 56, of 28672 x 4096 at 16 rows 26 / 32; but of
  // 16384 x 4096 at 64 rows 42 / 32, of 32768 x 4096 at 32 rows 41 / 33.
  if (rows < 128 && (8 * wide <= cus || (rows <= kF8StreamTile && 2 * wide <= cus))) return p;
  const long long items = (static_cast<long long>(M) / 256 + active / 2) * ((N + 255) / 256);
  p.tile_rows = rows <= 26 ? (rows >= 16 ? 32 : 64)
                : rows < 128 || exact || items < cus ? 128 : 256;
  // cutting items of few steps saves less than the second launch takes
  if (p.tile_rows == 256 && Kp / kF8Block >= 16) p.max_parts = cus;
  p.part_bytes = static_cast<size_t>(p.max_parts) * kF8PartFloats * sizeof(float);
  return p;
}

// The two products of an expert call of R slots, K a token. narrow: slots' results wait in 16 bits.
struct F8Experts {
  F8Path up, down;
  bool exact_up, exact_down, narrow;
};

inline F8Experts f8_experts(int R, int H, int I, int E, int K, int dtype, int cus) {
  F8Experts p{};
  // Where the weights' stream bounds the call exact products cost little (us, scaled / exact: A
  // (above) at 32 rows 290 / 295, 64 rows 320 / 342, 100 rows 348 / 403; B at 36 rows 157 /
  // 161, 96 rows 194 / 229). A bf16 result of few tokens is off by up to 0.0025 of its size
  // with the scaled ones, by 0.0017 with these.
  const int rows = R / std::max(1, std::min(R, E));
  p.exact_up = dtype != MOE355_BF16 || rows <= 40;
  p.exact_down = dtype == MOE355_F32;
  p.up = f8_path(R, 2 * I, f8_pad(H), E, p.exact_up, cus);
  if (p.up.tile_rows == 0) p.exact_up = true;  // the only gate_up that streams
  p.down = f8_path(R, H, f8_pad(I), E, p.exact_down, cus);
  // Results of a bf16 call's slots wait in 16 bits until they are weighed and added: f16 with a
  // power of two per 64 columns, whose 11 bits add little to the 8 of the result (4096 tokens of
  // 2 of 8 experts, H 4096, I 14336 1554 us, so 1539; 2048 of 6 of 64, H 2048, I 1408 238, so 225).
  // f16 results, whose own rounding is no finer, and a single slot keep fp32.
  p.narrow = dtype == MOE355_BF16 && K > 1 && p.down.tile_rows == 256;
  return p;
}

}  // namespace moe355
