// Which kernel and tile shape an int8 projection of these sizes runs on. Plain C++,
// so a CPU test can check it.
#pragma once

#include <algorithm>
#include <cstdint>

#include "proj_tile.h"

namespace h3hip {

enum class ProjI8Tile {
  kRows,        // the kernel for few rows (proj_i8.hip)
  k256x256,     // proj_i8_gemm_kernel, channels x tokens
  k256x224,
  k256x192,
  k256x160,
  k256x128,
  k128x192,
  k128x160,
  k128x128,
  k128x64,
};

struct ProjI8Shape {
  ProjI8Tile tile;
  int channels, tokens;
  double cost;   // time of a tile where all CUs work, that of 256 x 256 being 1
};
constexpr ProjI8Shape kProjI8Shapes[] = {
    {ProjI8Tile::k256x256, 256, 256, 1.00}, {ProjI8Tile::k256x224, 256, 224, 0.90},
    {ProjI8Tile::k256x192, 256, 192, 0.78}, {ProjI8Tile::k256x160, 256, 160, 0.67},
    {ProjI8Tile::k256x128, 256, 128, 0.57}, {ProjI8Tile::k128x192, 128, 192, 0.50},
    {ProjI8Tile::k128x160, 128, 160, 0.40}, {ProjI8Tile::k128x128, 128, 128, 0.39},
    {ProjI8Tile::k128x64, 128, 64, 0.28},
};

// Whether a shape's tiles can be counted and launched: 16 bits each way in a tile's
// number (tile_order.h), and a grid of fewer than 2^32 threads of 256 a workgroup, whose
// lists may be two chunks apart.
inline bool proj_i8_fits(int64_t tokens, int64_t channels, int tile_tokens, int tile_channels) {
  const int64_t m = (tokens + tile_tokens - 1) / tile_tokens;
  const int64_t n = (channels + tile_channels - 1) / tile_channels;
  return m <= 65535 && n <= 65535 && m * n <= (1 << 23);
}

// The launch order of a grid that fits; the last channel tile may be part used.
inline ProjGrid proj_i8_grid(int tokens, int channels, int tile_tokens, int tile_channels) {
  const int n = (int)(((int64_t)channels + tile_channels - 1) / tile_channels);
  return proj_grid(tokens, n * tile_channels, tile_tokens, tile_channels);
}

// The tile whose rounds take the least time, of those whose grid over `padded` rows
// (tokens and the zero rows behind them, which cost little) fits a launch. heads: the output is written by heads, so a
// tile may not hold channels of two of Q, K and V.
inline ProjI8Tile pick_proj_i8_tile(int tokens, int padded, int channels, bool heads) {
  if (tokens <= 16) return ProjI8Tile::kRows;
  double best = 0;
  ProjI8Tile tile = ProjI8Tile::kRows;
  for (const ProjI8Shape& s : kProjI8Shapes) {
    if ((heads && channels / 3 % s.channels != 0) ||
        !proj_i8_fits(padded, channels, s.tokens, s.channels))
      continue;
    const double cost = s.cost * proj_i8_grid(tokens, channels, s.tokens, s.channels).rounds;
    if (tile == ProjI8Tile::kRows || cost < best) {
      best = cost;
      tile = s.tile;
    }
  }
  return tile;
}

}  // namespace h3hip
