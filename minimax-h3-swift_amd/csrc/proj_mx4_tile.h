// Which tile shape a 4-bit projection of these sizes runs on. Plain C++, so a CPU test
// can check it.
#pragma once

#include <algorithm>
#include <cstdint>

#include "proj_tile.h"

namespace h3hip {

enum class ProjMx4Tile {   // channels x tokens; p: two workgroups a CU
  k256x256,
  k256x224,
  k256x192,
  k256x160,
  k256x128,
  k128x192,
  k128x160,
  k128x128,
  k128x128p,
  k128x64p,
  k128x32p,
  k64x64p,
  k32x64p,
  k32x32p,
  kNone,
};

// Microseconds of a launch: start + rounds * (tile + step * reduction steps), rounds
// being the tiles the busiest CU runs.
struct ProjMx4Shape {
  ProjMx4Tile tile;
  int channels, tokens;
  float start, per_tile, per_step;
};
constexpr ProjMx4Shape kProjMx4Shapes[] = {
    {ProjMx4Tile::k256x256, 256, 256, 0.0f, 12.0f, 1.04f},
    {ProjMx4Tile::k256x224, 256, 224, 0.0f, 10.9f, 0.94f},
    {ProjMx4Tile::k256x192, 256, 192, 0.1f, 9.5f, 0.83f},
    {ProjMx4Tile::k256x160, 256, 160, 0.5f, 8.7f, 0.72f},
    {ProjMx4Tile::k256x128, 256, 128, 0.8f, 7.2f, 0.63f},
    {ProjMx4Tile::k128x192, 128, 192, 1.1f, 6.0f, 0.50f},
    {ProjMx4Tile::k128x160, 128, 160, 1.5f, 5.1f, 0.46f},
    {ProjMx4Tile::k128x128, 128, 128, 1.8f, 4.3f, 0.42f},
    {ProjMx4Tile::k128x128p, 128, 128, 4.7f, 1.1f, 0.51f},
    {ProjMx4Tile::k128x64p, 128, 64, 3.2f, 1.3f, 0.29f},
    {ProjMx4Tile::k128x32p, 128, 32, 3.2f, 1.2f, 0.24f},
    {ProjMx4Tile::k64x64p, 64, 64, 3.2f, 1.3f, 0.18f},
    {ProjMx4Tile::k32x64p, 32, 64, 3.1f, 1.0f, 0.125f},
    {ProjMx4Tile::k32x32p, 32, 32, 3.2f, 0.8f, 0.080f},
};

// Whether a shape's tiles can be counted and launched: 16 bits each way in a tile's
// number (tile_order.h), and a grid of fewer than 2^32 threads of 256 a workgroup, whose
// lists may be two chunks apart.
inline bool proj_mx4_fits(int64_t tokens, int64_t channels, const ProjMx4Shape& s) {
  const int64_t m = (tokens + s.tokens - 1) / s.tokens;
  const int64_t n = (channels + s.channels - 1) / s.channels;
  return m <= 65535 && n <= 65535 && m * n <= (1 << 23);
}

// The launch order of a grid that fits; the last channel tile may be part used.
inline ProjGrid proj_mx4_grid(int tokens, int channels, int tile_tokens, int tile_channels) {
  const int n = (int)(((int64_t)channels + tile_channels - 1) / tile_channels);
  return proj_grid(tokens, n * tile_channels, tile_tokens, tile_channels);
}

// The shape whose launch takes least; kNone if none fits one. heads: the output is
// written by heads, so a tile holds whole ones.
//
// The constants are least squares over 440 sizes (1 to 18,102 tokens, 777 to 15,360
// channels, 3 to 56 steps, without norm) of every shape on MI355X, whose times they give to
// 9-19% (rms). What they pick is within 0.9% of the fastest shape on average, 15% at most, and
// within 1.4-2.4% (31%) on 1,074 sizes of the QKV forms, which they were not fitted to. They
// rank shapes and are no time of a call: neither the norm nor W's bytes are in them (QKV of
// 1,151 x 56 heads x 5,376 is 89 us by them and takes 116-120). Few
// rows are where it matters: one token x 5,120 x 5,120 takes 7.5 us on 160 tiles of 32 x 32,
// 15.7 on 40 of 128 x 64 and 27 on 20 of 256 x 128; 125 tokens 12.7 on 64 x 64, 15.4 on 32 x 32.
inline ProjMx4Tile pick_proj_mx4_tile(int tokens, int channels, int steps, bool heads) {
  float best = 0.f;
  ProjMx4Tile tile = ProjMx4Tile::kNone;
  for (const ProjMx4Shape& s : kProjMx4Shapes) {
    if ((heads && s.channels < 128) || !proj_mx4_fits(tokens, channels, s)) continue;
    const float round = s.per_tile + s.per_step * (float)steps;
    // A round for each tile a CU gets at least: most shapes need no look at their lists.
    const int tiles_m = (int)(((int64_t)tokens + s.tokens - 1) / s.tokens);
    const int tiles_n = (int)(((int64_t)channels + s.channels - 1) / s.channels);
    const int least = (tiles_m * tiles_n + 32 * kOrderXcds - 1) / (32 * kOrderXcds);
    if (tile != ProjMx4Tile::kNone && s.start + (float)least * round >= best) continue;
    const int rounds = proj_mx4_grid(tokens, channels, s.tokens, s.channels).rounds;
    const float cost = s.start + (float)rounds * round;
    if (tile == ProjMx4Tile::kNone || cost < best) {
      best = cost;
      tile = s.tile;
    }
  }
  return tile;
}

}  // namespace h3hip
