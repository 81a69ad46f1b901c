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

// Microseconds of a launch: start + rounds * (round + round_step * reduction steps) + share *
// (tile + tile_step * steps), rounds being the tiles the busiest CU runs and share all tiles over
// the CUs: what a CU waits for goes by rounds, what all of them share, the power limit and the
// caches, by share.
struct ProjMx4Shape {
  ProjMx4Tile tile;
  int channels, tokens;
  float start, round, round_step, per_tile, tile_step;
};
constexpr ProjMx4Shape kProjMx4Shapes[] = {
    {ProjMx4Tile::k256x256, 256, 256, 4.56f, 4.45f, 0.965f, 6.75f, 0.632f},
    {ProjMx4Tile::k256x224, 256, 224, 5.17f, 3.29f, 0.869f, 6.00f, 0.447f},
    {ProjMx4Tile::k256x192, 256, 192, 4.46f, 3.04f, 0.727f, 5.55f, 0.405f},
    {ProjMx4Tile::k256x160, 256, 160, 3.79f, 2.70f, 0.712f, 4.62f, 0.337f},
    {ProjMx4Tile::k256x128, 256, 128, 4.36f, 3.27f, 0.615f, 3.55f, 0.245f},
    {ProjMx4Tile::k128x192, 128, 192, 2.80f, 3.03f, 0.609f, 2.63f, 0.312f},
    {ProjMx4Tile::k128x160, 128, 160, 2.83f, 2.91f, 0.384f, 2.34f, 0.264f},
    {ProjMx4Tile::k128x128, 128, 128, 2.46f, 2.67f, 0.261f, 1.93f, 0.219f},
    {ProjMx4Tile::k128x128p, 128, 128, 4.31f, 0.00f, 0.393f, 2.61f, 0.109f},
    {ProjMx4Tile::k128x64p, 128, 64, 3.69f, 0.00f, 0.237f, 1.64f, 0.093f},
    {ProjMx4Tile::k128x32p, 128, 32, 3.56f, 0.00f, 0.196f, 1.05f, 0.024f},
    {ProjMx4Tile::k64x64p, 64, 64, 2.44f, 0.91f, 0.179f, 0.50f, 0.052f},
    {ProjMx4Tile::k32x64p, 32, 64, 2.13f, 1.19f, 0.176f, 0.27f, 0.001f},
    {ProjMx4Tile::k32x32p, 32, 32, 2.45f, 0.63f, 0.088f, 0.42f, 0.000f},
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

// Time of a launch of `tiles` tiles in `rounds` rounds.
inline float proj_mx4_cost(const ProjMx4Shape& s, int tiles, int rounds, int steps) {
  return s.start + (float)rounds * (s.round + s.round_step * (float)steps) +
         (float)tiles / (32 * kOrderXcds) * (s.per_tile + s.tile_step * (float)steps);
}

// The shape whose launch takes least; kNone if none fits one. heads: the output is
// written by heads, so a tile holds whole ones. steps: of 256 values of the reduction.
//
// The constants were fitted to what they pick: 7,571 sizes of both forms (1 to 32,000 tokens, 200 to
// 21,504 channels, 1 to 28 steps; heads with norm in H3HIP_ROUND_ONCE) timed on every shape on MI355X.
// On the 30% of them (2,243) that the search did not see the pick is 1.0% slower than the best shape
// on average, 1.9% past 2,000 tokens; with int8's constants, a term in rounds alone, 1.6% and 3.8%. Every
// shape is the pick for 30 of the sizes or more, and without it those take 3-20% longer. A cost
// ranks shapes and is no time of its own: of nine in ten picks it is 0.79 to 1.16 of the time. Shapes in
// turn (replays, medians of 7, us; * the pick):
//   31,885 x 5,120 x 5,120          256 x 256 385, x 224* 399, x 192 405, x 160 420, 128 x 192 542
//   31,885 x 5,120 x 40 heads       256 x 256 1,224, x 224* 1,246, x 192 1,273, x 160 1,328, 128 x 192 1,507
//   1,151 x 5,376 x 56 heads        256 x 256 83, x 224 80, x 192* 73, x 160 82, 128 x 192 81
// Which of the first three is best depends on how warm the chip is: one after another without a
// pause, on another card, 469, 445, 434; 1,342, 1,294, 1,334; 89, 84, 78.
inline ProjMx4Tile pick_proj_mx4_tile(int tokens, int channels, int steps, bool heads) {
  float best = 0.f;
  ProjMx4Tile tile = ProjMx4Tile::kNone;
  for (const ProjMx4Shape& s : kProjMx4Shapes) {
    if ((heads && s.channels < 128) || !proj_mx4_fits(tokens, channels, s)) continue;
    // A round for each tile a CU gets at least: most shapes need no look at their lists.
    const int tiles_m = (int)(((int64_t)tokens + s.tokens - 1) / s.tokens);
    const int tiles_n = (int)(((int64_t)channels + s.channels - 1) / s.channels);
    const int tiles = tiles_m * tiles_n;
    const int least = (tiles + 32 * kOrderXcds - 1) / (32 * kOrderXcds);
    if (tile != ProjMx4Tile::kNone && proj_mx4_cost(s, tiles, least, steps) >= best) continue;
    const int rounds = proj_mx4_grid(tokens, channels, s.tokens, s.channels).rounds;
    const float cost = proj_mx4_cost(s, tiles, rounds, steps);
    if (tile == ProjMx4Tile::kNone || cost < best) {
      best = cost;
      tile = s.tile;
    }
  }
  return tile;
}

}  // namespace h3hip
