"""The rule that picks a 4-bit projection's tile shape (csrc/proj_mx4_tile.h, compiled here
with g++): every size gets a shape that fits a launch and, for outputs written by heads, one
that holds whole heads; more rows or channels never make the picked
launch cheaper; and the shapes the GPU tests are meant to reach are reached."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "minimax-h3-swift_amd", "csrc")

HARNESS = r"""
#include "proj_mx4_tile.h"
#include <cstdio>
#include <cstdlib>
#include <set>
using namespace h3hip;
int main(int argc, char** argv) {
  for (int a = 1; a + 3 < argc; a += 4) {
    const int t = std::atoi(argv[a]), n = std::atoi(argv[a + 1]), k = std::atoi(argv[a + 2]);
    const ProjMx4Tile tile = pick_proj_mx4_tile(t, n, k, std::atoi(argv[a + 3]) != 0);
    if (tile == ProjMx4Tile::kNone) { std::printf("0 0 0 1 0\n"); continue; }
    const ProjMx4Shape& s = kProjMx4Shapes[(int)tile];
    const ProjGrid g = proj_mx4_grid(t, n, s.tokens, s.channels);
    bool once = s.tile == tile;
    const long tiles = (long)((t + s.tokens - 1L) / s.tokens) * ((n + s.channels - 1L) / s.channels);
    if (tiles < 100000) {
      std::set<long> seen;
      long count = 0;
      for (int x = 0; x < kOrderXcds; x++)
        for (int p = 0; p < g.order.length(x); p++, count++) {
          const uint32_t v = g.order.tile(x, p);
          if ((long)(v >> 16) * s.tokens < t && (long)(v & 0xffff) * s.channels < n) seen.insert(v);
        }
      once = once && count == tiles && (long)seen.size() == tiles;
    }
    once = once && 8L * g.longest * 256 < (1L << 32);
    std::printf("%d %d %d %d %f\n", (int)tile, s.channels, s.tokens, once ? 1 : 0,
                proj_mx4_cost(s, (int)tiles, g.rounds, k));
  }
}
"""


@pytest.fixture(scope="module")
def pick(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    d = tmp_path_factory.mktemp("tile4")
    (d / "t.cpp").write_text(HARNESS)
    subprocess.run([gxx, "-O1", "-std=c++17", f"-I{CSRC}", str(d / "t.cpp"), "-o", str(d / "t")],
                   check=True)

    def run(cases):
        out = subprocess.run([str(d / "t")] + [str(int(v)) for c in cases for v in c], check=True,
                             capture_output=True, text=True).stdout
        return [tuple(float(v) for v in ln.split()) for ln in out.splitlines()]
    return run


TOKENS = (1, 2, 16, 31, 33, 64, 65, 100, 125, 129, 300, 637, 917, 1151, 4096, 18102, 31885)


def test_every_tile_once_in_a_launch_that_fits(pick):
    cases = [(t, n, k, 0) for t in TOKENS for n in (1, 100, 777, 5120, 15360) for k in (1, 8, 40)]
    cases += [(1, 16_000_000, 1, 0), (1_100_000, 24, 32, 0), (16_776_960, 200, 1, 0),
              (40, 1_100_000, 32, 0), (150_000, 16384, 1, 0), (2_000_000, 8, 1, 0)]
    assert all(once and ch for _, ch, _, once, _ in pick(cases))
    # Past what any shape can count: refused, not wrapped.
    assert [c[1] for c in pick([(16_776_961, 200, 1, 0), (2**31 - 1, 1, 1, 0),
                                (1, 2**31 - 1, 1, 0), (10_000_000, 1_000_000, 1, 0)])] == [0] * 4


def test_heads_are_whole(pick):
    cases = [(t, 384 * h, k, 1) for t in TOKENS for h in (1, 2, 3, 5, 7, 40, 56) for k in (1, 8, 40)]
    for (t, n, k, _), (_, ch, _, once, _) in zip(cases, pick(cases)):
        assert once and ch in (128, 256), (t, n, k, ch)


def test_larger_calls_are_not_cheaper(pick):
    for n in (777, 5120, 15360):
        cost = [c[4] for c in pick([(t, n, 40, 0) for t in TOKENS])]
        assert cost == sorted(cost), (n, cost)


NAMES = ["256x256", "256x224", "256x192", "256x160", "256x128", "128x192", "128x160", "128x128",
         "128x128p", "128x64p", "128x32p", "64x64p", "32x64p", "32x32p"]


def test_gpu_tests_reach_every_shape(pick):
    """The sizes that test_gpu_proj_mx4.py and test_gpu_qkv_proj_mx4.py name by shape."""
    import test_gpu_proj_mx4 as out
    import test_gpu_qkv_proj_mx4 as qkv
    assert [s[0] for s in out.SHAPES] == NAMES and [s[0] for s in qkv.SHAPES] == NAMES[:11]
    cases = [(S, N, K // 256, 0) for _, S, K, N in out.SHAPES]
    cases += [(S, 384 * H, K // 256, 1) for _, S, K, H, _ in qkv.SHAPES]
    assert [NAMES[int(c[0])] for c in pick(cases)] == NAMES + NAMES[:11]
    # Odd head counts on tiles of two heads: both kinds of tile that hold two parts' or one head.
    odd = pick([(S, 384 * H, K // 256, 1) for S, K, H, _ in qkv.ODD_HEADS])
    assert [NAMES[int(c[0])] for c in odd[:5]] == NAMES[:5]
