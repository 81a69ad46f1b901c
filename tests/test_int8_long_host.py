"""test_gpu_int8_long.py's sizes are what it says (CPU only): the rule takes the shape that each
names, on more steps than its rings hold and its loop unrolls."""
import test_gpu_int8_long as long
from test_gemm_i8_loop_gen import G
from test_proj_i8_tile_host import NAMES, pick  # noqa: F401  (a fixture)


def test_sizes_reach_their_shapes_on_long_reductions(pick):  # noqa: F811
    cases = [(name, (S, N, K // 128, 0)) for name, S, K, N in long.LONG]
    cases += [(name, (S, 384 * H, K // 128, 1)) for name, S, K, H, _ in long.LONG_QKV]
    assert [name for name, _ in cases] == NAMES + NAMES[:11]
    assert [NAMES[int(c[0])] for c in pick([c for _, c in cases])] == NAMES + NAMES[:11]
    for name, (_, _, steps, _) in cases:
        g = G.Gen(name)
        assert steps > max(g.rw, g.rx) + g.unroll, (name, steps)
