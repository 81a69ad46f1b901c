"""The int8 projections' tile shapes on reductions that go round their rings: every slot is
refilled inside the loop and its second contents multiplied. The sizes that name each shape in
test_gpu_proj_i8.py and test_gpu_qkv_proj_i8.py have one reduction each, for some of two steps;
these are sizes at which the rule takes the same shape on more steps than the ring's and the
unrolled loop's together (test_int8_long_host.py checks both)."""
import pytest
import torch

from _gpu import note
from _int8 import bits16, check_product, int8_operands, product64
from test_gpu_qkv_proj_i8 import D, EPS, _gammas, _rope
from test_gpu_qkv_proj_i8_once import ONCE, _check, _formula64

pytestmark = pytest.mark.gpu

# shape, rows, in, out
LONG = [("256x256", 2691, 7168, 5000), ("256x224", 2321, 7168, 5000),
        ("256x192", 2728, 7168, 3840), ("256x160", 2210, 7168, 3840),
        ("256x128", 2321, 7168, 2500), ("128x192", 1951, 7168, 2500),
        ("128x160", 1544, 7168, 2500), ("128x128", 2506, 7168, 777),
        ("128x128p", 2321, 1280, 15360), ("128x64p", 2728, 7168, 384),
        ("128x32p", 2691, 7168, 384), ("64x64p", 1359, 7168, 384),
        ("32x64p", 2062, 7168, 100), ("32x32p", 1, 7168, 100)]
# shape, rows, hidden, heads, rot
LONG_QKV = [("256x256", 1152, 5120, 33, 128), ("256x224", 2311, 5120, 13, 96),
            ("256x192", 654, 5120, 40, 128), ("256x160", 1553, 5120, 13, 96),
            ("256x128", 392, 5120, 33, 128), ("128x192", 330, 5120, 33, 96),
            ("128x160", 132, 5120, 56, 128), ("128x128", 66, 5120, 56, 96),
            ("128x128p", 2311, 1280, 40, 128), ("128x64p", 66, 5120, 33, 96),
            ("128x32p", 2, 5120, 5, 128)]


@pytest.mark.parametrize("shape,S,K,N", LONG, ids=[s[0] for s in LONG])
def test_product(h3, shape, S, K, N):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, N, S + N)
    note(f"proj_i8 long {shape} S={S} K={K} N={N}")
    check_product(ops.proj_i8(x, xs, w, ws), product64(x, xs, w, ws))


@pytest.mark.parametrize("shape,S,K,H,rot", LONG_QKV, ids=[s[0] for s in LONG_QKV])
def test_qkv(h3, shape, S, K, H, rot):
    """Q, K and V the prologue's bits in both of its roundings; in ROUND_ONCE the formula's."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, S + K + H)
    gammas, inner = _gammas(S), H * D
    y = ops.proj_i8(x, xs, w, ws)
    check_product(y, product64(x, xs, w, ws))
    for rounding in (0, 1, ONCE):
        pos, ax, inv, table = _rope(S, rot, rounding)
        note(f"qkv_proj_i8 long {shape} S={S} K={K} H={H} rot={rot} rounding={rounding}")
        got = ops.qkv_proj_i8(x, xs, w, ws, *gammas, table, heads=H, eps=EPS, rounding=rounding)
        if rounding == ONCE:
            _check([t[:, :S] for t in got[:2]],
                   _formula64(x, xs, w, ws, gammas, table, H, rot))
            continue
        want = ops.qk_norm_rope(y[:, :inner], y[:, inner:2 * inner], *gammas, pos, ax, inv, heads=H,
                                eps=EPS, rot=rot, rounding=rounding, v_in=y[:, 2 * inner:])
        torch.cuda.synchronize()
        for name, a, b in zip("qkv", got, want):
            assert (bits16(a) == bits16(b)).all(), (name, rounding)
