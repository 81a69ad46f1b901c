"""h3hip_qkv_proj_i8 in ROUND_ONCE on the GPU: the product stays in fp32 through the head
norm and the rotation, and Q and K are rounded to bf16 once.

Against the formula in 64 bits. Of what is rounded to fp32 (2^-24 each, relative): the sum's
conversion and its two products with the scales (3); a sum of 128 squares, at most twice
3 + 1 a square and 16 + 3 in adding them (27), the eps (1), half of which the inverse root
keeps, and its own (1); two products with root and gamma (2): y is off by less than
3 + 14 + 1 + 2 = 20 x 2^-24. A rotated pair c a - s b adds a product and the sum: 22 x 2^-24 of
|c a| + |s b|, less than 2^-19. The store rounds by 2^-8 of the value. In FP32 rounding, whose
product is bf16, the first term is 2^-7."""
import numpy as np
import pytest
import torch

from _gpu import note
from _int8 import bits16, int8_operands, product64
from test_gpu_qkv_proj_i8 import CASES, D, EPS, _gammas, _rope

pytestmark = pytest.mark.gpu

ONCE = 3


def _formula64(x, xs, w, ws, gammas, table, H, rot):
    """[(want, size)] of Q and K: the values in 64 bits and what their pairs add up."""
    S = x.shape[0]
    z = product64(x, xs, w, ws).view(S, 3, H, D)
    t = table[:S].double()
    c, s = t[:, None, :, 0, 0], t[:, None, :, 1, 0]
    half, res = rot // 2, []
    for i, gamma in enumerate(gammas):
        y = z[:, i]
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma.double()
        a, b, rest = y[..., :half], y[..., half:rot], y[..., rot:]
        res.append((torch.cat([c * a - s * b, s * a + c * b, rest], -1),
                    torch.cat([(c * a).abs() + (s * b).abs(), (s * a).abs() + (c * b).abs(),
                               rest.abs()], -1)))
    return res


def _check(got, formula):
    for name, t, (want, size) in zip("qk", got, formula):
        d = (t.transpose(0, 1).double() - want).abs()
        worst = float((d / (size * 2.0 ** -19 + want.abs() * 2.0 ** -8 + 1e-30)).max())
        print(f"qkv_proj_i8 once {name}: worst error / bound {worst:.3f}", flush=True)
        assert worst <= 1.0, name


# Every tile shape and odd head counts, as the other roundings are tested.
@pytest.mark.parametrize("S,K,H,rot", CASES)
def test_against_64_bits(h3, S, K, H, rot):
    """Q and K to one rounding; V the bits of the other modes; rows past S zero."""
    from h3hip import ops
    assert h3.ROUND_ONCE == ONCE
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, S + K + H)
    gammas = _gammas(S)
    table = _rope(S, rot, ONCE)[3]
    assert table.dtype == torch.float32 and torch.equal(table, _rope(S, rot, 1)[3])
    pad = (S + 127) // 128 * 128
    out = [torch.full((H, pad, D), float("nan"), dtype=torch.bfloat16, device="cuda")
           for _ in range(3)]
    note(f"qkv_proj_i8 once S={S} K={K} H={H} rot={rot}")
    q, k, v = ops.qkv_proj_i8(x, xs, w, ws, *gammas, table, heads=H, eps=EPS, rounding=ONCE, out=out)
    torch.cuda.synchronize()
    assert not any(t[:, S:].any() for t in (q, k, v))
    _check((q[:, :S], k[:, :S]), _formula64(x, xs, w, ws, gammas, table, H, rot))
    y = ops.proj_i8(x, xs, w[2 * H * D:], ws[2 * H * D:]).view(S, H, D)
    assert (bits16(v[:, :S]) == bits16(y.transpose(0, 1))).all()


@pytest.mark.parametrize("S", [1, 40, 700])
def test_rows_do_not_depend_on_the_others(h3, S):
    """A row's bits are the same alone, in a small call and in a large one: sums are exact, and
    every shape normalises and rotates a row with the same code."""
    from h3hip import ops
    H = 5
    x, xs, w, ws = int8_operands(1500, 640, 3 * H * D, 8)
    gammas, table = _gammas(8), _rope(1500, 128, ONCE)[3]
    note(f"qkv_proj_i8 once, first {S} of 1500 rows")
    run = lambda n: ops.qkv_proj_i8(x[:n], xs[:n], w, ws, *gammas, table, heads=H, rounding=ONCE)
    for a, b in zip(run(S), run(1500)):
        assert (bits16(a[:, :S]) == bits16(b[:, :S])).all()


@pytest.mark.parametrize("S,K,H", [(3, 256, 3), (300, 384, 4), (900, 384, 39), (1100, 640, 6)])
def test_padding_zeros_and_nan(h3, S, K, H):
    """Rows behind the last are zero up to a far seq_pad; a row of zeros stays zeros; a row whose
    scale is NaN is NaN in Q, K and V, and no other is."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, S)
    x[1], xs[2] = 0, float("nan")
    gammas, table = _gammas(2), _rope(S, 128, ONCE)[3]
    pad = (S + 127) // 128 * 128 + 640
    out = [torch.full((H, pad, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    note(f"qkv_proj_i8 once S={S} seq_pad={pad}")
    ops.qkv_proj_i8(x, xs, w, ws, *gammas, table, heads=H, seq_pad=pad, rounding=ONCE, out=out)
    near = ops.qkv_proj_i8(x, xs, w, ws, *gammas, table, heads=H, rounding=ONCE)
    nan = torch.zeros(S, dtype=torch.bool, device="cuda")
    nan[2] = True
    for a, b in zip(out, near):
        assert not a[:, S:].any() and not a[:, 1].any()
        assert torch.equal(torch.isnan(a[:, :S]), nan[None, :, None].expand(H, S, D))
        assert (bits16(a[:, :S]) == bits16(b[:, :S])).all()


@pytest.mark.parametrize("S", [1, 600])
def test_captured_and_replayed(h3, S):
    from h3hip import ops
    H = 3
    _, _, w, ws = int8_operands(1, 1024, 3 * H * D, 3)
    gammas, table = _gammas(3), _rope(S, 96, ONCE)[3]
    x = torch.randn((S, 1000), device="cuda").to(torch.bfloat16)
    run = lambda: ops.qkv_proj_i8(*ops.quant_rows(x), w, ws, *gammas, table, heads=H, rounding=ONCE)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note(f"qkv_proj_i8 once captured S={S}")
    with torch.cuda.graph(graph):
        got = run()
    for rep in range(4):
        x.copy_(torch.randn((S, 1000), device="cuda").to(torch.bfloat16))
        want = [bits16(t) for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all((bits16(a) == b).all() for a, b in zip(got, want)), rep


def test_layer(h3):
    """An int8 layer takes a ROUND_ONCE rotation; the bf16 projections refuse it."""
    from test_gpu_layer_int8 import _layer, _make
    from h3hip.layer import RopeState
    S, H = 300, 3
    x, wqkv, wout, qg, kg, rope = _make(S, 256, H)
    once = RopeState.build(rope.pos, rope.pair_axis, rope.pair_inv, rope.rot, ONCE)
    layer, ctx = _layer(h3, S, H, (wqkv, wout, qg, kg), projection="int8")
    note("int8 layer in ROUND_ONCE")
    from h3hip import ops
    q, k, _ = layer._project_int8(x, once, 384)
    w = layer.qkv_weight
    _check((q, k), _formula64(*ops.quant_rows(x), w.values, w.scale, (qg, kg), once.table, H,
                              once.rot))
    assert torch.isfinite(layer(x, once, ctx)).all()
    for path in ("fused", "hipblaslt"):
        other, _ = _layer(h3, S, H, (wqkv, wout, qg, kg), projection=path)
        with pytest.raises(ValueError, match="ROUND_ONCE"):
            other(x, once, ctx)
