"""AttentionLayer with projection="int8" on the GPU: activations rounded, the int8 QKV
product with norm and rotation, block-sparse attention, the int8 out-projection, run
together as a render runs them.

Each stage's input is the bits that the stage before it left, so each is held to its own
bound in 64 bits (_int8.py, test_gpu_qkv_proj_i8.py) and the layer's output to the out-projection's:
weights and activations rounded to int8 here from the definition, products, scales. How far
int8 itself is from the bf16 layer is bounded from the roundings: a code is off by half a
step, so a rounded row or channel by a relative sqrt(K / 12) s / |row| in 2-norm."""
import math

import pytest
import torch

from _gpu import note
from _int8 import bits16, check_product, quant64, to64
from test_gpu_layer import _setup

pytestmark = pytest.mark.gpu


def _make(S, hidden, H, seed=3):
    x, wqkv, wout, qg, kg, rope, H, D = _setup(S, hidden, H, seed)
    return x, wqkv, wout, qg, kg, rope


def _layer(h3, S, H, weights, **kw):
    from h3hip.backend import AttentionContext, H3HIPBackend
    from h3hip.layer import AttentionLayer
    plan = h3.TilePlan(h3.MaskRule.dense(S), heads=H)
    ctx = AttentionContext(4, 8, 0.5, S)
    return AttentionLayer(*weights, heads=H, eps=1e-6, backend=H3HIPBackend(plan), **kw), ctx


def _product64(x, w):
    """bf16 x . w^T on the codes and scales of the definition, float64 on the GPU."""
    (q, s), (wq, ws) = quant64(to64(x)), quant64(to64(w))
    t = lambda a: torch.from_numpy(a).double().cuda()
    return torch.mm(t(q), t(wq).t().contiguous()) * t(s)[:, None] * t(ws)


@pytest.mark.parametrize("S,hidden,H", [(300, 256, 2), (300, 200, 3), (917, 640, 5)])
def test_stages_and_layer(h3, S, hidden, H):
    from h3hip import ops
    x, wqkv, wout, qg, kg, rope = _make(S, hidden, H)
    layer, ctx = _layer(h3, S, H, (wqkv, wout, qg, kg), projection="int8")
    note(f"int8 layer S={S} hidden={hidden} H={H}")
    y = layer(x, rope, ctx)
    torch.cuda.synchronize()
    # V is the product itself; Q and K are the prologue of the product's bits.
    xq = ops.quant_rows(x)
    w = layer.qkv_weight
    prod = ops.proj_i8(*xq, w.values, w.scale)
    check_product(prod, _product64(x, wqkv))
    inner = H * 128
    q, k, v = layer._project_int8(x, rope, (S + 127) // 128 * 128)
    want = ops.qk_norm_rope(prod[:, :inner], prod[:, inner:2 * inner], qg, kg, rope.pos,
                            rope.pair_axis, rope.pair_inv, heads=H, eps=1e-6, rot=rope.rot,
                            v_in=prod[:, 2 * inner:])
    for got, ref in zip((q, k, v), want):
        assert (bits16(got) == bits16(ref[:, :S])).all()
    merged = layer._attend(q, k, v, ctx)
    check_product(y, _product64(merged, wout))


def test_distance_from_the_bf16_layer(h3):
    """The product of rounded operands is off by at most |dx||w| + |x||dw| + |dx||dw| a pair of
    row and channel, whatever the values."""
    x, wqkv, wout, qg, kg, rope = _make(300, 512, 2)
    (q, s), (wq, ws) = quant64(to64(x)), quant64(to64(wqkv))
    from h3hip import ops
    note("int8 product against the unrounded one")
    y = ops.proj_i8(*ops.quant_rows(x), *ops.quant_rows(wqkv)).double()
    want = torch.mm(x.double(), wqkv.double().t().contiguous())
    half = math.sqrt(512) / 2
    dx = torch.from_numpy(s).double().cuda() * half
    dw = torch.from_numpy(ws).double().cuda() * half
    nx, nw = x.double().norm(dim=1), wqkv.double().norm(dim=1)
    bound = dx[:, None] * nw + nx[:, None] * dw + dx[:, None] * dw + want.abs() * 2.0 ** -7
    assert ((y - want).abs() <= bound).all()


def test_weights_rounded_once_and_given(h3):
    """An Int8Weight given is used as it is; the layer keeps no bf16 weight; the same bits."""
    from h3hip.layer import AttentionLayer, Int8Weight
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 2)
    a, ctx = _layer(h3, 300, 2, (wqkv, wout, qg, kg), projection="int8")
    given = Int8Weight.round(wqkv), Int8Weight.round(wout)
    b, _ = _layer(h3, 300, 2, (*given, qg, kg), projection="int8")
    assert isinstance(a.qkv_weight, Int8Weight) and b.qkv_weight is given[0]
    note("int8 layer, weights given")
    assert (bits16(a(x, rope, ctx)) == bits16(b(x, rope, ctx))).all()
    assert (bits16(a(x, None, ctx)) == bits16(b(x, None, ctx))).all()
    with pytest.raises(ValueError, match="projection='int8'"):
        AttentionLayer(*given, qg, kg, heads=2)
    with pytest.raises(ValueError, match="256"):
        a(x[:, :200], rope, ctx)


def test_captured_and_replayed(h3):
    """The whole layer in one graph, replayed on new activations with eager calls between."""
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 2)
    layer, ctx = _layer(h3, 300, 2, (wqkv, wout, qg, kg), projection="int8")
    layer(x, rope, ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note("int8 layer captured")
    with torch.cuda.graph(graph):
        y = layer(x, rope, ctx)
    for rep in range(4):
        x.copy_(torch.randn_like(x, dtype=torch.float32).to(torch.bfloat16))
        want = bits16(layer(x, rope, ctx))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (bits16(y) == want).all(), rep
