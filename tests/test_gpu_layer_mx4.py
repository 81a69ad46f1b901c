"""AttentionLayer with projection="mx4" and AttentionBlock on the GPU: norm and modulation, the
4-bit QKV product with norm and rotation, block-sparse attention, the 4-bit out-projection,
post-norm, gate and residual, run together as a render runs them.

Each stage's input is the bits that the stage before it left, so each is held to its own bound
in 64 bits (_mx4.py, test_gpu_qkv_proj_mx4.py, test_gpu_norm_residual.py). How far 4 bits
themselves are from the bf16 product is bounded from the roundings: with a block's largest
magnitude a and its scale s, 4 s <= a < 8 s, a value below 4 s is off by at most s / 2, one up to 6 s
by s, both at most a / 4, and one between 6 s and a by a - 6 s < a / 4."""
import pytest
import torch

from _gpu import note
from _mx4 import bits16, check_product, product64
from test_gpu_layer_int8 import _layer, _make
from test_gpu_norm_residual import _after64, _check, _norm64, _segment

pytestmark = pytest.mark.gpu


def _tables(hidden, segments, seed=5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = [(0.3 * torch.randn((segments, hidden), generator=g, device="cuda")).to(torch.bfloat16)
         for _ in range(3)]
    gam = [(1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(torch.bfloat16)
           for _ in range(2)]
    return (*t, *gam)


@pytest.mark.parametrize("S,hidden,H", [(300, 256, 2), (300, 200, 3), (917, 640, 5)])
def test_stages_and_layer(h3, S, hidden, H):
    from h3hip import ops
    x, wqkv, wout, qg, kg, rope = _make(S, hidden, H)
    layer, ctx = _layer(h3, S, H, (wqkv, wout, qg, kg), projection="mx4")
    note(f"4-bit layer S={S} hidden={hidden} H={H}")
    y = layer(x, rope, ctx)
    torch.cuda.synchronize()
    w, xq = layer.qkv_weight, ops.quant_rows_mx4(x)
    assert torch.equal(w.values, ops.quant_rows_mx4(wqkv).values)
    prod = ops.proj_mx4(xq, w)
    check_product(prod, xq, w)
    inner = H * 128
    q, k, v = layer._project_mx4(x, rope, (S + 127) // 128 * 128)
    want = ops.qk_norm_rope(prod[:, :inner], prod[:, inner:2 * inner], qg, kg, rope.pos,
                            rope.pair_axis, rope.pair_inv, heads=H, eps=1e-6, rot=rope.rot,
                            v_in=prod[:, 2 * inner:])
    for got, ref in zip((q, k, v), want):
        assert (bits16(got) == bits16(ref[:, :S])).all()
    merged = layer._attend(q, k, v, ctx)
    check_product(y, ops.quant_rows_mx4(merged), layer.out_weight)


@pytest.mark.parametrize("S", [1, 2, 5])
@pytest.mark.parametrize("rounding", [0, 3])
def test_few_tokens(h3, S, rounding):
    """A layer and a block of a few appended tokens: one launch a projection of one or two."""
    from h3hip import ops
    from h3hip.layer import AttentionBlock, Modulation, RopeState
    x, wqkv, wout, qg, kg, rope = _make(300, 264, 3)
    x = x[:S]
    rope = RopeState.build(rope.pos[-S:].contiguous(), rope.pair_axis, rope.pair_inv, rope.rot,
                           rounding)
    layer, ctx = _layer(h3, S, 3, (wqkv, wout, qg, kg), projection="mx4")
    scale, shift, gate, gamma, post_gamma = _tables(264, 1)
    block = AttentionBlock(layer, gamma, post_gamma)
    note(f"4-bit block of {S} tokens, rounding {rounding}")
    r = block(x, rope, ctx, Modulation(scale, shift, gate))
    h = ops.norm_modulate(x, gamma, scale, shift)
    q, k, v = layer._project_mx4(h, rope, 128)
    merged = layer._attend(q, k, v, ctx)
    y = ops.proj_mx4(merged, layer.out_weight)
    check_product(y, ops.quant_rows_mx4(merged), layer.out_weight)
    want = ops.gated_residual(x, y, gate, post_gamma=post_gamma)
    assert (bits16(r) == bits16(want)).all()


def test_distance_from_the_bf16_product(h3):
    """The product of rounded operands is off by at most |dx||w| + |x||dw| + |dx||dw| a pair of
    row and channel, whatever the values."""
    from h3hip import ops
    x, wqkv, *_ = _make(300, 512, 2)
    note("4-bit product against the unrounded one")
    y = ops.proj_mx4(x, wqkv_q := ops.quant_rows_mx4(wqkv)).double()
    want = torch.mm(x.double(), wqkv.double().t().contiguous())

    def off(t):
        top = t.double().view(t.shape[0], -1, 32).abs().amax(-1)
        return (32 * (top / 4).square()).sum(1).sqrt()
    dx, dw, nx, nw = off(x), off(wqkv), x.double().norm(dim=1), wqkv.double().norm(dim=1)
    bound = dx[:, None] * nw + nx[:, None] * dw + dx[:, None] * dw
    assert ((y - want).abs() <= bound * 1.01 + want.abs() * 2.0 ** -7).all()
    assert wqkv_q.cols == 512


def test_weights_rounded_once_and_given(h3):
    from h3hip import ops
    from h3hip.layer import AttentionLayer
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 2)
    a, ctx = _layer(h3, 300, 2, (wqkv, wout, qg, kg), projection="mx4")
    given = ops.quant_rows_mx4(wqkv), ops.quant_rows_mx4(wout)
    b, _ = _layer(h3, 300, 2, (*given, qg, kg), projection="mx4")
    assert isinstance(a.qkv_weight, ops.Mx4Rows) and b.qkv_weight is given[0]
    note("4-bit layer, weights given")
    assert (bits16(a(x, rope, ctx)) == bits16(b(x, rope, ctx))).all()
    assert (bits16(a(x, None, ctx)) == bits16(b(x, None, ctx))).all()
    with pytest.raises(ValueError, match="projection='mx4'"):
        AttentionLayer(*given, qg, kg, heads=2)
    with pytest.raises(ValueError, match="256"):
        a(x[:, :200], rope, ctx)


@pytest.mark.parametrize("projection", ["mx4", "int8", "fused"])
@pytest.mark.parametrize("post", [False, True])
def test_block_stage_by_stage(h3, projection, post):
    """Around any projection: h of x, the layer's own output of h, r and the next h of both."""
    from h3hip.layer import AttentionBlock, Modulation
    S, hidden, H = 300, 256, 2
    x, wqkv, wout, qg, kg, rope = _make(S, hidden, H)
    layer, ctx = _layer(h3, S, H, (wqkv, wout, qg, kg), projection=projection)
    scale, shift, gate, gamma, post_gamma = _tables(hidden, 3)
    block = AttentionBlock(layer, gamma, post_gamma if post else None, residual_scale=0.875)
    starts, nxt = [0, 40, 57], dict(gamma=post_gamma, scale=shift, shift=scale)
    note(f"block projection={projection} post={post}")
    r, h = block(x, rope, ctx, Modulation(scale, shift, gate), segments=starts, next_norm=nxt)
    from h3hip import ops
    pre = ops.norm_modulate(x, gamma, scale, shift, segments=starts, eps=1e-6)
    seg = _segment(S, starts)
    want, bound = _norm64(x.double(), torch.zeros_like(x, dtype=torch.float64),
                          dict(gamma=gamma, scale=scale, shift=shift), seg)
    _check("h", pre, want, bound)
    y = layer(pre, rope, ctx)
    want, d = _after64(x, y, dict(post=post_gamma, gate=gate), 0.875, post, seg)
    _check("r", r, want, d + 2.0 ** -8 * want.abs() + 2.0 ** -133)
    _check("next h", h, *_norm64(want, d, nxt, seg))
    # The next half on what this one normed for it.
    again = block(r, rope, ctx, Modulation(shift, scale, gate), segments=starts, normed=h)
    direct = ops.gated_residual(r, layer(h, rope, ctx), gate,
                                post_gamma=post_gamma if post else None, residual_scale=0.875,
                                segments=starts)
    assert (bits16(again) == bits16(direct)).all()


def test_block_without_modulation(h3):
    from h3hip import ops
    from h3hip.layer import AttentionBlock
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 2)
    layer, ctx = _layer(h3, 300, 2, (wqkv, wout, qg, kg), projection="mx4")
    note("block without modulation")
    r = AttentionBlock(layer)(x, rope, ctx)
    want = ops.gated_residual(x, layer(ops.norm_modulate(x), rope, ctx))
    assert (bits16(r) == bits16(want)).all()


def test_block_captured_and_replayed(h3):
    """The whole half of a block in one graph, replayed on new inputs with eager calls between."""
    from h3hip.layer import AttentionBlock, Modulation
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 2)
    layer, ctx = _layer(h3, 300, 2, (wqkv, wout, qg, kg), projection="mx4")
    scale, shift, gate, gamma, post_gamma = _tables(256, 2)
    block = AttentionBlock(layer, gamma, post_gamma)

    def run():
        return block(x, rope, ctx, Modulation(scale, shift, gate), segments=[0, 100])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note("4-bit block captured")
    with torch.cuda.graph(graph):
        r = run()
    for rep in range(4):
        x.copy_(torch.randn_like(x, dtype=torch.float32).to(torch.bfloat16))
        want = bits16(run())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (bits16(r) == want).all(), rep


def test_round_once(h3):
    """A 4-bit layer takes a ROUND_ONCE rotation."""
    from h3hip.layer import RopeState
    x, wqkv, wout, qg, kg, rope = _make(300, 256, 3)
    once = RopeState.build(rope.pos, rope.pair_axis, rope.pair_inv, rope.rot, 3)
    layer, ctx = _layer(h3, 300, 3, (wqkv, wout, qg, kg), projection="mx4")
    note("4-bit layer in ROUND_ONCE")
    from test_gpu_qkv_proj_mx4 import _formula64
    from h3hip import ops
    q, k, _ = layer._project_mx4(x, once, 384)
    xq = ops.quant_rows_mx4(x)
    z = product64(xq, layer.qkv_weight).view(300, 3, 3, 128)
    from _mx4 import decode64
    size = torch.mm(decode64(xq).abs(), decode64(layer.qkv_weight).abs().t().contiguous())
    # The sums are not exact here: each is off by K / 16 * 2^-23 of its magnitudes' sum.
    slack = (size * (256 / 16 * 2.0 ** -23)).view(300, 3, 3, 128)
    for i, (t, (want, mag)) in enumerate(zip((q, k), _formula64(z, (qg, kg), once.table, once.rot))):
        rms = z[:, i].square().mean(-1, keepdim=True).sqrt()
        # A head's values and its root mean square are off by the largest of its sums' errors.
        drift = 4 * slack[:, i].amax(-1, keepdim=True) / rms * 2 * (1 + z[:, i].abs().amax(-1, keepdim=True) / rms)
        d = (t.transpose(0, 1).double() - want).abs()
        assert (d <= mag * 2.0 ** -19 + drift + want.abs() * 2.0 ** -8).all()
    assert torch.isfinite(layer(x, once, ctx)).all()
