"""h3hip_qkv_proj_mx4 on the GPU.

- REFERENCE and FP32 rounding: Q and K are, bit for bit, h3hip_qk_norm_rope of
  h3hip_proj_mx4's result on the same operands, V is that result head-major: both rotary
  widths, odd head counts, one row to several tiles, rows past seq_len zero.
- ROUND_ONCE against the formula in 64 bits, on operands whose sums are exact in fp32
  (_mx4.py). Of what is rounded to fp32 (2^-24 each, relative): a sum of 128 squares, at most 1 a
  square and 16 + 3 in adding them (20), the eps (1), half of which the inverse root keeps, and its
  own (1); two products with root and gamma (2): y is off by less than 11 + 1 + 2 = 14 x 2^-24. A
  rotated pair c a - s b adds a product and the sum: 16 x 2^-24 of |c a| + |s b|, less than
  2^-19. The store rounds by 2^-8 of the value."""
import pytest
import torch

from _gpu import note
from _mx4 import bits16, check_exact, mx4_operand, product64
from test_gpu_qkv_proj_i8 import D, EPS, _gammas, _rope

pytestmark = pytest.mark.gpu

ONCE = 3

# One size for each tile shape (rows, hidden, heads, rot); test_proj_mx4_tile_host.py
# checks which shape each one takes.
SHAPES = [("256x256", 1000, 768, 40, 128), ("256x224", 641, 256, 45, 96),
          ("256x192", 1301, 256, 24, 128), ("256x160", 385, 256, 48, 96),
          ("256x128", 201, 5120, 43, 128), ("128x192", 1301, 512, 12, 96),
          ("128x160", 257, 512, 36, 128), ("128x128", 100, 1792, 43, 96),
          ("128x128p", 201, 256, 31, 128), ("128x64p", 33, 256, 36, 96), ("128x32p", 1, 256, 1, 128)]
# Odd head counts on tiles of 256 channels: the tiles between Q and K and between K and V
# hold a head of each, the last one a single head.
ODD_HEADS = [(1000, 768, 41, 128), (641, 256, 45, 96), (1301, 512, 23, 128), (385, 256, 49, 96),
             (201, 5120, 43, 128)]
CASES = [s[1:] for s in SHAPES] + ODD_HEADS
CASES += [(1000, 768, 40, 96), (641, 512, 45, 128), (1301, 256, 24, 96), (385, 256, 48, 128),
          (201, 5120, 43, 96), (1301, 512, 12, 128), (257, 512, 36, 96), (100, 1792, 43, 128),
          (201, 256, 31, 96), (33, 256, 36, 128), (1, 256, 1, 96), (650, 768, 39, 96), (4000, 512, 1, 128),
         (1, 256, 1, 128), (1, 5120, 40, 128), (5, 512, 3, 96), (16, 768, 2, 128),
         (17, 1280, 2, 96), (33, 256, 5, 128), (65, 2304, 4, 96), (128, 512, 1, 96),
         (129, 1000, 4, 128), (300, 2048, 7, 128), (637, 5120, 40, 128), (1151, 5376, 56, 96),
         (700, 2304, 40, 128), (2100, 512, 6, 128), (2, 33, 7, 96), (31, 1001, 3, 128)]


def _nan_out(H, pad):
    return [torch.full((H, pad, D), float("nan"), dtype=torch.bfloat16, device="cuda")
            for _ in range(3)]


@pytest.mark.parametrize("S,K,H,rot", CASES)
@pytest.mark.parametrize("rounding", [0, 1])
def test_equals_the_prologue_of_its_product(h3, S, K, H, rot, rounding):
    from h3hip import ops
    x, w = mx4_operand(S, K, S + K, -20, 40), mx4_operand(3 * H * D, K, S + H, -20, 40)
    gq, gk = _gammas(S)
    pos, ax, inv, table = _rope(S, rot, rounding)
    inner, pad = H * D, (S + 127) // 128 * 128
    note(f"qkv_proj_mx4 S={S} K={K} H={H} rot={rot} rounding={rounding}")
    y = ops.proj_mx4(x, w)
    q, k, v = ops.qkv_proj_mx4(x, w, gq, gk, table, heads=H, eps=EPS, rounding=rounding,
                               out=_nan_out(H, pad))
    want = ops.qk_norm_rope(y[:, :inner], y[:, inner:2 * inner], gq, gk, pos, ax, inv, heads=H,
                            eps=EPS, rot=rot, rounding=rounding, v_in=y[:, 2 * inner:])
    torch.cuda.synchronize()
    for name, got, ref in zip("qkv", (q, k, v), want):
        assert (bits16(got) == bits16(ref)).all(), name


def _formula64(z, gammas, table, rot):
    """[(want, size)] of Q and K [S, H, D]: values in 64 bits and what their pairs add up."""
    t = table[:z.shape[0]].double()
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


def _check_once(got, z, gammas, table, rot):
    for name, t, (want, size) in zip("qk", got, _formula64(z, gammas, table, rot)):
        d = (t.transpose(0, 1).double() - want).abs()
        worst = float((d / (size * 2.0 ** -19 + want.abs() * 2.0 ** -8 + 1e-30)).max())
        print(f"qkv_proj_mx4 once {name}: worst error / bound {worst:.3f}", flush=True)
        assert worst <= 1.0, name


@pytest.mark.parametrize("S,K,H,rot", CASES)
def test_one_rounding_against_64_bits(h3, S, K, H, rot):
    from h3hip import ops
    x, w = mx4_operand(S, K, S + K), mx4_operand(3 * H * D, K, S + H)
    gammas, table = _gammas(S), _rope(S, rot, ONCE)[3]
    pad = (S + 127) // 128 * 128
    note(f"qkv_proj_mx4 once S={S} K={K} H={H} rot={rot}")
    q, k, v = ops.qkv_proj_mx4(x, w, *gammas, table, heads=H, eps=EPS, rounding=ONCE,
                               out=_nan_out(H, pad))
    torch.cuda.synchronize()
    assert not any(t[:, S:].any() for t in (q, k, v))
    z = product64(x, w).view(S, 3, H, D)
    _check_once((q[:, :S], k[:, :S]), z, gammas, table, rot)
    check_exact(v[:, :S].transpose(0, 1), z[:, 2])


@pytest.mark.parametrize("S,K,H", [(1, 5120, 40), (3, 1001, 3), (16, 768, 5), (17, 512, 2),
                                   (300, 333, 4), (1151, 1280, 3)])
@pytest.mark.parametrize("rounding", [0, 1, 3])
def test_bf16_rows_are_rounded_on_the_way(h3, S, K, H, rounding):
    """Of bf16 rows: V, whose sums are exact here, to the bit; Q and K as of the 4-bit form."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(S + K)
    # Whole numbers up to 8, one of them 4 at least in every block: exponents 0 and 1.
    x = torch.randint(-8, 9, (S, K), generator=g, device="cuda").to(torch.bfloat16)
    x[:, ::32] = 4.0
    w = mx4_operand(3 * H * D, K, 5)
    gammas, table = _gammas(3), _rope(S, 96, rounding)[3]
    note(f"qkv_proj_mx4 of bf16 rows S={S} K={K} H={H} rounding={rounding}")
    got = ops.qkv_proj_mx4(x, w, *gammas, table, heads=H, eps=EPS, rounding=rounding)
    q = ops.quant_rows_mx4(x)
    want = ops.qkv_proj_mx4(q, w, *gammas, table, heads=H, eps=EPS, rounding=rounding)
    z = product64(q, w).view(S, 3, H, D)
    check_exact(got[2][:, :S].transpose(0, 1), z[:, 2])
    assert not any(t[:, S:].any() for t in got)
    if rounding == ONCE:
        _check_once([t[:, :S] for t in got[:2]], z, gammas, table, 96)
    else:
        for a, b in zip(got, want):
            assert (bits16(a) == bits16(b)).all()


@pytest.mark.parametrize("S", [1, 2, 3])
@pytest.mark.parametrize("K,H,rot", [(8, 1, 128), (264, 3, 96), (1000, 5, 128), (5376, 7, 96),
                                     (10248, 2, 128)])
def test_one_and_two_bf16_rows(h3, S, K, H, rot):
    """Every rounding and the plain product, on whole numbers (exact sums): the bits of the 4-bit
    form's call, whichever way the sums were added, and zeros up to a far seq_pad."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(S + K)
    x = torch.randint(-8, 9, (S, K), generator=g, device="cuda").to(torch.bfloat16)
    w = mx4_operand(3 * H * D, K, H)
    q, gammas = ops.quant_rows_mx4(x), _gammas(K)
    size = product64(q._replace(values=q.values & 0x77), w._replace(values=w.values & 0x77))
    assert float(4 * size.max()) < 2 ** 24      # any partial sum is exact in fp32
    for rounding in (0, 1, ONCE):
        args = (*gammas, _rope(S, rot, rounding)[3])
        note(f"qkv_proj_mx4 of {S} bf16 rows K={K} H={H} rot={rot} rounding={rounding}")
        out = [torch.full((H, 384, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        got = ops.qkv_proj_mx4(x, w, *args, heads=H, eps=EPS, rounding=rounding, out=out, seq_pad=384)
        want = ops.qkv_proj_mx4(q, w, *args, heads=H, eps=EPS, rounding=rounding)
        for a, b in zip(got, want):
            assert (bits16(a[:, :128]) == bits16(b)).all() and not a[:, S:].any()
    for a, b in zip(ops.qkv_proj_mx4(x, w, heads=H), ops.qkv_proj_mx4(q, w, heads=H)):
        assert (bits16(a) == bits16(b)).all()


@pytest.mark.parametrize("S,K,H", [(3, 512, 3), (300, 1280, 4), (1500, 512, 2)])
def test_plain_product_head_major(h3, S, K, H):
    from h3hip import ops
    x, w = mx4_operand(S, K, 7), mx4_operand(3 * H * D, K, 8)
    note(f"qkv_proj_mx4 plain S={S} K={K} H={H}")
    y = ops.proj_mx4(x, w).view(S, 3, H, D)
    for i, got in enumerate(ops.qkv_proj_mx4(x, w, heads=H)):
        assert (bits16(got[:, :S]) == bits16(y[:, i].transpose(0, 1))).all()
        assert not got[:, S:].any()


@pytest.mark.parametrize("S", [1, 40, 700])
def test_rows_do_not_depend_on_the_others(h3, S):
    from h3hip import ops
    H = 5
    x, w = mx4_operand(1500, 1280, 8, -20, 40), mx4_operand(3 * H * D, 1280, 9, -20, 40)
    gammas, table = _gammas(8), _rope(1500, 128, ONCE)[3]
    some = ops.Mx4Rows(x.values[:S], x.scale[:, :(S + 15) // 16].contiguous(), x.cols)
    note(f"qkv_proj_mx4 once, first {S} of 1500 rows")
    for a, b in zip(*(ops.qkv_proj_mx4(r, w, *gammas, table, heads=H, rounding=ONCE)
                      for r in (some, x))):
        assert (bits16(a[:, :S]) == bits16(b[:, :S])).all()


@pytest.mark.parametrize("S,K,H", [(3, 512, 3), (300, 768, 4), (900, 768, 39), (1100, 1280, 6)])
@pytest.mark.parametrize("rounding", [0, 1, 3])
def test_padding_zeros_and_nan(h3, S, K, H, rounding):
    """Rows behind the last are zero up to a far seq_pad; a row of zeros stays zeros; a row with
    a NaN block is NaN in Q, K and V, and no other is. From 4-bit and from bf16 rows."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(S)
    xb = torch.randn((S, K), generator=g, device="cuda").to(torch.bfloat16)
    xb[1], xb[2, K - 1] = 0, float("nan")
    w = mx4_operand(3 * H * D, K, S)
    gammas, table = _gammas(2), _rope(S, 128, rounding)[3]
    pad = (S + 127) // 128 * 128 + 640
    for x in (ops.quant_rows_mx4(xb), xb):
        out = [torch.full((H, pad, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        note(f"qkv_proj_mx4 S={S} seq_pad={pad} rounding={rounding} of {type(x).__name__}")
        ops.qkv_proj_mx4(x, w, *gammas, table, heads=H, seq_pad=pad, rounding=rounding, out=out)
        near = ops.qkv_proj_mx4(x, w, *gammas, table, heads=H, rounding=rounding)
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
    w = mx4_operand(3 * H * D, 1000, 3, -3, 6)
    gammas, table = _gammas(3), _rope(S, 96, ONCE)[3]
    x = torch.randn((S, 1000), device="cuda").to(torch.bfloat16)

    def run():
        return ops.qkv_proj_mx4(x, w, *gammas, table, heads=H, rounding=ONCE)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note(f"qkv_proj_mx4 once captured S={S}")
    with torch.cuda.graph(graph):
        got = run()
    for rep in range(4):
        x.copy_(torch.randn((S, 1000), device="cuda").to(torch.bfloat16))
        want = [bits16(t) for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all((bits16(a) == b).all() for a, b in zip(got, want)), rep
