"""h3hip_qkv_proj_i8 on the GPU.

- Q and K are, bit for bit, h3hip_qk_norm_rope of h3hip_proj_i8's result on the same
  operands, V is that result head-major: both roundings, both rotary widths, odd head
  counts, one row to several tiles, rows past seq_len zero.
- FP32 rounding against the formula in 64 bits. The product z is rounded to bf16
  (2^-8 relative), so its root mean square is off by at most 2^-8 too and a normalised
  channel by 2^-7 and a term of second order; a rotated pair c a - s b by that of
  |c a| + |s b|, and the store rounds by 2^-8. The fp32 arithmetic between (sums of 128
  squares, the inverse root, three products, a sum) adds less than 2^-16."""
import numpy as np
import pytest
import torch

from _gpu import note
from _int8 import bits16, int8_operands, product64

pytestmark = pytest.mark.gpu

D, EPS = 128, 1e-6


def _rope(S, rot, rounding, seed=0):
    from h3hip import ops
    pos = torch.from_numpy(np.random.default_rng(seed).uniform(0, 60, (S, 3)).astype(np.float32)).cuda()
    dims = (32, 48, 48) if rot == 128 else (32, 32, 32)
    ax, inv = (torch.from_numpy(a).cuda() for a in ops.rope_pairs_axes(10000.0, dims))
    return pos, ax, inv, ops.rope_table(pos, ax, inv, rounding=rounding)


def _gammas(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [(0.8 + 0.4 * torch.rand(D, generator=g, device="cuda")).to(torch.bfloat16)
            for _ in range(2)]


# One size for each tile shape (rows, hidden, heads, rot); test_proj_i8_tile_host.py
# checks which shape each one takes.
SHAPES = [("256x256", 1000, 384, 40, 128), ("256x224", 801, 256, 40, 96),
          ("256x192", 641, 384, 40, 96), ("256x160", 1000, 256, 24, 128),
          ("256x128", 385, 384, 40, 96), ("128x192", 500, 128, 24, 96),
          ("128x160", 257, 128, 40, 128), ("128x128", 129, 640, 40, 96),
          ("128x128p", 129, 128, 40, 128), ("128x64p", 65, 128, 40, 96),
          ("128x32p", 1, 128, 1, 96)]
# Odd head counts on tiles of 256 channels: the tiles between Q and K and between K and V
# hold a head of each, the last one a single head.
ODD_HEADS = [(900, 384, 39, 128), (2500, 256, 13, 96), (650, 384, 39, 96), (900, 256, 25, 128),
             (385, 384, 41, 96), (4000, 256, 1, 128)]
CASES = [s[1:] for s in SHAPES] + ODD_HEADS
CASES += [(1, 128, 1, 128), (1, 5120, 40, 128), (5, 256, 3, 96), (16, 384, 2, 128),
         (17, 640, 2, 96), (33, 128, 5, 128), (65, 1152, 4, 96), (128, 256, 1, 96),
         (129, 512, 4, 128), (300, 1024, 7, 128), (637, 5120, 40, 128), (1151, 5376, 56, 96),
         (700, 1152, 40, 128), (2100, 256, 6, 128)]


@pytest.mark.parametrize("S,K,H,rot", CASES)
@pytest.mark.parametrize("rounding", [0, 1])
def test_equals_the_prologue_of_its_product(h3, S, K, H, rot, rounding):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, S + K + H)
    gq, gk = _gammas(S)
    pos, ax, inv, table = _rope(S, rot, rounding)
    inner, pad = H * D, (S + 127) // 128 * 128
    note(f"qkv_proj_i8 S={S} K={K} H={H} rot={rot} rounding={rounding}")
    y = ops.proj_i8(x, xs, w, ws)
    out = [torch.full((H, pad, D), float("nan"), dtype=torch.bfloat16, device="cuda")
           for _ in range(3)]
    q, k, v = ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, eps=EPS, rounding=rounding,
                              out=out)
    want = ops.qk_norm_rope(y[:, :inner], y[:, inner:2 * inner], gq, gk, pos, ax, inv, heads=H,
                            eps=EPS, rot=rot, rounding=rounding, v_in=y[:, 2 * inner:])
    torch.cuda.synchronize()
    for name, got, ref in zip("qkv", (q, k, v), want):
        assert (bits16(got) == bits16(ref)).all(), name


@pytest.mark.parametrize("S,K,H", [(3, 256, 3), (300, 640, 4), (1500, 256, 2)])
def test_plain_product_head_major(h3, S, K, H):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, 7)
    note(f"qkv_proj_i8 plain S={S} K={K} H={H}")
    y = ops.proj_i8(x, xs, w, ws).view(S, 3, H, D)
    for i, got in enumerate(ops.qkv_proj_i8(x, xs, w, ws, heads=H)):
        assert (bits16(got[:, :S]) == bits16(y[:, i].transpose(0, 1))).all()
        assert not got[:, S:].any()


@pytest.mark.parametrize("S,K,H,rot", [(1, 128, 2, 128), (40, 640, 3, 96), (300, 1024, 4, 128),
                                       (900, 256, 8, 96)])
def test_fp32_rounding_against_64_bits(h3, S, K, H, rot):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, 3 * S + K)
    gq, gk = _gammas(5)
    _, _, _, table = _rope(S, rot, 1)
    note(f"qkv_proj_i8 fp32 S={S} K={K} H={H} rot={rot}")
    got = ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, eps=EPS, rounding=1)
    z = product64(x, xs, w, ws).view(S, 3, H, D)
    t = table.double()
    c, s = t[:, None, :, 0, 0], t[:, None, :, 1, 0]
    half = rot // 2
    for i, gamma in enumerate((gq, gk)):
        y = z[:, i]
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma.double()
        a, b, rest = y[..., :half], y[..., half:rot], y[..., rot:]
        want = torch.cat([c * a - s * b, s * a + c * b, rest], -1)
        size = torch.cat([(c * a).abs() + (s * b).abs(), (s * a).abs() + (c * b).abs(),
                          rest.abs()], -1)
        d = (got[i][:, :S].transpose(0, 1).double() - want).abs()
        bound = size * (2.0 ** -7 * 1.01 + 2.0 ** -16) + want.abs() * 2.0 ** -8 + 1e-30
        worst = float((d / bound).max())
        print(f"qkv_proj_i8 {'qk'[i]}: worst error / bound {worst:.3f}", flush=True)
        assert worst <= 1.0


@pytest.mark.parametrize("S,H", [(3, 2), (300, 3), (1000, 39)])
def test_scales_at_any_address(h3, S, H):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, 256, 3 * H * D, S)
    gq, gk = _gammas(4)
    table = _rope(S, 96, 1)[3]
    odd_x, odd_w = torch.zeros(S + 1, device="cuda")[1:], torch.zeros(3 * H * D + 3, device="cuda")[3:]
    odd_x.copy_(xs), odd_w.copy_(ws)
    note(f"qkv_proj_i8 scales at odd addresses S={S} H={H}")
    want = ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, rounding=1)
    got = ops.qkv_proj_i8(x, odd_x, w, odd_w, gq, gk, table, heads=H, rounding=1)
    for a, b in zip(got, want):
        assert (bits16(a) == bits16(b)).all()


def test_more_padding_than_a_tile(h3):
    """seq_pad may lie far behind seq_len: every row between is zero, in all three parts."""
    from h3hip import ops
    for S, K, H in ((3, 256, 3), (300, 384, 4), (1100, 640, 6), (900, 384, 39)):
        x, xs, w, ws = int8_operands(S, K, 3 * H * D, S)
        gq, gk = _gammas(2)
        table = _rope(S, 128, 1)[3]
        pad = (S + 127) // 128 * 128 + 640
        out = [torch.full((H, pad, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        note(f"qkv_proj_i8 S={S} seq_pad={pad}")
        ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, seq_pad=pad, rounding=1, out=out)
        near = ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, rounding=1)
        for a, b in zip(out, near):
            assert not a[:, S:].any()
            assert (bits16(a[:, :S]) == bits16(b[:, :S])).all()


def test_rows_of_zeros_and_nan(h3):
    """A row of zeros normalises to zeros; a row whose scale is NaN is NaN in Q, K and V
    and leaves the others alone."""
    from h3hip import ops
    S, K, H = 40, 256, 2
    x, xs, w, ws = int8_operands(S, K, 3 * H * D, 11)
    gq, gk = _gammas(1)
    table = _rope(S, 128, 0)[3]
    clean = ops.qkv_proj_i8(x, xs, w, ws, gq, gk, table, heads=H, eps=EPS)
    x2, xs2 = x.clone(), xs.clone()
    x2[3], xs2[9] = 0, float("nan")
    note("qkv_proj_i8 rows of zeros and NaN")
    got = ops.qkv_proj_i8(x2, xs2, w, ws, gq, gk, table, heads=H, eps=EPS)
    keep = [i for i in range(S) if i not in (3, 9)]
    for a, b in zip(got, clean):
        assert not a[:, 3].any() and torch.isnan(a[:, 9]).all()
        assert (bits16(a[:, keep]) == bits16(b[:, keep])).all()
