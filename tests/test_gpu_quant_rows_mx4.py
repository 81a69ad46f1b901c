"""h3hip_quant_rows_mx4 and h3hip_dequant_rows_mx4 on the GPU, value for value against the
format's definition in 64 bits: every bf16 value under every scale, sizes that end inside a
block, a step or a group of rows, strides, addresses, what is written and what is not."""
import numpy as np
import pytest
import torch

from _gpu import note
from _mx4 import GRID, quant64, unpack

pytestmark = pytest.mark.gpu


def _to64(t):
    return t.double().cpu().numpy()


def _check(x, rows):
    """Codes, exponents, the zeros past the columns and the scales of what does not exist."""
    S, K = x.shape
    codes, e = quant64(_to64(x))
    got = unpack(rows.values)
    assert rows.values.shape == (S, (K + 255) // 256 * 128) and rows.cols == K
    assert (got[:, :K] == codes).all() and not got[:, K:].any()
    assert (rows.exponents().cpu().numpy() == e).all()
    every = rows.scale.cpu().numpy()
    slabs, groups = every.shape[:2]
    every = every.reshape(slabs, groups, 4, 16, 4).transpose(1, 3, 0, 4, 2).reshape(16 * groups, -1)
    assert not every[S:].any() and not every[:, e.shape[1]:].any()


def _check_values(x, rows, back):
    codes, e = quant64(_to64(x))
    want = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7] * np.ldexp(
        1.0, np.repeat(e, 32, 1)[:, :x.shape[1]] - 127)
    bad = np.repeat(e == 255, 32, 1)[:, :x.shape[1]]
    got = _to64(back)
    assert np.isnan(got[bad]).all() and (got[~bad] == want[~bad]).all()


def _rows(S, K, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((S, K), generator=g, device="cuda") * torch.exp(
        3 * torch.randn((S, K), generator=g, device="cuda"))
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("top", range(0, 255, 2))
def test_every_value_under_every_scale(h3, top):
    """Blocks of a largest magnitude of each exponent field (two a test) and 31 values of the
    whole bf16 range below it: all of them, both signs."""
    from h3hip import ops
    for field in (top, top + 1):
        if field == 255:
            continue
        head = field << 7
        below = np.arange(0, head + 128, dtype=np.int64)
        # Values of 20 binades below the largest decide a code; far smaller ones are zeros.
        below = below[max(0, len(below) - 20 * 128):]
        blocks = -(-len(below) // 31)
        bits = np.zeros((blocks, 32), dtype=np.int64)
        bits[:, 1:].flat[:len(below)] = below
        bits[:, 0] = np.maximum(bits.max(1), head)    # the exponent asked for
        x = np.concatenate([bits, bits | 0x8000]).astype(np.uint16).reshape(1, -1)
        t = torch.from_numpy(x.view(np.int16)).cuda().view(torch.bfloat16)
        if field in (0, 1, 127, 254):
            note(f"quant_rows_mx4 exponent field {field}")
        rows = ops.quant_rows_mx4(t)
        _check(t, rows)
        _check_values(t, rows, ops.dequant_rows_mx4(rows))


@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 33, 100])
@pytest.mark.parametrize("K", [1, 2, 7, 8, 31, 32, 33, 255, 256, 257, 511, 512, 513, 1001, 5120])
def test_sizes(h3, S, K):
    from h3hip import ops
    x = _rows(S, K, S * 10007 + K)
    note(f"quant_rows_mx4 S={S} K={K}")
    rows = ops.quant_rows_mx4(x)
    _check(x, rows)
    _check_values(x, rows, ops.dequant_rows_mx4(rows))


def test_no_rows(h3):
    from h3hip import ops
    rows = ops.quant_rows_mx4(torch.empty((0, 100), dtype=torch.bfloat16, device="cuda"))
    assert rows.values.shape == (0, 128) and rows.scale.shape == (1, 0, 64, 4)
    assert ops.dequant_rows_mx4(rows).shape == (0, 100)


def test_infinities_nan_and_zeros(h3):
    """A block with an infinity or a NaN is NaN as a whole, its neighbours are not."""
    from h3hip import ops
    x = _rows(40, 300, 5)
    x[0, 5], x[1, 33], x[2, 299], x[3] = float("inf"), float("-inf"), float("nan"), 0.0
    x[4, 64:96] = float("nan")
    x[5] = torch.finfo(torch.bfloat16).max
    x[6] = -torch.finfo(torch.bfloat16).max
    x[7] = 2.0 ** -133
    x[8] = -0.0
    note("quant_rows_mx4 special values")
    rows = ops.quant_rows_mx4(x)
    _check(x, rows)
    back = ops.dequant_rows_mx4(rows)
    _check_values(x, rows, back)
    nan = torch.zeros((40, 300), dtype=torch.bool)
    nan[0, :32] = nan[1, 32:64] = nan[2, 288:] = nan[4, 64:96] = True
    assert torch.equal(torch.isnan(back).cpu(), nan)


@pytest.mark.parametrize("S,K,ldx,first", [(19, 333, 400, 0), (19, 333, 337, 1), (5, 512, 1031, 3),
                                           (33, 64, 67, 7), (1, 1000, 1000, 5)])
def test_strides_and_addresses(h3, S, K, ldx, first):
    from h3hip import ops
    buf = _rows(1, S * ldx + first, 3)[0]
    x = buf[first:].as_strided((S, K), (ldx, 1))
    note(f"quant_rows_mx4 strided S={S} K={K} ldx={ldx} first={first}")
    width = (K + 255) // 256 * 128
    store = torch.full((S + 1, width + 48), 0x55, dtype=torch.uint8, device="cuda")
    plain = ops.quant_rows_mx4(x.contiguous())
    out = ops.Mx4Rows(store[:S, :width], torch.empty_like(plain.scale), K)
    got = ops.quant_rows_mx4(x, out=out)
    assert got is out
    _check(x, got)
    assert torch.equal(got.values, plain.values) and torch.equal(got.scale, plain.scale)
    assert (store[:, width:] == 0x55).all() and (store[S] == 0x55).all()
    ys = torch.full(((S + 1) * ldx + first,), 7.0, dtype=torch.bfloat16, device="cuda")
    y = ys[first:first + S * ldx].as_strided((S, K), (ldx, 1))
    _check_values(x, got, ops.dequant_rows_mx4(got, out=y))
    rest = torch.ones_like(ys, dtype=torch.bool)
    rest[first:first + S * ldx].as_strided((S, K), (ldx, 1))[:] = False
    assert (ys[rest] == 7.0).all()


def test_any_checkpoint_rows(h3):
    """pack() of random codes and exponents of the whole range: dequantised values are the
    format's, past bf16's range infinities, NaN under 255; exponents() gives them back."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    for S, n, cols in ((50, 1024, 1024), (17, 352, 333), (3, 40, 1)):
        codes = torch.randint(0, 256, (S, n // 2), generator=g, device="cuda", dtype=torch.uint8)
        e = torch.randint(0, 256, (S, -(-n // 32)), generator=g, device="cuda", dtype=torch.uint8)
        rows = ops.Mx4Rows.pack(codes, e, cols)
        nb = -(-cols // 32)
        assert torch.equal(rows.exponents(), e[:, :nb])
        c = unpack(codes)[:, :cols]
        es = np.repeat(e.cpu().numpy().astype(np.int64), 32, 1)[:, :cols]
        want = np.where(c & 8, -1.0, 1.0) * GRID[c & 7] * np.ldexp(1.0, es - 127)
        got = _to64(ops.dequant_rows_mx4(rows))
        assert np.isnan(got[es == 255]).all()
        ok = es != 255
        big = ok & (np.abs(want) > 3.4e38)
        assert (got[big] == np.sign(want[big]) * np.inf).all()
        assert (got[ok & ~big] == want[ok & ~big]).all()


@pytest.mark.parametrize("S,K", [(1_200_000, 2048), (3, 33_000_000)])
def test_offsets_past_32_bits(h3, S, K):
    """More than 2^31 elements, or the widest rows: the ends are right."""
    from h3hip import ops
    x = torch.zeros((S, K), dtype=torch.bfloat16, device="cuda")
    x[-20:, -700:] = _rows(min(S, 20), 700, 1)
    x[:20, :700] = _rows(min(S, 20), 700, 2)
    note(f"quant_rows_mx4 large S={S} K={K}")
    rows = ops.quant_rows_mx4(x)
    back = ops.dequant_rows_mx4(rows)
    k0 = K - K % 32 - 640
    for part, got in ((x[-20:, k0:], back[-20:, k0:]), (x[:20, :704], back[:20, :704])):
        _check_values(part, None, got)
    assert not back[-20:, 704:k0 - 96].any()      # between the two: zeros


def test_captured_replayed_and_on_two_streams(h3):
    from h3hip import ops
    x = _rows(100, 1000, 1)
    ops.dequant_rows_mx4(ops.quant_rows_mx4(x))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note("quant_rows_mx4 captured")
    with torch.cuda.graph(graph):
        y = ops.dequant_rows_mx4(ops.quant_rows_mx4(x))
    for rep in range(4):
        x.copy_(_rows(100, 1000, rep + 2))
        want = ops.dequant_rows_mx4(ops.quant_rows_mx4(x))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), rep
    sides = [(_rows(500, 3000, s), torch.cuda.Stream()) for s in (1, 2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (t, st) in enumerate(sides):
            with torch.cuda.stream(st):
                got[i].append(ops.quant_rows_mx4(t))
    torch.cuda.synchronize()
    for i, (t, _) in enumerate(sides):
        want = ops.quant_rows_mx4(t)
        for r in got[i]:
            assert torch.equal(r.values, want.values) and torch.equal(r.scale, want.scale)
