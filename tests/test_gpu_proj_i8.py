"""h3hip_proj_i8 on the GPU: the int8 product with scales for each token and channel,
against the same product in 64 bits, for one row to several thousand, odd widths,
strides and alignments, the whole range of values, and what it may not write."""
import pytest
import torch

from _gpu import note
from _int8 import bits16, check_product, int8_operands, product64

pytestmark = pytest.mark.gpu

# One size for each tile shape (rows, in, out), with rows and channels that end inside a
# tile; test_proj_i8_tile_host.py checks which shape each one takes.
SHAPES = [("256x256", 6001, 1024, 5000), ("256x224", 2500, 256, 5000), ("256x192", 2001, 384, 5000),
          ("256x160", 2500, 256, 3500), ("256x128", 641, 384, 9000), ("128x192", 500, 128, 9000),
          ("128x160", 801, 128, 5000), ("128x128", 385, 640, 5000), ("128x128p", 385, 128, 5000),
          ("128x64p", 100, 128, 9000), ("128x32p", 1, 128, 9000), ("64x64p", 1, 256, 9000),
          ("32x64p", 33, 128, 5000), ("32x32p", 1, 128, 100)]


@pytest.mark.parametrize("S,K,N", [
    (1, 128, 1), (1, 128, 16), (1, 5120, 5120), (2, 128, 17), (15, 256, 128), (16, 384, 130),
    (17, 384, 33), (31, 640, 127), (33, 128, 777), (64, 1152, 512), (65, 2048, 129),
    (125, 5120, 5120), (129, 256, 640), (130, 640, 256), (255, 896, 1000), (300, 1152, 520),
    (637, 1024, 777), (917, 5120, 5120), (1151, 7168, 5376), (2048, 256, 5120), (4100, 512, 700)])
def test_against_64_bits(h3, S, K, N):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, N, S + K + N)
    note(f"proj_i8 S={S} K={K} N={N}")
    y = ops.proj_i8(x, xs, w, ws)
    torch.cuda.synchronize()
    assert y.shape == (S, N) and y.dtype == torch.bfloat16
    check_product(y, product64(x, xs, w, ws))


@pytest.mark.parametrize("shape,S,K,N", SHAPES, ids=[s[0] for s in SHAPES])
def test_every_tile_shape(h3, shape, S, K, N):
    """At two lengths of reduction that take it, into rows that are and are not on 16 bytes;
    nothing past a row's channels or the last row is written."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, N, S + N)
    want = product64(x, xs, w, ws)
    for ldy, first in ((N + 8 - N % 8, 0), (N + 3, 1)):
        buf = torch.full(((S + 1) * ldy + first,), 7.0, dtype=torch.bfloat16, device="cuda")
        rows = buf[first:].view(S + 1, ldy)
        note(f"proj_i8 {shape} S={S} K={K} N={N} ldy={ldy}")
        check_product(ops.proj_i8(x, xs, w, ws, out=rows[:S, :N]), want)
        assert (rows[S] == 7.0).all() and (rows[:, N:] == 7.0).all() and (buf[:first] == 7.0).all()


@pytest.mark.parametrize("S,K,N,ldx,ldw,ldy,first", [
    (70, 256, 130, 272, 400, 136, 0),     # strided operands; rows of y on 16 bytes
    (70, 256, 130, 256, 256, 131, 0),     # odd row stride
    (300, 384, 512, 400, 384, 520, 8),    # wide output, gap behind each row
    (300, 384, 515, 384, 384, 520, 3),    # a base that is not on 16 bytes
    (5, 128, 64, 144, 160, 64, 1)])
def test_strides_and_what_is_not_written(h3, S, K, N, ldx, ldw, ldy, first):
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, K, N, S + N, ldx, ldw)
    buf = torch.full(((S + 2) * ldy + first,), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = buf[first:].view(S + 2, ldy)
    note(f"proj_i8 strided S={S} K={K} N={N} ldy={ldy} first={first}")
    y = ops.proj_i8(x, xs, w, ws, out=rows[1:S + 1, :N])
    torch.cuda.synchronize()
    check_product(y, product64(x, xs, w, ws))
    assert (rows[0] == 7.0).all() and (rows[S + 1] == 7.0).all() and (rows[:, N:] == 7.0).all()
    assert (buf[:first] == 7.0).all()


def test_largest_sums(h3):
    """130,944 products of -128 x -128 and of -128 x 127: the largest sums of either sign."""
    from h3hip import ops
    K = 130944
    for S, N in ((3, 20), (200, 300)):
        x = torch.full((S, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
        w[1::2] = 127
        xs, ws = torch.ones(S, device="cuda"), torch.ones(N, device="cuda")
        note(f"proj_i8 largest sums S={S} N={N}")
        check_product(ops.proj_i8(x, xs, w, ws), product64(x, xs, w, ws))


@pytest.mark.parametrize("S", [3, 300])
def test_scales_that_are_zero_or_nan(h3, S):
    """A zero scale gives zeros; a NaN scale makes its whole row (or channel) NaN and
    nothing else."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, 256, 200, 4)
    xs[0], xs[1], ws[5], ws[6] = 0.0, float("nan"), 0.0, float("nan")
    note(f"proj_i8 special scales S={S}")
    y = ops.proj_i8(x, xs, w, ws)
    nan = torch.zeros((S, 200), dtype=torch.bool, device="cuda")
    nan[1], nan[:, 6] = True, True
    assert torch.equal(torch.isnan(y), nan)
    assert not y[0, :6].any() and not y[2:, 5].any()
    check_product(torch.where(nan, 0, y), product64(x, xs, w, ws).masked_fill(nan, 0.0))


@pytest.mark.parametrize("S", [2, 300])
def test_scales_at_the_ends_of_fp32(h3, S):
    """A token's scale of any magnitude with a weight's: only the result's own overflow and
    underflow show. (sum * w_scale stays in fp32's range: at most 2^31 * 0.1.)"""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, 512, 300, 5)
    xs[0], xs[1] = 3.0e38, 1.5e-38
    note(f"proj_i8 extreme scales S={S}")
    y = ops.proj_i8(x, xs, w, ws)
    want = product64(x, xs, w, ws)
    top = torch.finfo(torch.bfloat16).max
    over = want.abs() > top * 1.01
    assert torch.isinf(y[over]).all() and (torch.sign(y[over]) == torch.sign(want[over])).all()
    near = (want.abs() > top * 0.99) | over
    check_product(torch.where(near, 0, y), want.masked_fill(near, 0.0))


def test_a_single_row_of_any_stride(h3):
    """One row has no row stride: whatever its tensor says is taken."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(1, 256, 100, 6)
    odd = torch.as_strided(x, (1, 256), (1000003, 1))
    y = torch.empty((40,) * 3, dtype=torch.bfloat16, device="cuda").view(-1)[8:108]
    note("proj_i8 single rows")
    want = bits16(ops.proj_i8(x, xs, w, ws))
    got = ops.proj_i8(odd, xs, w, ws, out=torch.as_strided(y, (1, 100), (3, 1)))
    assert (bits16(got) == want).all()
    b = torch.randn((1, 777), device="cuda").to(torch.bfloat16)
    q, s = ops.quant_rows(b)
    q2, s2 = ops.quant_rows(torch.as_strided(b, (1, 777), (5, 1)))
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("first,S,N", [(1, 3, 100), (3, 300, 517), (2, 700, 640), (5, 1500, 4000)])
def test_some_rows_of_a_weight(h3, first, S, N):
    """A weight's rows from any one on, with their scales: those channels' bits."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(S, 256, N + 9, N)
    note(f"proj_i8 channels {first}.. of {N + 9}, S={S}")
    every = bits16(ops.proj_i8(x, xs, w, ws))
    some = bits16(ops.proj_i8(x, xs, w[first:first + N], ws[first:first + N]))
    assert (some == every[:, first:first + N]).all()


def test_no_rows(h3):
    from h3hip import ops
    _, _, w, ws = int8_operands(1, 128, 40, 1)
    y = ops.proj_i8(torch.empty((0, 128), dtype=torch.int8, device="cuda"),
                    torch.empty(0, device="cuda"), w, ws)
    assert y.shape == (0, 40)


@pytest.mark.parametrize("S", [1, 40, 700])
def test_rows_do_not_depend_on_the_others(h3, S):
    """A row's bits are the same alone, in a small call and in a large one: every
    kernel adds exactly."""
    from h3hip import ops
    x, xs, w, ws = int8_operands(1500, 640, 1000, 8)
    note(f"proj_i8 first {S} of 1500 rows")
    all_rows = bits16(ops.proj_i8(x, xs, w, ws))
    some = bits16(ops.proj_i8(x[:S], xs[:S], w, ws))
    assert (some == all_rows[:S]).all()


@pytest.mark.parametrize("big", ["x", "w", "y"])
def test_offsets_past_32_bits(h3, big):
    """x, w and y of more than 4 GiB: the last rows are right."""
    from h3hip import ops
    S, K, N = {"x": (1_100_000, 4096, 24), "w": (40, 4096, 1_100_000),
               "y": (150_000, 128, 16384)}[big]
    x, xs, w, ws = int8_operands(S, K, N, 2)
    note(f"proj_i8 large {big}: S={S} K={K} N={N}")
    y = ops.proj_i8(x, xs, w, ws)
    rows = slice(max(0, S - 300), S)
    cols = slice(max(0, N - 300), N)
    check_product(y[rows, cols], product64(x[rows], xs[rows], w[cols], ws[cols]))
    check_product(y[:40, :40], product64(x[:40], xs[:40], w[:40], ws[:40]))


def test_other_streams_and_two_calls_at_once(h3):
    """Calls that overlap on two streams share nothing."""
    from h3hip import ops
    sides = []
    for seed in (1, 2):
        x, xs, w, ws = int8_operands(900, 1024, 1000, seed)
        sides.append(((x, xs, w, ws), product64(x, xs, w, ws), torch.cuda.Stream()))
    torch.cuda.synchronize()
    note("proj_i8 on two streams")
    got = [[], []]
    for _ in range(4):
        for i, (args, _, st) in enumerate(sides):
            with torch.cuda.stream(st):
                got[i].append(ops.proj_i8(*args))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(sides):
        for y in got[i]:
            check_product(y, want)


@pytest.mark.parametrize("S", [1, 17, 600])
def test_captured_and_replayed(h3, S):
    """quant_rows and proj_i8 in one graph, replayed on new inputs with eager work
    between, against the same calls made eagerly."""
    from h3hip import ops
    _, _, w, ws = int8_operands(1, 1024, 520, 3)
    x = torch.randn((S, 1000), device="cuda").to(torch.bfloat16)
    ops.proj_i8(*ops.quant_rows(x), w, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note(f"proj_i8 captured S={S}")
    with torch.cuda.graph(graph):
        y = ops.proj_i8(*ops.quant_rows(x), w, ws)
    for rep in range(4):
        x.copy_(torch.randn((S, 1000), device="cuda").to(torch.bfloat16))
        want = bits16(ops.proj_i8(*ops.quant_rows(x), w, ws))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (bits16(y) == want).all(), rep
