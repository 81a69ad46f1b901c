"""h3hip_proj_mx4 on the GPU against the product of the decoded operands in 64 bits: equal
bits where every sum is exact, the derived bound elsewhere; one row to several thousand, odd
widths, strides and alignments, every scale, and what it may not write."""
import pytest
import torch

from _gpu import note
from _mx4 import bits16, check_exact, check_product, decode64, mx4_operand, product64

pytestmark = pytest.mark.gpu

# One size for each tile shape (rows, in, out), with rows and channels that end inside a tile;
# test_proj_mx4_tile_host.py checks which shape each one takes.
SHAPES = [("256x256", 3001, 768, 5000), ("256x224", 4000, 512, 3500), ("256x192", 1301, 256, 9000),
          ("256x160", 4000, 256, 2500), ("256x128", 641, 3584, 9000), ("128x192", 1700, 1024, 3500),
          ("128x160", 3001, 768, 1300), ("128x128", 385, 1792, 5000), ("128x128p", 201, 256, 12000),
          ("128x64p", 100, 256, 9000), ("128x32p", 65, 256, 9000), ("64x64p", 1, 256, 9000),
          ("32x64p", 33, 256, 5000), ("32x32p", 1, 256, 100)]
SIZES = [(1, 256, 1), (1, 32, 16), (1, 5120, 5120), (2, 256, 17), (7, 31, 33), (15, 512, 128),
         (16, 768, 130), (17, 768, 33), (31, 1280, 127), (33, 256, 777), (64, 2304, 512),
         (65, 4096, 129), (125, 5120, 5120), (129, 512, 640), (130, 1280, 256), (255, 1792, 1000),
         (300, 2304, 520), (637, 1000, 777), (917, 5120, 5120), (1151, 7168, 5376),
         (2048, 512, 5120), (4100, 1024, 700), (2500, 257, 5000), (6001, 300, 1300)]


@pytest.mark.parametrize("S,K,N", SIZES)
def test_exact_sums(h3, S, K, N):
    """Exponents 0, 1, 2: the sums are exact, so a wrong scale, value or row shows in bits."""
    from h3hip import ops
    x, w = mx4_operand(S, K, S + K), mx4_operand(N, K, S + N)
    note(f"proj_mx4 S={S} K={K} N={N}")
    y = ops.proj_mx4(x, w)
    torch.cuda.synchronize()
    assert y.shape == (S, N) and y.dtype == torch.bfloat16
    check_exact(y, product64(x, w))


@pytest.mark.parametrize("shape,S,K,N", SHAPES, ids=[s[0] for s in SHAPES])
def test_every_tile_shape(h3, shape, S, K, N):
    """Into rows that are and are not on 16 bytes; nothing past a row's channels or the last row
    is written. The reduction one block short of its last step, too."""
    from h3hip import ops
    for k, ldy, first in ((K, N + 8 - N % 8, 0), (K - 32, N + 3, 1)):
        x, w = mx4_operand(S, k, S + k), mx4_operand(N, k, S + N)
        buf = torch.full(((S + 1) * ldy + first,), 7.0, dtype=torch.bfloat16, device="cuda")
        rows = buf[first:].view(S + 1, ldy)
        note(f"proj_mx4 {shape} S={S} K={k} N={N} ldy={ldy}")
        check_exact(ops.proj_mx4(x, w, out=rows[:S, :N]), product64(x, w))
        assert (rows[S] == 7.0).all() and (rows[:, N:] == 7.0).all() and (buf[:first] == 7.0).all()


@pytest.mark.parametrize("S,K,N", [(1, 5120, 300), (40, 2304, 512), (300, 1280, 1000),
                                   (1151, 7168, 640), (2500, 512, 3500)])
@pytest.mark.parametrize("low,span", [(-12, 25), (-60, 100), (-126, 3)])
def test_scales_of_any_size(h3, S, K, N, low, span):
    from h3hip import ops
    x, w = mx4_operand(S, K, S, low, span), mx4_operand(N, K, N, low, span)
    note(f"proj_mx4 scales {low}+{span} S={S} K={K} N={N}")
    check_product(ops.proj_mx4(x, w), x, w)


def test_largest_and_smallest_scales(h3):
    """2^127 against 2^-127, and products past either end of fp32."""
    from h3hip import ops
    from _mx4 import product_bound
    x, w = mx4_operand(40, 512, 1, 0, 1), mx4_operand(60, 512, 2, 0, 1)
    note("proj_mx4 extreme scales")
    for ex, ew in ((254, 0), (0, 254), (254, 10), (130, 124)):
        a, b = x._replace(scale=torch.full_like(x.scale, ex)), w._replace(scale=torch.full_like(w.scale, ew))
        want = product64(a, b)
        assert ((ops.proj_mx4(a, b).double() - want).abs() <= product_bound(a, b, want)).all()
    a, b = x._replace(scale=torch.full_like(x.scale, 254)), w._replace(scale=torch.full_like(w.scale, 254))
    y, want = ops.proj_mx4(a, b), product64(a, b)
    # Every product that is not zero is past fp32: a sum of one sign is infinite, of both NaN.
    assert not torch.isfinite(y[want != 0]).any()
    a, b = x._replace(scale=torch.zeros_like(x.scale)), w._replace(scale=torch.zeros_like(w.scale))
    assert not ops.proj_mx4(a, b).any()


@pytest.mark.parametrize("S,N,K", [(3, 200, 512), (300, 200, 800), (700, 1000, 256)])
def test_scales_that_are_nan(h3, S, N, K):
    """One block's NaN makes its row (or channel) NaN and nothing else."""
    from h3hip import ops
    x, w = mx4_operand(S, K, 4), mx4_operand(N, K, 5)
    want = product64(x, w)
    for rows, r, b in ((x, 1, K // 32 - 1), (w, 6, 0)):
        rows.scale[b // 16, r // 16, 16 * (b % 4) + r % 16, b // 4 % 4] = 255
    note(f"proj_mx4 NaN scales S={S}")
    y = ops.proj_mx4(x, w)
    nan = torch.zeros((S, N), dtype=torch.bool, device="cuda")
    nan[1], nan[:, 6] = True, True
    assert torch.equal(torch.isnan(y), nan)
    check_exact(torch.where(nan, 0, y), want.masked_fill(nan, 0.0))


@pytest.mark.parametrize("S,K,N", [(5, 40, 30), (300, 300, 515), (65, 1000, 129)])
def test_scales_of_rows_that_do_not_exist(h3, S, K, N):
    """Whatever bytes lie in the groups behind the last row (NaN here) reach nothing."""
    from h3hip import ops
    x, w = mx4_operand(S, K, 1), mx4_operand(N, K, 2)
    want = product64(x, w)
    for rows, n in ((x, S), (w, N)):
        every = rows.scale.view(rows.scale.shape[0], -1, 4, 16, 4)
        if n % 16:
            every[:, -1, :, n % 16:] = 255
    note(f"proj_mx4 stray scales S={S} N={N}")
    check_exact(ops.proj_mx4(x, w), want)


@pytest.mark.parametrize("S,K,N,ldx,ldw,ldy,first", [
    (70, 512, 130, 272, 400, 136, 0), (70, 512, 130, 256, 256, 131, 0),
    (300, 768, 512, 400, 384, 520, 8), (300, 768, 515, 384, 384, 520, 3),
    (5, 256, 64, 144, 160, 64, 1), (2, 256, 777, 128, 128, 1001, 5), (1300, 512, 1000, 256, 272, 1003, 1)])
def test_strides_and_what_is_not_written(h3, S, K, N, ldx, ldw, ldy, first):
    from h3hip import ops
    x, w = mx4_operand(S, K, S, stride=ldx), mx4_operand(N, K, N, stride=ldw)
    buf = torch.full(((S + 2) * ldy + first,), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = buf[first:].view(S + 2, ldy)
    note(f"proj_mx4 strided S={S} K={K} N={N} ldy={ldy} first={first}")
    y = ops.proj_mx4(x, w, out=rows[1:S + 1, :N])
    torch.cuda.synchronize()
    check_exact(y, product64(x, w))
    assert (rows[0] == 7.0).all() and (rows[S + 1] == 7.0).all() and (rows[:, N:] == 7.0).all()
    assert (buf[:first] == 7.0).all()


@pytest.mark.parametrize("S,K,N", [(1, 5120, 700), (3, 33, 50), (16, 1000, 777), (33, 5120, 256),
                                   (300, 1001, 640), (1151, 512, 1000)])
def test_bf16_rows_are_rounded_on_the_way(h3, S, K, N):
    """proj_mx4 of bf16 rows is proj_mx4 of their 4-bit form: equal bits where sums are exact."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(S + K)
    # Each block's largest magnitude in [4, 32]: quarters, few enough for exact sums.
    x = (torch.rand((S, K), generator=g, device="cuda") * 2 - 1) * 2.0 ** torch.randint(
        3, 6, (S, K), generator=g, device="cuda")
    x[:, ::32] = 4.0
    x = x.to(torch.bfloat16)
    w = mx4_operand(N, K, N)
    q = ops.quant_rows_mx4(x)
    assert int(q.exponents().min()) >= 127
    size = torch.mm(decode64(q).abs(), decode64(w).abs().t().contiguous())
    assert float(4 * size.max()) < 2 ** 24      # any partial sum is exact in fp32
    note(f"proj_mx4 of bf16 rows S={S} K={K} N={N}")
    y = ops.proj_mx4(x, w)
    check_exact(y, product64(q, w))
    assert (bits16(y) == bits16(ops.proj_mx4(q, w))).all()
    out = torch.empty((S, N), dtype=torch.bfloat16, device="cuda")
    assert ops.proj_mx4(x, w, out=out) is out and (bits16(out) == bits16(y)).all()
    # Strided rows, at an address that is no multiple of 16.
    buf = torch.empty(S * (K + 5) + 3, dtype=torch.bfloat16, device="cuda")
    xs = buf[3:].view(S, K + 5)[:, :K]
    xs.copy_(x)
    assert (bits16(ops.proj_mx4(xs, w)) == bits16(y)).all()


@pytest.mark.parametrize("S", [1, 2, 3])
@pytest.mark.parametrize("K,N", [(8, 5), (256, 16), (264, 17), (1000, 300), (2560, 33), (5120, 40),
                                 (6000, 31), (9984, 100), (10240, 16), (10248, 48), (20480, 20),
                                 (30000, 18), (61000, 7), (100_000, 3)])
def test_one_and_two_bf16_rows(h3, S, K, N):
    """Every number of units in flight, whole and part batches, and the sizes that take the other
    way: against the product of the rows' 4-bit form in 64 bits; nothing else is written."""
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(S + K)
    x = (torch.randn((S, K), generator=g, device="cuda") * torch.exp(
        torch.randn((S, K), generator=g, device="cuda"))).to(torch.bfloat16)
    w = mx4_operand(N, K, N, -8, 16)
    buf = torch.full((S + 1, N + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    note(f"proj_mx4 of {S} bf16 rows K={K} N={N}")
    y = ops.proj_mx4(x, w, out=buf[:S, :N])
    check_product(y, ops.quant_rows_mx4(x), w)
    assert (buf[S] == 7.0).all() and (buf[:, N:] == 7.0).all()


@pytest.mark.parametrize("S", [1, 2, 9, 16, 17, 40, 400])
def test_bf16_rows_that_are_not_finite(h3, S):
    from h3hip import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn((S, 600), generator=g, device="cuda").to(torch.bfloat16)
    w = mx4_operand(300, 600, 3)
    want = ops.proj_mx4(x, w)
    x[S - 1, 599], x[S // 2, 0] = float("inf"), float("nan")
    note(f"proj_mx4 of bf16 rows that are not finite S={S}")
    y = ops.proj_mx4(x, w)
    bad = torch.zeros(S, dtype=torch.bool, device="cuda")
    bad[S - 1] = bad[S // 2] = True
    assert torch.isnan(y[bad]).all()
    assert (bits16(y[~bad]) == bits16(want[~bad])).all()


def test_no_rows(h3):
    from h3hip import ops
    w = mx4_operand(40, 128, 1)
    assert ops.proj_mx4(torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"), w).shape == (0, 40)
    x = ops.quant_rows_mx4(torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"))
    assert ops.proj_mx4(x, w).shape == (0, 40)


@pytest.mark.parametrize("S", [1, 40, 700])
def test_rows_do_not_depend_on_the_others(h3, S):
    """A row's bits are the same alone, in a small call and in a large one."""
    from h3hip import ops
    x, w = mx4_operand(1500, 1280, 8, -20, 40), mx4_operand(1000, 1280, 9, -20, 40)
    note(f"proj_mx4 first {S} of 1500 rows")
    groups = (S + 15) // 16
    some = ops.Mx4Rows(x.values[:S], x.scale[:, :groups].contiguous(), x.cols)
    assert (bits16(ops.proj_mx4(some, w)) == bits16(ops.proj_mx4(x, w))[:S]).all()


@pytest.mark.parametrize("big", ["x", "w", "y"])
def test_offsets_past_32_bits(h3, big):
    """x, w and y of more than 4 GiB: the last rows are right."""
    from h3hip import ops
    S, K, N = {"x": (1_100_000, 8192, 24), "w": (40, 8192, 1_100_000),
               "y": (150_000, 256, 16384)}[big]
    x, w = mx4_operand(S, K, 1, 0, 2), mx4_operand(N, K, 2, 0, 2)
    note(f"proj_mx4 large {big}: S={S} K={K} N={N}")
    y = ops.proj_mx4(x, w)

    def part(rows, lo, hi):      # whole groups of 16
        return rows._replace(values=rows.values[lo:hi],
                             scale=rows.scale[:, lo // 16:(hi + 15) // 16].contiguous())
    for lo, n in ((0, 48), (1, 48)):
        a = (max(0, S - n) // 16 * 16, S) if lo else (0, min(S, n))
        b = (max(0, N - n) // 16 * 16, N) if lo else (0, min(N, n))
        check_exact(y[a[0]:a[1], b[0]:b[1]], product64(part(x, *a), part(w, *b)))


def test_other_streams_and_two_calls_at_once(h3):
    from h3hip import ops
    sides = []
    for seed in (1, 2):
        x, w = mx4_operand(900, 2048, seed), mx4_operand(1000, 2048, seed + 5)
        sides.append((x, w, product64(x, w), torch.cuda.Stream()))
    few = torch.randn((3, 2048), device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    note("proj_mx4 on two streams")
    got, small = [[], []], [[], []]
    for _ in range(4):
        for i, (x, w, _, st) in enumerate(sides):
            with torch.cuda.stream(st):
                got[i].append(ops.proj_mx4(x, w))
                small[i].append(ops.proj_mx4(few, w))
    torch.cuda.synchronize()
    for i, (x, w, want, _) in enumerate(sides):
        alone = bits16(ops.proj_mx4(few, w))
        for y, z in zip(got[i], small[i]):
            check_exact(y, want)
            assert (bits16(z) == alone).all()


@pytest.mark.parametrize("S", [1, 17, 600])
def test_captured_and_replayed(h3, S):
    """proj_mx4 of bf16 rows in a graph, replayed on new inputs with eager work between."""
    from h3hip import ops
    w = mx4_operand(520, 1000, 3, -3, 6)
    x = torch.randn((S, 1000), device="cuda").to(torch.bfloat16)
    ops.proj_mx4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note(f"proj_mx4 captured S={S}")
    with torch.cuda.graph(graph):
        y = ops.proj_mx4(x, w)
    for rep in range(4):
        x.copy_(torch.randn((S, 1000), device="cuda").to(torch.bfloat16))
        want = bits16(ops.proj_mx4(x, w))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (bits16(y) == want).all(), rep


def test_decoding_of_the_tests_own(h3):
    """decode64 is what dequant_rows_mx4 gives."""
    from h3hip import ops
    x = mx4_operand(37, 777, 1, -30, 60)
    assert torch.equal(decode64(x), ops.dequant_rows_mx4(x).double())


@pytest.mark.parametrize("first,S,N", [(16, 3, 100), (0, 300, 517), (32, 700, 640)])
def test_some_rows_of_a_weight(h3, first, S, N):
    """rows() of a weight: those channels' bits."""
    from h3hip import ops
    x, w = mx4_operand(S, 512, S, -5, 10), mx4_operand(N + 41, 512, N, -5, 10)
    note(f"proj_mx4 channels {first}.. of {N + 41}, S={S}")
    every = bits16(ops.proj_mx4(x, w))
    some = bits16(ops.proj_mx4(x, w.rows(first, N)))
    assert (some == every[:, first:first + N]).all()
