"""h3hip_quant_rows on the GPU: rows of bf16 rounded to int8, exactly as defined
(half to even, from the unrounded quotient), for widths around every chunk, any
alignment and row stride, and the rows where rounding can go wrong."""
import numpy as np
import pytest
import torch

from _gpu import note
from _int8 import quant64, rows_bf16, to64

pytestmark = pytest.mark.gpu


def _check(x, q, s):
    K = x.shape[1]
    want_q, want_s = quant64(to64(x))
    got = q.cpu().numpy()
    assert got.shape[1] == (K + 127) // 128 * 128
    assert not got[:, K:].any(), "columns past the row are not zeros"
    bad = np.argwhere(got[:, :K] != want_q)
    assert bad.size == 0, (bad[:4], got[tuple(bad[0])], want_q[tuple(bad[0])])
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)


@pytest.mark.parametrize("S,K", [
    (1, 1), (1, 15), (3, 16), (17, 127), (1, 128), (20, 129), (4, 1000), (5, 1023), (6, 1024),
    (7, 1025), (33, 2048), (18, 2049), (18, 3073), (18, 4096), (18, 5120), (18, 5376), (3, 8191),
    (2, 8192), (3, 8193), (17, 12288), (18, 12289), (17, 16384), (17, 16385), (17, 20000), (2049, 2500),
    (2051, 3100), (2050, 4096), (2049, 4097), (2048, 2500),
    (1, 131072), (1000, 640)])
def test_rows_exact(h3, S, K):
    from h3hip import ops
    x = rows_bf16(S, K, 10 * K + S)
    note(f"quant_rows S={S} K={K}")
    _check(x, *ops.quant_rows(x))


@pytest.mark.parametrize("K,ld,first", [(777, 777, 0), (777, 781, 0), (640, 648, 0), (640, 640, 1),
                                        (640, 643, 3), (9000, 9001, 5), (1, 3, 1)])
def test_any_alignment_and_stride(h3, K, ld, first):
    """Rows that do not begin on 16 bytes, and a base that does not."""
    from h3hip import ops
    S = 19
    flat = torch.full((S * ld + first + 8,), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = flat[first:first + S * ld].view(S, ld)[:, :K]
    x.copy_(rows_bf16(S, K, K + ld))
    note(f"quant_rows K={K} ld={ld} first={first}")
    _check(x, *ops.quant_rows(x))


def test_rows_that_have_no_int8_form(h3):
    """An infinity or a NaN anywhere makes its row's scale NaN and its values 0, and
    no other row's."""
    from h3hip import ops
    for K in (130, 1500, 5120, 9000, 20000):
        x = rows_bf16(12, K, 5, special=False)
        x[1, 0], x[3, K - 1], x[5, K // 2] = float("inf"), float("-inf"), float("nan")
        note(f"quant_rows not finite K={K}")
        q, s = ops.quant_rows(x)
        _check(x, q, s)
        assert torch.isnan(s[[1, 3, 5]]).all() and not q[[1, 3, 5]].any()
        assert torch.isfinite(s[[0, 2, 4, 6]]).all()


def test_writes_only_its_rows(h3):
    from h3hip import ops
    S, K = 21, 300
    x = rows_bf16(S, K, 3)
    q = torch.full((S + 2, 400), 77, dtype=torch.int8, device="cuda")
    s = torch.full((S + 3,), 5.0, device="cuda")
    note("quant_rows into strided outputs")
    ops.quant_rows(x, out=(q[1:S + 1, :384], s[1:S + 1]))
    _check(x, q[1:S + 1, :384], s[1:S + 1])
    assert (q[0] == 77).all() and (q[S + 1] == 77).all() and (q[:, 384:] == 77).all()
    assert s[0] == 5.0 and (s[S + 1:] == 5.0).all()


def test_no_rows(h3):
    from h3hip import ops
    q, s = ops.quant_rows(torch.empty((0, 300), dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 384) and s.shape == (0,)


def test_rows_past_four_gigabytes(h3):
    """x of 4.4 GiB: the offsets of its last rows pass 32 bits."""
    from h3hip import ops
    S, K = 1_150_000, 2048
    x = torch.zeros((S, K), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rows_bf16(3, K, 9)
    x[0] = x[-1]
    note(f"quant_rows S={S} K={K}")
    q, s = ops.quant_rows(x)
    _check(x[-3:], q[-3:], s[-3:])
    _check(x[:2], q[:2], s[:2])
    assert float(s[1:-3].abs().max()) == 0.0


def test_more_rows_than_a_launch_takes(h3):
    """2^24 + 5 rows of one element: the launch covers 2^24, the next one the rest."""
    from h3hip import ops
    S = (1 << 24) + 5
    x = torch.zeros((S, 1), dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, (1 << 24) - 1, 1 << 24, S - 1]
    x[rows, 0] = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0], dtype=torch.bfloat16, device="cuda")
    note(f"quant_rows S={S}")
    q, s = ops.quant_rows(x)
    assert q[rows, 0].tolist() == [127, -127, 127, -127, 127] and not q[:, 1:].any()
    assert int((s != 0).sum()) == 5 and int(q[:, 0].abs().sum()) == 5 * 127
    want = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0]) / 127
    assert torch.equal(s[rows].cpu(), want)
