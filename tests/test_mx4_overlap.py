"""One or two bf16 rows are read by every workgroup of their product's launch while others of it
store: outputs on top of them are refused before any device call (CPU only). More rows are
rounded in a launch of their own first, and outputs beside the rows in one buffer are no overlap."""
import ctypes

import pytest
import torch

K = 512
X = 1 << 20                       # addresses that no refused call reads
FAR = 1 << 24
FEW = [1, 2]


def _p(n):
    return ctypes.c_void_p(n)


def _linear(h3, rows, y, ldx=K, ldy=K, n=K):
    work = h3.lib().h3hip_linear_mx4_workspace(rows, K)
    return h3.lib().h3hip_linear_mx4(_p(X), ldx, _p(FAR), K // 2, _p(FAR), K, n, rows, _p(y), ldy,
                                     _p(FAR) if work else None, work, None)


def _qkv(h3, rows, out):
    return h3.lib().h3hip_qkv_linear_mx4(_p(X), K, _p(FAR), K // 2, _p(FAR), K, _p(FAR), _p(FAR), 1e-6,
                                         _p(FAR), 128, 0, rows, 128, 2, 128, *(_p(o) for o in out),
                                         None, 0, None)


def _refused(h3, rc):
    from h3hip import _lib
    return rc == _lib.EINVAL and "overlap" in h3.last_error()


@pytest.mark.parametrize("rows", FEW)
@pytest.mark.parametrize("at", [0, 2, 2 * K - 2, 2 - 2 * K])
def test_linear_over_its_rows(h3, rows, at):
    assert _refused(h3, _linear(h3, rows, X + at))


def test_linear_second_row(h3):
    """Of either: the rows of x and y have strides of their own."""
    assert _refused(h3, _linear(h3, 2, X + 2 * 4096, ldx=4096))
    assert _refused(h3, _linear(h3, 2, X - 2 * 4096, ldy=4096))
    assert _refused(h3, _linear(h3, 2, X + 2 * 4096, ldx=8192, ldy=4096))


@pytest.mark.parametrize("rows", FEW)
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("at", [0, 256, -(2 * 128 * 128 * 2 - 256), 2 * K - 16])
def test_qkv_over_its_rows(h3, rows, which, at):
    """Anywhere in the [2, 128, 128] heads, whose rows behind the tokens hold the sums."""
    out = [FAR, 2 * FAR, 3 * FAR]
    out[which] = X + at
    assert _refused(h3, _qkv(h3, rows, out))


def test_what_is_no_overlap(h3):
    """Where there is no GPU: the calls come as far as their launch, which fails."""
    if torch.cuda.is_available():
        pytest.skip("the launches must not happen")
    assert not _refused(h3, _linear(h3, 3, X))
    for rows in FEW:
        assert not _refused(h3, _linear(h3, rows, X + 2 * K * rows))
        assert not _refused(h3, _linear(h3, rows, X - 2 * K * rows))
        # x | y and y | x in rows of one buffer
        assert not _refused(h3, _linear(h3, rows, X + 2 * K, ldx=2 * K, ldy=2 * K))
        assert not _refused(h3, _linear(h3, rows, X - 2 * K, ldx=2 * K, ldy=2 * K))
        assert not _refused(h3, _qkv(h3, rows, [FAR, 2 * FAR, X + 2 * K * rows]))
        assert not _refused(h3, _qkv(h3, rows, [X - 2 * 128 * 128 * 2, 2 * FAR, 3 * FAR]))
