"""More rows or channels than a launch of the int8 projections counts are refused with a
message, as the header says (CPU only: refused before any device call)."""
import pytest

from test_int8_refusals import _proj, _qkv

LIMIT = 16_776_960                 # 65,535 tiles of 256


@pytest.mark.parametrize("bad", [dict(rows=LIMIT + 1), dict(n=LIMIT + 1, ldy=LIMIT + 1),
                                 dict(rows=2**31 - 1), dict(rows=LIMIT, n=LIMIT, ldy=LIMIT)])
def test_proj_i8(h3, bad):
    from h3hip import _lib
    assert _proj(h3, **bad) == _lib.EINVAL and "too many rows or channels" in h3.last_error()


@pytest.mark.parametrize("rounding", [0, 1, 3])
@pytest.mark.parametrize("bad", [dict(S=LIMIT + 1, pad=LIMIT + 128), dict(H=LIMIT // 384 + 1)])
def test_qkv_proj_i8(h3, bad, rounding):
    from h3hip import _lib
    assert _qkv(h3, rounding=rounding, **bad) == _lib.EINVAL
    assert "too many rows or channels" in h3.last_error()


def test_the_header_says_so():
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "ch3hip.h")) as f:
        assert f"{LIMIT:,}" in f.read()
