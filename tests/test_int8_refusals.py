"""The int8 projections refuse what their kernels would read or write out of bounds,
before any device call: the C entry points by status, the torch wrappers by message
(CPU only)."""
import ctypes

import pytest
import torch

BUF = ctypes.c_void_p(4096)       # an aligned address no refused call reads


def _quant(h3, x=BUF, ldx=256, rows=4, cols=200, q=BUF, ldq=256, scale=BUF):
    return h3.lib().h3hip_quant_rows(x, ldx, rows, cols, q, ldq, scale, None)


def _proj(h3, x=BUF, ldx=256, xs=BUF, w=BUF, ldw=256, ws=BUF, k=256, n=64, rows=4, y=BUF, ldy=64):
    return h3.lib().h3hip_proj_i8(x, ldx, xs, w, ldw, ws, k, n, rows, y, ldy, None)


def _qkv(h3, x=BUF, ldx=256, xs=BUF, w=BUF, ldw=256, ws=BUF, k=256, gq=BUF, gk=BUF, table=BUF,
         rot=128, rounding=0, S=4, pad=128, H=2, D=128, q=BUF, ko=BUF, v=BUF):
    return h3.lib().h3hip_qkv_proj_i8(x, ldx, xs, w, ldw, ws, k, gq, gk, 1e-6, table, rot, rounding,
                                      S, pad, H, D, q, ko, v, None)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "shape"), (dict(cols=0), "shape"), (dict(cols=2**31 - 5), "shape"),
    (dict(ldx=199), "ldx"), (dict(ldq=240), "ldq"), (dict(ldq=264), "ldq"), (dict(x=None), "NULL"),
    (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=ctypes.c_void_p(4097)), "aligned"),
    (dict(q=ctypes.c_void_p(4104)), "aligned"), (dict(scale=ctypes.c_void_p(4098)), "aligned")])
def test_quant_rows(h3, bad, word):
    from h3hip import _lib
    assert _quant(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_no_rows_are_no_work(h3):
    from h3hip import _lib
    assert _quant(h3, rows=0, x=None, q=None, scale=None) == _lib.OK
    assert _proj(h3, rows=0, x=None, xs=None, y=None) == _lib.OK


@pytest.mark.parametrize("bad,word", [
    (dict(k=0), "shape"), (dict(n=0), "shape"), (dict(rows=-1), "shape"), (dict(ldx=240), "ldx"),
    (dict(ldx=264), "ldx"), (dict(ldw=128), "ldw"), (dict(ldy=63), "ldy"), (dict(x=None), "NULL"),
    (dict(xs=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"), (dict(y=None), "NULL"),
    (dict(x=ctypes.c_void_p(4104)), "aligned"), (dict(w=ctypes.c_void_p(4104)), "aligned"),
    (dict(ws=ctypes.c_void_p(4098)), "aligned"), (dict(xs=ctypes.c_void_p(4098)), "aligned"),
    (dict(y=ctypes.c_void_p(4097)), "aligned"), (dict(ldx=1 << 26), "2 GiB"),
    (dict(ldw=1 << 26), "2 GiB")])
def test_proj_i8(h3, bad, word):
    from h3hip import _lib
    assert _proj(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_proj_i8_declines(h3):
    from h3hip import _lib
    for k in (64, 200, 131072):
        assert _proj(h3, k=k, ldx=1 << 20, ldw=1 << 20) == _lib.DECLINED
        assert "in_features" in h3.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(k=0), "hidden"), (dict(S=0), "shape"), (dict(S=0, pad=0, x=None), "shape"), (dict(H=0), "shape"), (dict(pad=64), "shape"),
    (dict(S=129), "shape"), (dict(H=6_000_000), "shape"), (dict(gq=None), "gammas"),
    (dict(table=None), "table"), (dict(rounding=2), "rounding"), (dict(q=None), "NULL"),
    (dict(v=ctypes.c_void_p(4104)), "aligned"), (dict(table=ctypes.c_void_p(4104)), "aligned"),
    (dict(ldx=128), "ldx"), (dict(x=None), "NULL")])
def test_qkv_proj_i8(h3, bad, word):
    from h3hip import _lib
    assert _qkv(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_qkv_proj_i8_declines(h3):
    from h3hip import _lib
    for bad in (dict(D=64), dict(rot=64), dict(k=192, ldx=192, ldw=192), dict(k=131072)):
        assert _qkv(h3, **bad) == _lib.DECLINED and "declined" in h3.last_error()


def _i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def test_wrappers(h3):
    from h3hip import ops
    bf = torch.zeros((4, 200), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.quant_rows(bf)
    with pytest.raises(ValueError, match="unit column stride"):
        ops.quant_rows(bf.t())
    with pytest.raises(ValueError, match="K > 0"):
        ops.quant_rows(bf[:, :0])
    s, t = torch.ones(4), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        ops.proj_i8(_i8(4, 128), s, _i8(8, 128), t)
    for x, xs, w, ws, word in [
            (bf, s, _i8(8, 200), t, "int8"), (_i8(4, 128), s, _i8(8, 256), t, "w must be"),
            (_i8(4, 128), t, _i8(8, 128), t, "x_scale"), (_i8(4, 128), s, _i8(8, 128), s, "w_scale"),
            (_i8(4, 128), s.double(), _i8(8, 128), t, "x_scale"),
            (_i8(4, 128), s, _i8(128, 8).t(), t, "unit column stride"),
            (_i8(4, 128), torch.ones(8)[::2], _i8(8, 128), t, "x_scale")]:
        with pytest.raises(ValueError, match=word):
            ops.proj_i8(x, xs, w, ws)
