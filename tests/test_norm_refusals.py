"""h3hip_norm_modulate and h3hip_gated_residual refuse what their kernel would read or write
out of bounds, before any device call: the C entry points by status, the torch wrappers by
message (CPU only)."""
import ctypes

import pytest
import torch

BUF = ctypes.c_void_p(4096)       # an aligned address no refused call reads
ODD = ctypes.c_void_p(4097)
AWAY = ctypes.c_void_p(1 << 20)
NONE = object()


def _starts(v):
    return None if v is None else (ctypes.c_int32 * len(v))(*v)


def _norm(gamma=4096, scale=4096, shift=4096, ld_scale=100, ld_shift=100):
    from h3hip import _lib
    return _lib.NormC(gamma, scale, shift, ld_scale, ld_shift)


def _before(h3, x=BUF, ldx=100, rows=4, hidden=100, norm=None, starts=(0, 2), segments=2, h=BUF,
            ldh=100):
    n = None if norm is NONE else ctypes.byref(norm or _norm())
    return h3.lib().h3hip_norm_modulate(x, ldx, rows, hidden, n, 1e-6, _starts(starts), segments, h,
                                        ldh, None)


def _after(h3, x=BUF, ldx=100, y=BUF, ldy=100, rows=4, hidden=100, gate=BUF, ld_gate=100, post=BUF,
           norm=None, starts=(0, 2), segments=2, r=BUF, ldr=100, h=BUF, ldh=100):
    n = None if norm is NONE else ctypes.byref(norm or _norm())
    return h3.lib().h3hip_gated_residual(x, ldx, y, ldy, rows, hidden, gate, ld_gate, post, 1.0, n,
                                         1e-6, _starts(starts), segments, r, ldr, h, ldh, None)


SHARED = [(dict(rows=-1), "shape"), (dict(hidden=0), "shape"), (dict(segments=0), "segments"),
          (dict(segments=17, starts=range(17)), "segments"), (dict(starts=None), "starts"),
          (dict(starts=(1, 2)), "row 0"), (dict(starts=(0, -1)), "descend"),
          (dict(starts=(0, 5, 4), segments=3), "descend"), (dict(ldx=99), "cover"),
          (dict(ldh=99), "cover"), (dict(x=None), "NULL"), (dict(h=None), "NULL"),
          (dict(x=ODD), "aligned"), (dict(h=ODD), "aligned"), (dict(norm=("gamma", 4097)), "aligned"),
          (dict(norm=("scale", 4097)), "aligned"), (dict(norm=("shift", 4097)), "aligned"),
          (dict(norm=("ld_scale", 99)), "cover"), (dict(norm=("ld_shift", 99)), "cover")]
AFTER = [(dict(ldy=99), "cover"), (dict(ldr=99), "cover"), (dict(ld_gate=99), "cover"),
         (dict(y=None), "NULL"), (dict(r=None), "NULL"), (dict(y=ODD), "aligned"),
         (dict(r=ODD), "aligned"), (dict(gate=ODD), "aligned"), (dict(post=ODD), "aligned"),
         # r, h, x and y are one address in these calls, which in place they have to be with one
         # stride; r and h never.
         (dict(), "two tensors"), (dict(h=AWAY, ldr=104), "stride"), (dict(r=AWAY, ldh=104), "stride"),
         (dict(h=AWAY, ldy=104), "stride"), (dict(r=AWAY, ldy=104), "stride")]


def _args(bad):
    bad = dict(bad)
    if isinstance(bad.get("norm"), tuple):
        bad["norm"] = _norm(**{bad["norm"][0]: bad["norm"][1]})
    return bad


@pytest.mark.parametrize("bad,word", SHARED + [(dict(norm=NONE), "NULL"), (dict(ldh=104), "stride")])
def test_norm_modulate(h3, bad, word):
    from h3hip import _lib
    assert _before(h3, **_args(bad)) == _lib.EINVAL and word in h3.last_error()


@pytest.mark.parametrize("bad,word", SHARED + AFTER)
def test_gated_residual(h3, bad, word):
    from h3hip import _lib
    assert _after(h3, **_args(bad)) == _lib.EINVAL and word in h3.last_error()


def test_no_rows_and_declines(h3):
    from h3hip import _lib
    assert _before(h3, rows=0, x=None, h=None) == _lib.OK
    assert _after(h3, rows=0, x=None, y=None, r=None, h=None) == _lib.OK
    assert _after(h3, rows=0, norm=NONE, h=None, ldh=0, gate=None, ld_gate=0, post=None) == _lib.OK
    for call in (_before, _after):
        big = dict(hidden=16385, ldx=20000, ldh=20000, norm=_norm(ld_scale=20000, ld_shift=20000))
        if call is _after:
            big.update(ldy=20000, ldr=20000, ld_gate=20000)
        assert call(h3, **big) == _lib.DECLINED and "hidden" in h3.last_error()


def test_wrappers(h3):
    from h3hip import ops
    x = torch.zeros((4, 100), dtype=torch.bfloat16)
    for call in (ops.norm_modulate, lambda t: ops.gated_residual(t, t)):
        for t, word in ((x, "GPU"), (x.float(), "bfloat16"), (x.t(), "unit column stride"),
                        (x[0], "2-D"), (x[:, :0], "K > 0")):
            with pytest.raises(ValueError, match=word):
                call(t)
    wide = torch.empty((1, 2 ** 31), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.norm_modulate(wide)


def test_wrapper_checks_of_tables(h3):
    """The checks behind the one of the device, on their own."""
    from h3hip import ops
    cpu = torch.device("cpu")
    good = torch.zeros((2, 100), dtype=torch.bfloat16)
    assert ops._norm_table("scale", good, 2, 100, cpu)[1] == 100
    assert ops._norm_table("scale", good[0], 1, 100, cpu)[0] == good.data_ptr()
    assert ops._norm_table("scale", None, 2, 100, cpu)[0] is None
    for t in (good[0], good[:, :99], good.float(), good[:1],
              torch.zeros((2, 200), dtype=torch.bfloat16)[:, ::2]):
        with pytest.raises(ValueError, match="scale"):
            ops._norm_table("scale", t, 2, 100, cpu)
    for t in (good, good[0, :99], good[0].float(), torch.zeros(200, dtype=torch.bfloat16)[::2]):
        with pytest.raises(ValueError, match="gamma"):
            ops._norm_gamma("gamma", t, 100, cpu)
    import numpy as np
    assert list(ops._segments(np.array([0, 3]))[0]) == list(ops._segments(torch.tensor([0, 3]))[0])
    for s in ([], range(17), [0, -1], [0, 2 ** 31], [-1]):
        with pytest.raises(ValueError, match="segments"):
            ops._segments(s)
    assert ops._segments(None) == (None, 1) and list(ops._segments([0, 3])[0]) == [0, 3]
