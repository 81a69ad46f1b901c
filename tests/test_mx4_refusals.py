"""The 4-bit rows and projections refuse what their kernels would read or write out of bounds,
before any device call: the C entry points by status, the torch wrappers by message (CPU only)."""
import ctypes

import pytest
import torch

BUF = ctypes.c_void_p(4096)       # an aligned address no refused call reads
WIDE = 2 ** 32 + 256


def at(n):
    return ctypes.c_void_p(4096 + n)


def _quant(h3, x=BUF, ldx=256, rows=4, cols=200, q=BUF, ldq=128, scale=BUF):
    return h3.lib().h3hip_quant_rows_mx4(x, ldx, rows, cols, q, ldq, scale, None)


def _dequant(h3, q=BUF, ldq=128, scale=BUF, rows=4, cols=200, x=BUF, ldx=200):
    return h3.lib().h3hip_dequant_rows_mx4(q, ldq, scale, rows, cols, x, ldx, None)


def _proj(h3, x=BUF, ldx=256, xs=BUF, w=BUF, ldw=256, ws=BUF, k=512, n=64, rows=4, y=BUF, ldy=64):
    return h3.lib().h3hip_proj_mx4(x, ldx, xs, w, ldw, ws, k, n, rows, y, ldy, None)


def _qkv(h3, x=BUF, ldx=256, xs=BUF, w=BUF, ldw=256, ws=BUF, k=512, gq=BUF, gk=BUF, table=BUF,
         rot=128, rounding=0, S=4, pad=128, H=2, D=128, q=BUF, ko=BUF, v=BUF):
    return h3.lib().h3hip_qkv_proj_mx4(x, ldx, xs, w, ldw, ws, k, gq, gk, 1e-6, table, rot, rounding,
                                       S, pad, H, D, q, ko, v, None)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "shape"), (dict(cols=0), "shape"), (dict(cols=33_553_921), "shape"),
    (dict(ldx=199), "ldx"), (dict(ldq=112), "ldq"), (dict(ldq=136), "ldq"), (dict(x=None), "NULL"),
    (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=at(1)), "aligned"),
    (dict(q=at(8)), "aligned"), (dict(scale=at(2)), "aligned")])
def test_quant_rows(h3, bad, word):
    from h3hip import _lib
    assert _quant(h3, **bad) == _lib.EINVAL and word in h3.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "shape"), (dict(cols=0), "shape"), (dict(cols=33_553_921), "shape"),
    (dict(ldx=199), "ldx"), (dict(ldq=96), "ldq"), (dict(ldq=130), "ldq"), (dict(x=None), "NULL"),
    (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=at(1)), "aligned"),
    (dict(q=at(2)), "aligned")])
def test_dequant_rows(h3, bad, word):
    from h3hip import _lib
    assert _dequant(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_no_rows_are_no_work(h3):
    from h3hip import _lib
    assert _quant(h3, rows=0, x=None, q=None, scale=None) == _lib.OK
    assert _dequant(h3, rows=0, x=None, q=None, scale=None) == _lib.OK
    assert _proj(h3, rows=0, x=None, xs=None, y=None) == _lib.OK


@pytest.mark.parametrize("bad,word", [
    (dict(k=0), "shape"), (dict(n=0), "shape"), (dict(rows=-1), "shape"), (dict(ldx=240), "ldx"),
    (dict(ldx=264), "ldx"), (dict(ldw=128), "ldw"), (dict(ldy=63), "ldy"), (dict(x=None), "NULL"),
    (dict(xs=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"), (dict(y=None), "NULL"),
    (dict(x=at(8)), "aligned"), (dict(w=at(8)), "aligned"), (dict(ws=at(2)), "aligned"),
    (dict(xs=at(2)), "aligned"), (dict(y=at(1)), "aligned"), (dict(ldx=1 << 26), "2 GiB"),
    (dict(ldw=1 << 26), "2 GiB"), (dict(rows=16_777_200), "too many"),
    (dict(rows=1, n=16_777_217, ldy=1 << 26), "too many")])
def test_proj(h3, bad, word):
    from h3hip import _lib
    assert _proj(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_declines(h3):
    from h3hip import _lib
    for k in (128, 200, 513):
        assert _proj(h3, k=k, ldx=1 << 20, ldw=1 << 20) == _lib.DECLINED
        assert "in_features" in h3.last_error()
    for bad in (dict(D=64), dict(rot=64), dict(k=384)):
        assert _qkv(h3, **bad) == _lib.DECLINED and "declined" in h3.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(k=0), "hidden"), (dict(S=0), "shape"), (dict(H=0), "shape"), (dict(pad=64), "shape"),
    (dict(S=129), "shape"), (dict(H=6_000_000), "shape"), (dict(gq=None), "gammas"),
    (dict(table=None), "table"), (dict(rounding=2), "rounding"), (dict(q=None), "NULL"),
    (dict(v=at(8)), "aligned"), (dict(table=at(8)), "aligned"), (dict(ldx=128), "ldx"),
    (dict(x=None), "NULL"), (dict(rounding=3, ko=at(8)), "aligned")])
def test_qkv_proj(h3, bad, word):
    from h3hip import _lib
    assert _qkv(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def _linear(h3, x=BUF, ldx=500, w=BUF, ldw=256, ws=BUF, k=500, n=64, rows=4, y=BUF, ldy=64, work=BUF,
            size=1 << 20):
    return h3.lib().h3hip_linear_mx4(x, ldx, w, ldw, ws, k, n, rows, y, ldy, work, size, None)


def _qkv_linear(h3, x=BUF, ldx=500, w=BUF, ldw=256, ws=BUF, k=500, gq=BUF, gk=BUF, table=BUF, rot=128,
                rounding=0, S=4, pad=128, H=2, D=128, q=BUF, ko=BUF, v=BUF, work=BUF, size=1 << 20):
    return h3.lib().h3hip_qkv_linear_mx4(x, ldx, w, ldw, ws, k, gq, gk, 1e-6, table, rot, rounding,
                                         S, pad, H, D, q, ko, v, work, size, None)


LINEAR = [(dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"),
          (dict(ldx=499), "ldx"), (dict(ldw=240), "ldw"), (dict(ldw=264), "ldw"),
          (dict(x=at(1)), "aligned"), (dict(w=at(8)), "aligned"), (dict(ws=at(2)), "aligned"),
          (dict(ldw=1 << 26), "2 GiB"), (dict(k=1 << 25, ldx=1 << 26, ldw=1 << 25), "2 GiB"),
          (dict(work=None), "workspace"), (dict(work=at(8)), "workspace")]


@pytest.mark.parametrize("bad,word", LINEAR + [
    (dict(k=0), "shape"), (dict(n=0), "shape"), (dict(rows=-1), "shape"), (dict(y=None), "NULL"),
    (dict(ldy=63), "ldy"), (dict(y=at(1)), "aligned"), (dict(size=4 * 256 + 255), "workspace")])
def test_linear(h3, bad, word):
    from h3hip import _lib
    assert _linear(h3, **bad) == _lib.EINVAL and word in h3.last_error()


@pytest.mark.parametrize("bad,word", LINEAR + [
    (dict(k=0), "hidden"), (dict(S=0), "shape"), (dict(H=0), "shape"), (dict(pad=64), "shape"),
    (dict(gq=None), "gammas"), (dict(table=None), "table"), (dict(rounding=2), "rounding"),
    (dict(q=None), "NULL"), (dict(v=at(8)), "aligned"), (dict(size=4 * 256 + 255), "workspace"),
    (dict(S=2, size=2 * 256 + 255), "workspace")])
def test_qkv_linear(h3, bad, word):
    from h3hip import _lib
    assert _qkv_linear(h3, **bad) == _lib.EINVAL and word in h3.last_error()


def test_linear_workspace(h3):
    """Codes and scales of the rows; none for one or two rows, nor where there is nothing to do."""
    from h3hip import _lib
    size = h3.lib().h3hip_linear_mx4_workspace
    assert size(4, 500) == 4 * 256 + 256
    assert size(100, 5120) == 100 * 2560 + 10 * 7 * 256
    assert size(1, 8) == size(2, 504) == 0
    assert size(2, 500) == 2 * 256 + 256        # not a multiple of 8 columns
    assert size(2, 200_000) == 2 * 100_096 + 391 * 256    # codes past the LDS
    assert size(0, 500) == size(4, 0) == size(-1, -1) == 0
    assert _linear(h3, rows=0, x=None, y=None, work=None, size=0) == _lib.OK
    for bad in (dict(D=64), dict(rot=64)):
        assert _qkv_linear(h3, **bad) == _lib.DECLINED and "declined" in h3.last_error()


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def _op(S, K):
    from h3hip import ops
    return ops.Mx4Rows.pack(_u8(S, -(-K // 2)), _u8(S, -(-2 * (-(-K // 2)) // 32)), K)


def test_rows_wrappers(h3):
    from h3hip import ops
    bf = torch.zeros((4, 200), dtype=torch.bfloat16)
    for x, word in ((bf, "GPU"), (bf.t(), "unit column stride"), (bf[:, :0], "K > 0"),
                    (bf.float(), "bfloat16"), (bf[0], "2-D")):
        with pytest.raises(ValueError, match=word):
            ops.quant_rows_mx4(x)
    for r, word in ((bf, "Mx4Rows"), (_op(4, 200), "GPU"),
                    (_op(4, 200)._replace(cols=300), "columns"),
                    (_op(4, 200)._replace(cols=0), "sizes"),
                    (_op(4, 200)._replace(scale=_u8(1, 2, 64, 4)), "scale"),
                    (_op(4, 200)._replace(scale=torch.zeros((1, 1, 64, 4))), "scale"),
                    (_op(4, 200)._replace(values=_u8(4, 100)), "values"),
                    (_op(4, 200)._replace(values=_u8(128, 4).t()), "unit column stride")):
        with pytest.raises(ValueError, match=word):
            ops.dequant_rows_mx4(r)


def test_pack(h3):
    from h3hip import ops
    for codes, e, cols, word in (
            (torch.zeros((4, 16)), _u8(4, 1), None, "codes"), (_u8(4, 0), _u8(4, 0), None, "codes"),
            (_u8(64), _u8(4, 1), None, "codes"), (_u8(4, 16), _u8(4, 2), None, "exponents"),
            (_u8(4, 16), torch.zeros((4, 1)), None, "exponents"), (_u8(4, 16), _u8(4, 1), 33, "cols"),
            (_u8(4, 16), _u8(4, 1), 0, "cols")):
        with pytest.raises(ValueError, match=word):
            ops.Mx4Rows.pack(codes, e, cols)


@pytest.mark.parametrize("S,K", [(1, 1), (17, 33), (40, 1001), (3, 512)])
def test_pack_lays_scales_out_as_documented(h3, S, K):
    """Every exponent at its place, zeros at all others, values past the columns zero."""
    from h3hip import ops
    g = torch.Generator()
    g.manual_seed(S + K)
    n = -(-K // 2)
    codes = torch.randint(1, 256, (S, n), generator=g, dtype=torch.uint8)
    e = torch.randint(1, 256, (S, -(-2 * n // 32)), generator=g, dtype=torch.uint8)
    rows = ops.Mx4Rows.pack(codes, e, K)
    nb = -(-K // 32)
    left = rows.scale.clone()
    for r in range(S):
        for b in range(nb):
            i = (b // 16, r // 16, 16 * (b % 4) + r % 16, b // 4 % 4)
            assert rows.scale[i] == e[r, b]
            left[i] = 0
    assert not left.any() and torch.equal(rows.exponents(), e[:, :nb])
    want = codes.clone()
    if K % 2:
        want[:, -1] &= 15
    assert torch.equal(rows.values[:, :n], want) and not rows.values[:, n:].any()
    assert rows.shape == (S, K)


def test_product_wrappers(h3):
    from h3hip import ops
    bf = torch.zeros((4, 200), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="Mx4Rows"):
        ops.proj_mx4(bf, bf)
    with pytest.raises(ValueError, match="GPU"):
        ops.proj_mx4(bf, _op(8, 200))
    with pytest.raises(ValueError, match="GPU"):
        ops.qkv_proj_mx4(bf, _op(384, 200), heads=1)


def _meta(*shape, dtype=torch.uint8):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("S,K", [(1, WIDE), (2, 2 ** 31), (WIDE, 1)])
def test_sizes_past_32_bits(h3, S, K):
    from h3hip import ops
    with pytest.raises(ValueError, match="2\\^31"):
        ops.quant_rows_mx4(_meta(S, K, dtype=torch.bfloat16))
    rows = ops.Mx4Rows(_meta(S, -(-K // 256) * 128), _meta(-(-K // 512), -(-S // 16), 64, 4), K)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.dequant_rows_mx4(rows)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.proj_mx4(rows, rows)


def test_some_of_the_rows(h3):
    g = torch.Generator()
    g.manual_seed(1)
    from h3hip import ops
    codes = torch.randint(0, 256, (70, 20), generator=g, dtype=torch.uint8)
    e = torch.randint(0, 256, (70, 2), generator=g, dtype=torch.uint8)
    rows = ops.Mx4Rows.pack(codes, e, 39)
    for first, count in ((0, 70), (16, 16), (32, 5), (48, 22), (64, 0)):
        part, want = rows.rows(first, count), ops.Mx4Rows.pack(codes[first:first + count],
                                                               e[first:first + count], 39)
        assert torch.equal(part.values, want.values) and part.cols == 39
        assert torch.equal(part.exponents(), want.exponents())
        assert part.scale.shape == want.scale.shape
    for first, count in ((8, 4), (64, 7), (-16, 4), (0, -1)):
        with pytest.raises(ValueError, match="multiple of 16"):
            rows.rows(first, count)


@pytest.mark.parametrize("rows,k", [(1, 512), (2, 512), (1, 500), (3, 512), (16_776_961, 512)])
def test_too_many_rows_or_channels(h3, rows, k):
    """No launch holds them: refused before the rows are rounded, by the form for few rows too."""
    from h3hip import _lib
    n = 64 if rows > 3 else 16_776_961
    big = dict(rows=rows, k=k, ldx=512, n=n, ldy=1 << 26, size=1 << 50)
    assert _linear(h3, **big) == _lib.EINVAL and "too many" in h3.last_error()
    heads = 1 if rows > 3 else 43_691          # 3 * 43,691 * 128 channels
    pad = (rows + 127) // 128 * 128
    assert (_qkv_linear(h3, S=rows, pad=pad, k=k, ldx=512, H=heads, size=1 << 50) == _lib.EINVAL
            and "too many" in h3.last_error())
