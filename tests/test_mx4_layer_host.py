"""What a 4-bit layer and a block refuse when they are made (CPU only: weights without
memory)."""
import pytest
import torch


def _rows(out, inp):
    from h3hip.ops import Mx4Rows
    pad = (inp + 255) // 256 * 128
    return Mx4Rows(torch.empty((out, pad), dtype=torch.uint8, device="meta"),
                   torch.empty(((inp + 511) // 512, (out + 15) // 16, 64, 4), dtype=torch.uint8,
                               device="meta"), inp)


def _layer(hidden=256, heads=2, out=None, projection="mx4"):
    from h3hip.layer import AttentionLayer
    gamma = torch.empty(128, dtype=torch.bfloat16, device="meta")
    return AttentionLayer(_rows(384 * heads, hidden), _rows(out or hidden, 128 * heads), gamma, gamma,
                          heads=heads, projection=projection)


def test_layer(h3):
    from h3hip.layer import AttentionLayer
    assert _layer().projection == "mx4"
    for projection in ("fused", "hipblaslt"):
        with pytest.raises(ValueError, match="mx4"):
            _layer(projection=projection)
    with pytest.raises(ValueError, match="'mx4'"):
        _layer(projection="fp4")
    gamma = torch.empty(128, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="heads"):
        AttentionLayer(_rows(384, 256), _rows(256, 256), gamma, gamma, heads=2, projection="mx4")


def test_block(h3):
    from h3hip.layer import AttentionBlock
    assert AttentionBlock(_layer(16384)).residual_scale == 1.0
    with pytest.raises(NotImplementedError, match="16385"):
        AttentionBlock(_layer(16385))
    with pytest.raises(ValueError, match="out features"):
        AttentionBlock(_layer(256, out=300))


def test_the_widths_limit_is_the_librarys(h3):
    from h3hip import _lib, ops
    from test_norm_refusals import _before, _norm
    for hidden, rc in ((ops.NORM_MAX_HIDDEN + 1, _lib.DECLINED), (ops.NORM_MAX_HIDDEN, _lib.EINVAL)):
        big = dict(hidden=hidden, ldx=20000, ldh=20000, norm=_norm(ld_scale=20000, ld_shift=20000))
        assert _before(h3, x=None, **big) == rc     # then: a NULL operand
