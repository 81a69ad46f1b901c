"""An int8 layer whose reductions are longer than the int8 kernels' sums hold is refused when
it is made (CPU only: weights without memory). h3hip_proj_i8 declines such a width, and the
layer returned that call's None as its output."""
import pytest
import torch


def _weight(out, inp):
    from h3hip.layer import Int8Weight
    pad = (inp + 127) // 128 * 128
    return Int8Weight(torch.empty((out, pad), dtype=torch.int8, device="meta"),
                      torch.empty(out, device="meta"), inp)


def _layer(h3, hidden, heads):
    from h3hip.layer import AttentionLayer
    gamma = torch.empty(128, dtype=torch.bfloat16, device="meta")
    return AttentionLayer(_weight(384 * heads, hidden), _weight(hidden, 128 * heads), gamma, gamma,
                          heads=heads, projection="int8")


@pytest.mark.parametrize("hidden,heads,name", [
    (256, 1024, "out_weight"),         # 131,072 in features of the out-projection
    (131072, 2, "qkv_weight"),
    (130945, 2, "qkv_weight")])        # 131,072 padded
def test_too_long_a_reduction(h3, hidden, heads, name):
    with pytest.raises(NotImplementedError, match=name):
        _layer(h3, hidden, heads)


@pytest.mark.parametrize("hidden,heads", [(130944, 2), (256, 1023)])
def test_the_longest_are_taken(h3, hidden, heads):
    assert _layer(h3, hidden, heads).projection == "int8"


def test_the_limit_is_the_librarys(h3):
    from h3hip import _lib, ops
    from test_int8_refusals import _proj
    limit = ops.INT8_MAX_REDUCTION // 128 * 128
    for k, rc in ((limit + 128, _lib.DECLINED), (limit, _lib.EINVAL)):   # then: a NULL operand
        assert _proj(h3, x=None, k=k, ldx=1 << 20, ldw=1 << 20) == rc
