"""Outputs in the buffer of the bf16 rows they are computed from: refused on top of one or two rows,
which the product's launch reads while it writes, and right wherever they are taken."""
import pytest
import torch

from _gpu import note
from _mx4 import bits16, mx4_operand

pytestmark = pytest.mark.gpu


def _x(S, K, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn((S, K), generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("S", [1, 2])
def test_few_rows_in_place_are_refused(h3, S):
    from h3hip import ops
    from h3hip._lib import H3HIPError
    x, w = _x(S, 512), mx4_operand(512, 512, 2)
    kept = x.clone()
    with pytest.raises(H3HIPError, match="overlap"):
        ops.proj_mx4(x, w, out=x)
    out = torch.zeros((3, 1, 128, 128), dtype=torch.bfloat16, device="cuda")
    inside = out[2, 0].view(-1)[1024:1024 + S * 512].view(S, 512)
    with pytest.raises(H3HIPError, match="overlap"):
        ops.qkv_proj_mx4(inside, mx4_operand(384, 512, 3), heads=1, out=out.unbind(0))
    torch.cuda.synchronize()
    assert torch.equal(x, kept) and not out.any()


@pytest.mark.parametrize("S", [1, 2, 3, 40])
def test_beside_the_rows_in_one_buffer(h3, S):
    from h3hip import ops
    w = mx4_operand(264, 512, 4)
    buf = _x(S, 512 + 264)
    x, y = buf[:, :512], buf[:, 512:]
    want = ops.proj_mx4(x.clone(), w)
    note(f"proj_mx4 beside its rows S={S}")
    assert ops.proj_mx4(x, w, out=y) is y
    assert (bits16(y) == bits16(want)).all()


@pytest.mark.parametrize("S", [3, 40, 300])
def test_more_rows_in_place(h3, S):
    """They are rounded before the product begins."""
    from h3hip import ops
    x, w = _x(S, 512), mx4_operand(512, 512, 5)
    want = ops.proj_mx4(x.clone(), w)
    note(f"proj_mx4 in place S={S}")
    ops.proj_mx4(x, w, out=x)
    assert (bits16(x) == bits16(want)).all()
