"""h3hip_quant_rows_mx4 on blocks that hold a large value and far smaller ones: every bf16 magnitude,
both signs and all subnormals among them, under the scale of every larger exponent, value for
value against the format's definition in 64 bits."""
import numpy as np
import pytest
import torch

from _gpu import note
from _mx4 import quant64, unpack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", range(0, 255, 15))
def test_every_value_under_every_larger_scale(h3, first):
    """A block's largest magnitude is the first of an exponent field (its scale's), beside 31 of all
    the values below the field's end; 15 fields a test."""
    from h3hip import ops
    for field in range(first, first + 15):
        head = field << 7
        below = np.arange(head + 128, dtype=np.int64)
        blocks = -(-len(below) // 31)
        bits = np.zeros((blocks, 32), dtype=np.int64)
        bits[:, 1:].flat[:len(below)] = below
        bits[:, 0] = np.maximum(bits.max(1), head)
        bits = np.concatenate([bits, bits | 0x8000]).astype(np.uint16).reshape(1, -1)
        x = torch.from_numpy(bits.view(np.int16)).cuda().view(torch.bfloat16)
        if field == first:
            note(f"quant_rows_mx4 every value under fields {first} to {first + 14}")
        rows = ops.quant_rows_mx4(x)
        codes, e = quant64(x.double().cpu().numpy())
        got = unpack(rows.values)[:, :bits.size]
        bad = np.flatnonzero((got != codes)[0])
        assert not len(bad), (field, [hex(bits[0, i]) for i in bad[:8]], got[0, bad[:8]], codes[0, bad[:8]])
        assert (rows.exponents().cpu().numpy() == e).all(), field
        assert (e == max(field - 2, 0)).all(), field
