"""Sizes that the library's 32-bit parameters cannot hold are refused by the torch wrappers
before the call (CPU only: tensors without memory). ctypes would cut them: 2^32 + 128 columns
arrived as 128, and quant_rows() left the rest of its output as it was."""
import pytest
import torch

WIDE = 2 ** 32 + 128


def _meta(*shape, dtype):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("S,K", [(1, WIDE), (2, 2 ** 31), (WIDE, 1)])
def test_quant_rows(h3, S, K):
    from h3hip import ops
    with pytest.raises(ValueError, match="2\\^31"):
        ops.quant_rows(_meta(S, K, dtype=torch.bfloat16))


@pytest.mark.parametrize("S,K,N", [(1, WIDE, 1), (WIDE, 128, 384), (1, 128, WIDE)])
def test_projections(h3, S, K, N):
    from h3hip import ops
    args = (_meta(S, K, dtype=torch.int8), _meta(S, dtype=torch.float32),
            _meta(N, K, dtype=torch.int8), _meta(N, dtype=torch.float32))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.proj_i8(*args)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.qkv_proj_i8(*args, heads=1)


def test_rows_that_overlap(h3):
    """The one way in which such operands passed the library's check of strides."""
    from h3hip import ops
    x = _meta(WIDE + 128, dtype=torch.int8).as_strided((2, WIDE), (128, 1))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.proj_i8(x, _meta(2, dtype=torch.float32), x, _meta(2, dtype=torch.float32))


def test_sizes_that_fit_go_on_to_the_next_check(h3):
    from h3hip import ops
    with pytest.raises(ValueError, match="GPU"):
        ops.quant_rows(_meta(1, 2 ** 31 - 1, dtype=torch.bfloat16))
