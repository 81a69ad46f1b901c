"""How wide the reduction of a 4-bit linear call may be: 16,776,960, since 256 rows of codes are
reached with 32-bit offsets. Wider ones, and more rows than a launch holds, are refused before any
device call, and no workspace is asked for what every call refuses (CPU only)."""
import ctypes

import pytest

BUF = ctypes.c_void_p(4096)       # an aligned address no refused call reads
WIDEST = 16_776_960


def _linear(h3, k, rows=4, work=None, size=0):
    pad = (k + 255) // 256 * 256
    return h3.lib().h3hip_linear_mx4(BUF, k, BUF, pad // 2, BUF, k, 64, rows, ctypes.c_void_p(1 << 40),
                                     64, work, size, None)


def _qkv(h3, k, rows=4):
    pad = (k + 255) // 256 * 256
    return h3.lib().h3hip_qkv_linear_mx4(BUF, k, BUF, pad // 2, BUF, k, BUF, BUF, 1e-6, BUF, 128, 0,
                                         rows, (rows + 127) // 128 * 128, 1, 128, BUF, BUF, BUF, None,
                                         0, None)


@pytest.mark.parametrize("call", [_linear, _qkv])
def test_widest_reduction(h3, call):
    """At the limit only the workspace is missing; one column more is refused for its width."""
    from h3hip import _lib
    assert call(h3, WIDEST) == _lib.EINVAL and "workspace" in h3.last_error()
    for k in (WIDEST + 1, 33_553_920, 2 ** 31 - 1):
        assert call(h3, k) == _lib.EINVAL and "2 GiB" in h3.last_error()


def test_header_states_the_limit(h3):
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "ch3hip.h")).read()
    start = text.index("h3hip_proj_mx4 of bf16 rows")
    said = text[start:text.index("int h3hip_linear_mx4(", start)]
    assert "16,776,960" in said and "33,553,920" not in said


def test_no_workspace_for_what_is_refused(h3):
    size = h3.lib().h3hip_linear_mx4_workspace
    assert size(4, WIDEST) == 4 * (WIDEST // 2) + 256 * 32_768
    assert size(4, WIDEST + 1) == size(4, 33_553_920) == size(1000, 2 ** 31 - 1) == 0
    assert size(WIDEST, 256) == WIDEST * 128 + 256 * (WIDEST // 16)
    assert size(WIDEST + 1, 256) == size(2 ** 31 - 1, 2 ** 31 - 1) == 0
