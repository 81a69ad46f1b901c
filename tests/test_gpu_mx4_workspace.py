"""Both 4-bit projections of a layer through the C entry points with one workspace, as large as the
wider of them needs, on one stream: the bits of calls with workspaces of their own, eager and
replayed from a graph."""
import ctypes

import pytest
import torch

from _gpu import note
from _mx4 import bits16

pytestmark = pytest.mark.gpu

HEADS, HIDDEN = 7, 640         # padded to 1,024 and 768 columns
INNER = 128 * HEADS


@pytest.mark.parametrize("S", [1, 3, 40, 300])
def test_one_workspace_for_both_projections(h3, S):
    from h3hip import _lib, ops
    lib = h3.lib()
    g = torch.Generator(device="cuda")
    g.manual_seed(S)
    x, merged, qkv_w, out_w = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in (
        (S, HIDDEN), (S, INNER), (3 * INNER, HIDDEN), (HIDDEN, INNER)))
    qkv_w, out_w = ops.quant_rows_mx4(qkv_w), ops.quant_rows_mx4(out_w)
    need = [lib.h3hip_linear_mx4_workspace(S, k) for k in (HIDDEN, INNER)]
    assert need[1] >= need[0] and (S < 3 or need[1] > need[0])
    pad = (S + 127) // 128 * 128
    want = ops.qkv_proj_mx4(x, qkv_w, heads=HEADS), ops.proj_mx4(merged, out_w)
    work = torch.empty(max(need[1], 1), dtype=torch.uint8, device="cuda")
    heads = torch.empty((3, HEADS, pad, 128), dtype=torch.bfloat16, device="cuda")
    y = torch.empty((S, HIDDEN), dtype=torch.bfloat16, device="cuda")

    def calls(size=max(need)):
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        a = lib.h3hip_qkv_linear_mx4(
            x.data_ptr(), HIDDEN, qkv_w.values.data_ptr(), qkv_w.values.stride(0),
            qkv_w.scale.data_ptr(), HIDDEN, None, None, 1e-6, None, 128, 0, S, pad, HEADS, 128,
            heads[0].data_ptr(), heads[1].data_ptr(), heads[2].data_ptr(), work.data_ptr(), size, st)
        b = lib.h3hip_linear_mx4(
            merged.data_ptr(), INNER, out_w.values.data_ptr(), out_w.values.stride(0),
            out_w.scale.data_ptr(), INNER, HIDDEN, S, y.data_ptr(), HIDDEN, work.data_ptr(), size, st)
        return a, b

    def check():
        torch.cuda.synchronize()
        for t, w in zip(heads, want[0]):
            assert (bits16(t) == bits16(w)).all()
        assert (bits16(y) == bits16(want[1])).all()

    note(f"qkv_linear_mx4 and linear_mx4 with one workspace S={S}")
    assert calls() == (_lib.OK, _lib.OK)
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert calls() == (_lib.OK, _lib.OK)
    for _ in range(3):
        heads.fill_(7.0), y.fill_(7.0), work.fill_(0x55)
        torch.cuda.synchronize()
        graph.replay()
        check()
    if S >= 3:      # of the narrower's size the wider is refused
        assert calls(need[0]) == (_lib.OK, _lib.EINVAL) and "workspace" in h3.last_error()
        torch.cuda.synchronize()
