"""The int8 projections' reduction loops (csrc/gen_gemm_i8_loop.py ->
csrc/gemm_i8_loop.inc): the bf16 loops' stream with the int8 product, so the replay
of test_gemm_loop_gen.py runs on it with that product's name put back."""
import importlib.util
import os

import pytest

import test_gemm_loop_gen as bf16

CSRC = bf16.CSRC
spec = importlib.util.spec_from_file_location("gen_gemm_i8_loop",
                                              os.path.join(CSRC, "gen_gemm_i8_loop.py"))
G = importlib.util.module_from_spec(spec)
spec.loader.exec_module(G)

INT8, BF16 = "v_mfma_i32_16x16x64_i8", "v_mfma_f32_16x16x32_bf16"


def _lines(name):
    g = G.Gen(name)
    lines = [ln.replace("%=", "") for ln in g.generate()]
    assert not any(BF16 in ln for ln in lines)
    return g, [ln.replace(INT8, BF16) for ln in lines]


def test_generated_file_is_current():
    assert open(G.OUT).read() == G.render()


@pytest.mark.parametrize("name", list(G.VARIANTS))
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7, 12, 25])
def test_every_step_once_and_nothing_early(name, steps):
    g, lines = _lines(name)
    assert g.lds <= 163840 and g.n_vgpr <= 256
    bf16.replay(g, lines, steps)


@pytest.mark.parametrize("name", list(G.VARIANTS))
@pytest.mark.parametrize("mistake", list(bf16.PLANTED))
def test_replay_finds_a_planted_mistake(name, mistake):
    g, lines = _lines(name)
    with pytest.raises(bf16.Wrong):
        bf16.replay(g, bf16.PLANTED[mistake](lines), 13)
