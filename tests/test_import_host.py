"""h3hip's modules import, and its host tables work, on a torch built without a GPU backend
(CPU only, in a process of its own): such a torch._C has no stream or device functions."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "minimax-h3-swift_amd")

PROGRAM = """
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    delattr(torch._C, name)
from h3hip import ops, layer
assert ops.positions_grid(2, 1, 2, 2).shape == (6, 3)
"""


def test_modules_import_without_a_gpu_backend():
    env = dict(os.environ, PYTHONPATH=PKG)
    run = subprocess.run([sys.executable, "-c", PROGRAM], env=env, capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
