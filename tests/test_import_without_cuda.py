"""The package's host side (descriptors, validation, sharding) needs no CUDA build of torch."""
import os
import subprocess
import sys

import pytest

pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

IMPORT = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)         # a CPU build has none of them
import batchlas_b200 as bl
assert bl.shard_range(10, 0, 2) is not None
try:
    bl.quantize_i8(torch.zeros(2, 3))
except RuntimeError as e:
    assert "CUDA" in str(e)
else:
    raise AssertionError("a host tensor was accepted")
print("imported")
"""


def test_import_on_a_build_of_torch_without_cuda(lib):
    out = subprocess.run([sys.executable, "-c", IMPORT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "imported" in out.stdout, out.stderr[-2000:]
