"""What the 8-bit operators refuse, and what they do not depend on."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import double_attention as da


def test_import_without_device_support() -> None:
    """A torch that was built for the CPU alone lacks the private device calls:
    the package and its torch backend work there."""

    code = """
import sys
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
sys.path.insert(0, sys.argv[1])
import double_attention as da
config = da.experiment_config("a1", backend="torch", model_dim=32, routing_dim=8, dictionary_size=16)
model = da.DoubleAttentionLM(50, 12, config, 2, feedforward_dim=48, norm="rms")
assert model(torch.zeros(1, 5, dtype=torch.int64))[0].shape == (1, 5, 50)
"""
    package = Path(da.__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code, str(package)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
