"""CPU checks around the paged key-value cache: the package on a torch without CUDA,
what the C ABI refuses at its limits, and the documented bindings."""
import os
import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_package_imports_on_a_torch_without_cuda():
    """Such a torch lacks the raw stream call; the package imports and refuses per call."""
    code = """
import torch
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    del torch._C._cuda_getCurrentRawStream
import nnop
pool, i32 = torch.zeros(2, 1, 16, 16), torch.int32
try:
    nnop.paged_attention(pool[:1, :, :1], pool, pool, torch.zeros(1, 1, dtype=i32), torch.zeros(1, dtype=i32))
except nnop.NNopError as e:
    assert "CUDA tensors only" in str(e)
else:
    raise SystemExit("not refused")
"""
    env = dict(os.environ, PYTHONPATH=str(ROOT / "onionop.jl_b200"), CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1000:]
