"""The Python modules import where PyTorch has no device support: host work (registry, plan files) needs none."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
del torch._C._cuda_getCurrentRawStream          # what a PyTorch built without a device lacks
from forward_amd import lib, ops, torch_ops
assert lib.dll.fwdmi_registry_size() == 6
try:
    ops.linear(torch.zeros(2, 4), torch.zeros(3, 4))
except RuntimeError as e:
    print("refused:", e)
"""


def test_imports_without_device_support():
    p = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "refused: input must be a tensor in device memory" in p.stdout, p.stdout + p.stderr
