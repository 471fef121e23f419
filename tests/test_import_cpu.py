"""The package on a torch build without the private functions that its host path takes for speed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice", "_cuda_isCurrentStreamCapturing"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
sys.path.insert(0, {pkg!r})
import atflash
from atflash import _lib, cache, hf, interface, ops
assert _lib.current_device.__module__ == "torch.cuda" and callable(_lib.capturing)
try:
    ops.decode_paged_q8(*[torch.zeros(1)] * 5, 16, None, 0.1, None, 0)
except ValueError as e:
    assert "GPU only" in str(e)
else:
    raise SystemExit("a CPU tensor was taken")
print("imported")
"""


def test_imports_without_the_private_functions():
    code = CODE.format(pkg=os.path.join(ROOT, "atflash-kernel_amd"))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("imported"), run.stderr
