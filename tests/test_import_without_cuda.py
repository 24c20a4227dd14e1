"""The package on a torch built without CUDA: it imports, and its operators refuse CPU tensors."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
for name in [n for n in vars(torch._C) if n.startswith("_cuda_")]:  # a CPU-only build has none of them
    delattr(torch._C, name)
from spilltune_b200 import attention, codec, dense, dp, head, library, moe, nf4dq, ops, rotary, streaming
x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
r = torch.zeros(1, 4, dtype=torch.int32)
for call in (lambda: attention.attend(x, x, x, r, r), lambda: rotary.rotate(x, x, r, torch.ones(32))):
    try:
        call()
    except ValueError as e:
        assert "need CUDA tensors" in str(e), e
    else:
        raise AssertionError("no refusal")
assert attention.row_ranges(1, 2)[1].tolist() == [[1, 2]]
print("refused")
"""


def test_imports_and_refuses():
    out = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == ["refused"]
