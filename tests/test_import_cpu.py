"""The package imports, and says what is missing when called, on a torch that was built without CUDA."""
import os
import subprocess
import sys

ROOT = os.path.join(os.path.dirname(__file__), "..")


def test_imports_without_torchs_cuda_bindings():
    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from openattention_b200 import flash, kv4, llama, method, rotary
x = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
i = torch.zeros(1, dtype=torch.int32)
t = torch.zeros(8, 128)
for call in (lambda: rotary.qk_norm_rope(x, x, t, t, i),
             lambda: kv4.decode_attention(x, torch.zeros(1, 2, 3, 144, dtype=torch.uint8), i)):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA" in str(e), e
    else:
        raise SystemExit("not refused")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
