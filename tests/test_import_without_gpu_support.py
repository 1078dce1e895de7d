"""A torch built without GPU support lacks the raw device and stream queries: the package still
imports there, and its entry points refuse host tensors by name."""
import os
import subprocess
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import importlib
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream", "_cuda_isCurrentStreamCapturing"):
    delattr(torch._C, name)
pkg = importlib.import_module("llm-serve_amd")
lengths = torch.zeros(1, dtype=torch.int32)
try:
    pkg.kv_step(lengths, lengths, lengths[None], lengths, block_size=16, num_tokens=1)
except ValueError as e:
    print("refused:", e)
"""


def test_import_without_the_gpu_queries():
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "refused: KV step lengths must be GPU" in done.stdout
