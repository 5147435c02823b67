"""The package without a CUDA build of torch."""

import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent / "bridge-aware-kv-cache-eviction-for-efficient-long-context-transformers_b200"

SCRIPT = """
import sys, torch
for name in [x for x in dir(torch._C) if x.startswith("_cuda")]:
    delattr(torch._C, name)
sys.path.insert(0, sys.argv[1])
import cab_attention
from cab_attention.kernels import tree_attention
x = torch.zeros(1, 2, 1, 64)
i = torch.zeros(1, 1, dtype=torch.int32)
try:
    tree_attention(x, x, x, i, i[0])
except RuntimeError as e:
    assert "no CPU implementation" in str(e), e
    print("refused")
"""


def test_imports_without_cuda_in_torch():
    done = subprocess.run([sys.executable, "-c", SCRIPT, str(PKG)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "refused", done.stderr
