"""CPU: the package imports where torch has none of what only CUDA builds have."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_torch_without_cuda_or_8_bit_floats():
    """The router, dispatch and expert half needs neither names of torch's CUDA binding nor its 8-bit type to be imported."""
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "del torch.float8_e4m3fn\n"
            "from basalt_b200 import moe, paged\n"
            "print(moe.block_norm.__name__, paged.KVCache.__name__)\n")
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]
    assert got.stdout.split() == ["block_norm", "KVCache"]
