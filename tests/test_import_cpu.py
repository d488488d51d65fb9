"""The package imports, and the parts that need no GPU work, where torch was built without CUDA."""

import os
import subprocess
import sys

CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)  # what such a build lacks
import ltxq
from ltxq import cache, cache_build, denoise, kernels, latents, perturbations, rope
assert rope.video_positions(1, 2, 3, 2, 24.0).shape[0] == 1
assert rope.rotary_frequencies(64)[0].numel() == 32
"""


def test_torch_without_cuda():
    env = dict(os.environ, PYTHONPATH=os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-2-mlx_b200"))
    r = subprocess.run([sys.executable, "-c", CODE], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
