"""Where one kernel hands over to the next: the borders of the rules on rows and
tiles, scales that start at odd addresses, rows of heads that fill a CTA in part
or several of them.  Tolerances are those of the two operators' own tests."""

import numpy as np
import pytest
import torch

import test_gpu_fp4 as products
import test_gpu_rotary as rotations
from helpers import rng
from oracle import fp4 as of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", products.MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("m,n,k", [(16, 264, 320), (17, 264, 320), (16, 8, 32), (17, 8, 32), (767, 4096, 96), (768, 4096, 96),
                                   (768, 3840, 160), (769, 4104, 32), (33, 2048, 2080), (256, 520, 1056)])
def test_borders_of_the_rules(cuda, mode, compute, m, n, k):
    g = rng(m + n + k)
    lin, w = products._weight(g, n, k, mode)
    lin.set_compute(compute)
    x = products._values(g, (m, k))
    xv = of.dequantize(*of.quantize(x, mode), mode) if compute == "fp4" else x.astype(np.float64)
    products._check(lin(products._bf16(x)), xv, w, k)


@pytest.mark.parametrize("mode", products.MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("offset", [1, 2])
@pytest.mark.parametrize("m", [4, 40, 800])
def test_scales_at_odd_addresses(cuda, mode, compute, offset, m):
    g = rng(m)
    n, k = (4096 if m == 800 else 72), 192
    lin, w = products._weight(g, n, k, mode)
    wide = torch.zeros(lin.scales.numel() + offset, dtype=torch.uint8, device="cuda")
    moved = wide[offset:].view(lin.scales.shape)
    moved.copy_(lin.scales)
    lin.scales = moved
    lin.set_compute(compute)
    assert lin.scales.data_ptr() % 4 == offset
    x = products._values(g, (m, k))
    xv = of.dequantize(*of.quantize(x, mode), mode) if compute == "fp4" else x.astype(np.float64)
    products._check(lin(products._bf16(x)), xv, w, k)


PER_HEAD = [(1, 41, 40, 128, 128), (2, 1300, 3, 36, 36), (1, 5, 33, 6, 2), (3, 700, 5, 33, 20), (1, 2500, 8, 64, 64),
            (1, 1, 32, 128, 128), (1, 1, 1, 2, 2), (5, 7, 9, 80, 48), (1, 9, 70, 64, 32)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", PER_HEAD)
def test_rows_of_frequencies(cuda, layout, dtype, shape):
    rotations._run(*shape, layout, dtype, per_head=True, seed=4)
    rotations._run(*shape, layout, dtype, per_head=True, n_axes=3, pos_type=torch.float64, seed=5, inverse=True, scale=0.75)


def test_many_axes(cuda):
    for n_axes in (600, 2048):
        rotations._run(2, 7, 6, 64, 64, "half", torch.float32, per_head=True, n_axes=n_axes, pos_type=torch.float64)
