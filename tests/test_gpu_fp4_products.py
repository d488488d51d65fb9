"""Products over fp4 weights: what one kernel is chosen by, and what a row's result may depend on."""

import pytest
import torch

import test_gpu_fp4 as products
from helpers import rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", products.MODES)
@pytest.mark.parametrize("m,n,k", [(768, 4096, 96), (1024, 5120, 544), (1550, 2048, 256), (200, 2048, 544)])
def test_unsplit_products_run_the_same_kernels(cuda, mode, m, n, k):
    """``split_k=False`` leaves out the split tiles' sum and nothing else."""
    from ltxq import _lib

    g = rng(m + n)
    lin, w = products._weight(g, n, k, mode)
    x = products._values(g, (m, k))
    xd = products._bf16(x)

    def run(split_k):
        torch.cuda.synchronize()
        before = _lib.launch_count()
        out = lin(xd, split_k=split_k)
        return out, _lib.launch_count() - before

    split, unsplit = run(True), run(False)
    products._check(split[0], x.astype("float64"), w, k)
    products._check(unsplit[0], x.astype("float64"), w, k)
    dense = m >= 768  # the weight dequantized once, then the product
    assert unsplit[1] == (2 if dense else 1) and split[1] - unsplit[1] in (0, 1)
    if not dense or n == 5120:
        assert split[1] - unsplit[1] == 1  # these have tiles to split
