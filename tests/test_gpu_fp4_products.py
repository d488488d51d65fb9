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


# few rows, the fused kernel or two fp4 operands (one tile, several, ragged), the weight dequantized once
@pytest.mark.parametrize("mode", products.MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("m,n,k", [(2, 264, 320), (7, 264, 320), (16, 264, 320), (40, 264, 320), (129, 520, 1056), (300, 520, 1056),
                                   (600, 1048, 544), (1030, 2568, 288)])
def test_a_row_does_not_depend_on_the_others(cuda, mode, compute, m, n, k):
    """Rows keep their bits whatever stands in the other rows of the same batch,
    the last one of a ragged tile among them."""
    g = rng(m)
    lin, _ = products._weight(g, n, k, mode)
    lin.set_compute(compute)
    x = products._bf16(products._values(g, (m, k)))
    want = lin(x)
    keep = torch.zeros(m, dtype=torch.bool, device="cuda")
    keep[torch.from_numpy(g.permutation(m)[: max(1, m // 5)]).cuda()] = True
    for last in (True, False):
        keep[m - 1] = last
        if not keep.any():
            continue
        for others in (products._bf16(products._values(g, (m, k), "wide")), torch.full_like(x, float("nan")),
                       torch.full_like(x, float("inf")), torch.zeros_like(x)):
            got = lin(torch.where(keep[:, None], x, others))
            assert torch.equal(got[keep], want[keep])
