"""4-bit floating point on the GPU (mxfp4, nvfp4): quantizers, readers and both
products, against the numpy oracle in 64 bits.

Tolerances.  Quantizing and reading back are exact.  A product's output is the
fp32 sum of exact terms, rounded to bf16: off by at most half a bf16 step
(2^-9 to 2^-8 of the value: eps / 2 = 2^-8) plus what K fp32 additions may
lose, K * 2^-23 of the sum of the terms' magnitudes (one unit, not half, per
addition: tensor cores may truncate).
"""

import numpy as np
import pytest
import torch

from helpers import from_dev_bf16, rng
from oracle import fp4 as of

pytestmark = pytest.mark.gpu

MODES = ["mxfp4", "nvfp4"]


def _bf16(a):
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).cuda()


def _values(g, shape, kind="normal"):
    """bf16 values as float32: normal, or over many binades with zeros and exact ties among them."""
    a = g.standard_normal(shape)
    if kind == "wide":
        a = a * np.exp2(g.integers(-40, 40, shape[:-1] + (1,)))
        a[g.random(shape) < 0.1] = 0.0
    elif kind == "grid":  # multiples of a quarter: quotients hit the midpoints
        a = np.round(a * 8) / 4
    elif kind == "tiny":  # down to bf16's subnormals
        a = a * np.exp2(g.integers(-140, -110, shape[:-1] + (1,)))
    return torch.from_numpy(a.astype(np.float32)).to(torch.bfloat16).float().numpy()


def _weight(g, n, k, mode, gs=1.0, std=0.02, bias=False):
    """A QuantizedLinear over the oracle's arrays, and the weight's values in float64."""
    import ltxq

    w = _values(g, (n, k)) * std
    codes, scales = of.quantize(w, mode, gs)
    lin = ltxq.QuantizedLinear(torch.from_numpy(of.pack(codes)).cuda().view(torch.uint32), torch.from_numpy(scales).cuda(),
                               None, _bf16(g.standard_normal(n)) if bias else None, group_size=of.GROUP[mode], bits=4,
                               mode=mode, global_scale=gs)
    return lin, of.dequantize(codes, scales, mode, gs)


def _check(out, x, w, k):
    exact = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    err = np.abs(from_dev_bf16(out).astype(np.float64) - exact)
    tol = 2.0 ** -8 * np.abs(exact) + k * 2.0 ** -23 * size
    worst = np.max(err - tol)
    assert worst <= 0, (worst, np.unravel_index(np.argmax(err - tol), err.shape))


# ---------------------------------------------------------------- quantizers

SHAPES = [(1, 32), (1, 256), (3, 96), (31, 288), (128, 512), (129, 2080), (300, 4096)]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("kind", ["normal", "wide", "grid", "tiny"])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_is_exact(cuda, mode, kind, rows, k):
    import ltxq

    x = _values(rng(rows + k), (rows, k), kind)
    for gs in (1.0,) if mode == "mxfp4" else (1.0, 2.0 ** -6, 2.0 ** 5):
        t = ltxq.FP4Tensor.quantize(_bf16(x), mode, gs)
        codes, scales = of.quantize(x, mode, gs)
        got_c, got_s = (a.cpu().numpy() for a in t.tensors())
        assert np.array_equal(of.scale_atoms(scales, rows, k, mode)[_owned(rows, k, mode)], got_s[_owned(rows, k, mode)])
        assert np.array_equal(of.unpack(got_c), codes)
        v = of.dequantize(codes, scales, mode, gs)
        assert np.array_equal(from_dev_bf16(t.dequantize()), torch.from_numpy(v).to(torch.bfloat16).float().numpy())


def _owned(rows, k, mode):
    """Scale bytes that some row owns (the last row tile's others are not written)."""
    g = of.GROUP[mode]
    full = np.zeros((-(-rows // 128) * 128, -(-k // 256) * 256 // g), np.uint8)
    full[:rows] = 1
    return of.scale_atoms(full, full.shape[0], full.shape[1] * g, mode).astype(bool)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("n,k", [(8, 32), (40, 96), (129, 2080), (64, 4096)])
def test_weight_quantize_is_exact(cuda, mode, n, k):
    import ltxq

    for gs in (1.0,) if mode == "mxfp4" else (1.0, 2.0 ** -6):
        w = _values(rng(n), (n, k)) * np.float32(0.02)
        w = torch.from_numpy(w).to(torch.bfloat16).float().numpy()
        lin = ltxq.QuantizedLinear.from_linear(_bf16(w), mode=mode, global_scale=gs)
        codes, scales = of.quantize(w, mode, gs)
        assert lin.weight.dtype == torch.uint32 and lin.weight.shape == (n, k // 8)
        assert np.array_equal(lin.weight.cpu().view(torch.uint8).numpy(), of.pack(codes))
        assert np.array_equal(lin.scales.cpu().numpy(), scales)
        v = torch.from_numpy(of.dequantize(codes, scales, mode, gs)).to(torch.bfloat16).float().numpy()
        assert np.array_equal(from_dev_bf16(lin.dequantize()), v)
        lin.set_compute("fp4")
        want = of.scale_atoms(scales, n, k, mode)
        assert np.array_equal(lin.mx_scales().cpu().numpy(), want)


def test_nvfp4_odd_global_scale(cuda):
    """A tensor scale that is no power of two: x / g in fp32, then the formats' rule."""
    import ltxq

    gs = 0.0123
    x = _values(rng(5), (64, 512))
    y = (x / np.float32(gs)).astype(np.float32).astype(np.float64)
    codes, scales = of.quantize(y, "nvfp4")
    t = ltxq.FP4Tensor.quantize(_bf16(x), "nvfp4", gs)
    s = of.scale_values(scales, "nvfp4").astype(np.float32)
    q = np.abs(y.astype(np.float32)).reshape(64, -1, 16) / np.where(s > 0, s, np.float32(1))[..., None]  # fp32 quotient
    codes = (of.nearest(q.astype(np.float64), of.E2M1).reshape(64, 512) + 8 * np.signbit(x)).astype(np.uint8)
    assert np.array_equal(of.unpack(t.tensors()[0].cpu().numpy()), codes)
    v = of.E2M1[codes & 7] * np.where(codes & 8, -1, 1) * np.repeat(of.scale_values(scales, "nvfp4"), 16, axis=1)
    v = (v.astype(np.float32) * np.float32(gs)).astype(np.float32)
    assert np.array_equal(from_dev_bf16(t.dequantize()), torch.from_numpy(v).to(torch.bfloat16).float().numpy())


@pytest.mark.parametrize("mode", MODES)
def test_every_code_and_scale(cuda, mode):
    """Every scale byte with every code, read back: exact in float64, rounded once to bf16."""
    import ltxq

    g = of.GROUP[mode]
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, g // 16))
    codes = np.concatenate([codes, codes], axis=1) if g == 16 else codes
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], codes.shape[1] // g, axis=1)
    lin = ltxq.QuantizedLinear(torch.from_numpy(of.pack(codes)).cuda().view(torch.uint32), torch.from_numpy(scales).cuda(),
                               group_size=g, bits=4, mode=mode)
    v = torch.from_numpy(of.dequantize(codes, scales, mode)).to(torch.bfloat16).float().numpy()
    got = from_dev_bf16(lin.dequantize())
    assert np.array_equal(np.isnan(got), np.isnan(v))
    assert np.array_equal(got[~np.isnan(v)], v[~np.isnan(v)])


@pytest.mark.parametrize("mode", MODES)
def test_non_finite_groups(cuda, mode):
    import ltxq

    x = _values(rng(3), (5, 256))
    x[1, 40], x[2, 41], x[4, 255] = np.inf, np.nan, -np.inf
    t = ltxq.FP4Tensor.quantize(_bf16(x), mode)
    v = of.dequantize(*of.quantize(x, mode), mode)
    got = from_dev_bf16(t.dequantize())
    assert np.array_equal(np.isnan(got), np.isnan(v)) and np.isnan(v).sum() == 3 * of.GROUP[mode]
    assert np.array_equal(got[~np.isnan(v)], v[~np.isnan(v)].astype(np.float32))


def test_quantize_strided_empty_and_refused(cuda):
    import ltxq

    x = _values(rng(7), (33, 192))
    wide = _bf16(np.concatenate([x, x, x], axis=1))
    want = ltxq.FP4Tensor.quantize(_bf16(x), "nvfp4").dequantize()
    assert torch.equal(ltxq.FP4Tensor.quantize(wide[:, 192:384], "nvfp4").dequantize(), want)
    odd = torch.empty(33, 201, dtype=torch.bfloat16, device="cuda")  # rows off 16 bytes: copied
    odd[:, 1:193] = _bf16(x)
    assert torch.equal(ltxq.FP4Tensor.quantize(odd[:, 1:193], "nvfp4").dequantize(), want)
    assert torch.equal(ltxq.FP4Tensor.quantize(_bf16(x.T.copy()).t(), "nvfp4").dequantize(), want)
    assert torch.equal(ltxq.FP4Tensor.quantize(_bf16(x).view(3, 11, 192), "nvfp4").dequantize().view(33, 192), want)
    assert torch.equal(ltxq.FP4Tensor.quantize(_bf16(x[:1])[0], "nvfp4").dequantize(), want[0])
    assert ltxq.FP4Tensor.quantize(_bf16(x)[:0], "nvfp4").dequantize().shape == (0, 192)
    with pytest.raises(ValueError):
        ltxq.FP4Tensor.quantize(torch.zeros(4, 64, device="cuda"), "nvfp4")
    with pytest.raises(ValueError):
        ltxq.FP4Tensor.quantize(torch.zeros(4, 48, dtype=torch.bfloat16, device="cuda"), "nvfp4")


# ---------------------------------------------------------------- products

PRODUCTS = [(1, 8, 32), (1, 16, 64), (2, 24, 96), (5, 136, 288), (8, 1024, 512), (9, 1048, 2080), (17, 200, 1056),
            (64, 256, 256), (65, 264, 320), (129, 384, 2048), (200, 2048, 1024), (257, 520, 4096), (513, 192, 544),
            (700, 4096, 256), (1030, 264, 96), (1200, 2056, 544), (2050, 4104, 800)]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_dequantizing_product(cuda, mode, m, n, k):
    g = rng(m * n + k)
    lin, w = _weight(g, n, k, mode, 1.0 if mode == "mxfp4" else 0.0156)
    x = _values(g, (m, k))
    _check(lin(_bf16(x)), x.astype(np.float64), w, k)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_fp4_product(cuda, mode, m, n, k):
    import ltxq

    g = rng(m * n + k + 1)
    gs = 1.0 if mode == "mxfp4" else 0.0156
    lin, w = _weight(g, n, k, mode, gs)
    lin.set_compute("fp4")
    x = _values(g, (m, k))
    xq = of.dequantize(*of.quantize(x, mode), mode)
    out = lin(_bf16(x))
    _check(out, xq, w, k)
    t = ltxq.FP4Tensor.quantize(_bf16(x), mode)
    assert torch.equal(lin(t), out)  # one quantized tensor, the same product
    if mode == "nvfp4":
        t = ltxq.FP4Tensor.quantize(_bf16(x), mode, 0.25)
        _check(lin(t), of.dequantize(*of.quantize(x, mode, 0.25), mode, 0.25), w, k)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("m,n,k", [(3, 264, 512), (40, 1032, 288), (300, 456, 1024), (1100, 1536, 512)])
def test_epilogues(cuda, mode, compute, m, n, k):
    """Bias, GELU and both gated residuals equal the same epilogue applied by
    an identity-free recomputation: the plain product's bf16 output followed by
    the oracle's elementwise steps, bit for bit."""
    from oracle import ref_ops as ro
    from oracle.bf16 import rbf16

    g = rng(m + n)
    lin, _ = _weight(g, n, k, mode, bias=True)
    lin.set_compute(compute)
    x = _bf16(_values(g, (m, k)))
    bias, lin.bias = lin.bias, None
    plain = from_dev_bf16(lin(x))
    lin.bias = bias
    y = rbf16(plain + from_dev_bf16(bias)[None])
    assert np.array_equal(from_dev_bf16(lin(x)), y)
    assert np.array_equal(from_dev_bf16(lin(x, gelu=True)), ro.gelu_approx(y))
    res = _values(g, (m, n))
    gate = g.standard_normal(n).astype(np.float32)
    got = from_dev_bf16(lin(x, residual=_bf16(res), gate=torch.from_numpy(gate).cuda()[None]))
    assert np.array_equal(got, rbf16(res + y * gate[None]))
    got = from_dev_bf16(lin(x, residual=_bf16(res), gate=torch.from_numpy(gate).cuda()[None], gate_then_add=True))
    assert np.array_equal(got, rbf16(res + rbf16(y * gate[None])))
    rows = g.standard_normal((m, n)).astype(np.float32)
    got = from_dev_bf16(lin(x, residual=_bf16(res), gate=torch.from_numpy(rows).cuda()))
    assert np.array_equal(got, rbf16(res + y * rows))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("m", [1, 7, 40, 200, 700])
def test_nan_stays_in_its_row(cuda, mode, compute, m):
    """A NaN in one row of x or one group of the weight reaches that row's or
    that feature's outputs, and no other."""
    g = rng(m)
    lin, w = _weight(g, 256, 512, mode)
    lin.set_compute(compute)
    x = _values(g, (m, 512))
    x[m // 2, 77] = np.nan
    nan = np.isnan(from_dev_bf16(lin(_bf16(x))))
    assert nan[m // 2].all() and nan.sum() == 256
    lin.scales[100, 3] = 255 if mode == "mxfp4" else 127
    x[m // 2, 77] = 0.0
    nan = np.isnan(from_dev_bf16(lin(_bf16(x))))
    assert nan[:, 100].all() and nan.sum() == m


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
def test_rows_do_not_depend_on_their_neighbours(cuda, mode, compute):
    """The same row in a larger batch, at the same kernel's tile, twice over: repeats are bit-identical."""
    g = rng(11)
    lin, _ = _weight(g, 520, 1056, mode)
    lin.set_compute(compute)
    x = _bf16(_values(g, (600, 1056)))
    a, b = lin(x), lin(x)
    assert torch.equal(a, b)
    assert torch.equal(lin(x.view(3, 200, 1056)).view(600, 520), a)
    assert lin(x[:0]).shape == (0, 520)


@pytest.mark.parametrize("mode", MODES)
def test_adaln_feed_forward_and_prologue(cuda, mode):
    """The AdaLN prologue and the feed-forward run the same kernels: equal to
    their parts called one by one."""
    import ltxq

    gen = torch.Generator("cuda").manual_seed(1)
    w1 = (torch.randn(1024, 256, generator=gen, device="cuda") * 0.05).bfloat16()
    w2 = (torch.randn(256, 1024, generator=gen, device="cuda") * 0.05).bfloat16()
    x = torch.randn(2, 90, 256, generator=gen, device="cuda").bfloat16()
    scale, shift = (torch.randn(2, 1, 256, generator=gen, device="cuda") * 0.1 for _ in range(2))
    for compute in ("dequant", "fp4"):
        ff = ltxq.FeedForward.from_linear(w1, None, w2, None, mode=mode)
        ff.project_in.set_compute(compute)
        ff.project_out.set_compute(compute)
        h = ltxq.adaln_modulate(x, scale, shift, 1e-6)
        want = ff.project_out(ff.project_in(h, gelu=True))
        assert torch.equal(ff(h), want)
        assert torch.equal(ff.project_in(x, adaln=(scale, shift, 1e-6)), ff.project_in(h))


@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("m", [1, 33, 300])
def test_captured_and_replayed_on_another_stream(cuda, compute, m):
    g = rng(2)
    lin, _ = _weight(g, 512, 1024, "nvfp4")
    lin.set_compute(compute)
    xs = [_bf16(_values(g, (m, 1024))) for _ in range(3)]
    want = [lin(x) for x in xs]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    x = xs[0].clone()
    graphs = []
    for _ in range(2):  # two graphs of the same call: their workspaces are their own
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = lin(x)
        graphs.append((gr, out))
    for i in (1, 2, 0):
        x.copy_(xs[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for gr, _ in graphs:
                gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want[i])


def test_product_refusals(cuda):
    import ltxq

    g = rng(4)
    lin, _ = _weight(g, 64, 64, "nvfp4")
    x = _bf16(_values(g, (4, 64)))
    t = ltxq.FP4Tensor.quantize(x, "nvfp4")
    with pytest.raises(ValueError):
        lin(t)  # dequantizing compute takes bf16
    lin.set_compute("fp4")
    with pytest.raises(ValueError):
        lin(ltxq.FP4Tensor.quantize(x, "mxfp4"))
    with pytest.raises(ValueError):
        lin(ltxq.FP4Tensor.quantize(_bf16(_values(g, (4, 96))), "nvfp4"))
    with pytest.raises(ValueError):
        lin(x.float())
    with pytest.raises(ValueError):
        lin(t, adaln=(x, x, 1e-6))
    with pytest.raises(ValueError):
        lin(x, mx_out=1)
    with pytest.raises(ValueError):
        ltxq.QuantizedLinear.from_linear(torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda"), global_scale=2.0)
    assert lin(x, split_k=False).shape == (4, 64)


def test_allocation_free_entry_and_fp4_compute(cuda):
    """It has no workspace for quantized activations: a few rows, which need none, run; more are an error."""
    import ctypes

    from ltxq import _lib

    lin, _ = _weight(rng(4), 64, 64, "nvfp4")
    lin.set_compute("fp4")
    x = torch.randn(40, 64, device="cuda").bfloat16()
    out = torch.zeros(40, 64, dtype=torch.bfloat16, device="cuda")
    z = torch.zeros(64, device="cuda")
    v = _lib.Vec(z.data_ptr(), _lib.F32, 0, 0, 0)
    q = lin.qweight()
    call = lambda m: _lib.load().ltxq_adaln_qlinear_noalloc(  # noqa: E731
        x.data_ptr(), m, ctypes.byref(_lib.Prologue(_lib.NORM_RMS, 1e-6, v, v)), ctypes.byref(q), None, out.data_ptr(), None)
    torch.cuda.synchronize()
    assert call(40) == _lib.ERR_INVALID
    torch.cuda.synchronize()
    assert (out == 0).all()
    assert call(4) == _lib.OK
    torch.cuda.synchronize()
    assert torch.equal(out[:4], lin(x[:4], adaln=(z, z, 1e-6))) and (out[4:] == 0).all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(1, 16384, 4096), (4, 40, 16384), (7, 2408, 2080), (8, 4096, 8192), (16, 2048, 4096),
                                   (12, 1000, 4064), (16, 8, 32), (3, 3000, 96)])
def test_few_rows(cuda, mode, m, n, k):
    """Single tokens and short batches over every number of feature tiles and K blocks, from bf16 rows, quantized in
    the call and quantized before it."""
    import ltxq

    g = rng(m + n + k)
    lin, w = _weight(g, n, k, mode, 1.0 if mode == "mxfp4" else 0.0156)
    x = _values(g, (m, k))
    _check(lin(_bf16(x)), x.astype(np.float64), w, k)
    lin.set_compute("fp4")
    xq = of.dequantize(*of.quantize(x, mode), mode)
    out = lin(_bf16(x))
    _check(out, xq, w, k)
    assert torch.equal(lin(ltxq.FP4Tensor.quantize(_bf16(x), mode)), out)


@pytest.mark.parametrize("m", [2, 40, 300])
def test_large_mxfp4_scales(cuda, m):
    """Scales above 2 leave the one-multiplication decoding: groups of every size beside one another."""
    g = rng(m)
    n, k = 264, 512
    codes = g.integers(0, 16, (n, k)).astype(np.uint8)
    scales = g.choice(np.array([0, 1, 100, 127, 128, 129, 140, 200], np.uint8), (n, k // 32))
    scales[:64] = 127
    import ltxq

    lin = ltxq.QuantizedLinear(torch.from_numpy(of.pack(codes)).cuda().view(torch.uint32), torch.from_numpy(scales).cuda(),
                               group_size=32, bits=4, mode="mxfp4")
    x = _values(g, (m, k))
    _check(lin(_bf16(x)), x.astype(np.float64), of.dequantize(codes, scales, "mxfp4"), k)


def test_weights_made_in_inference_mode(cuda):
    import ltxq

    with torch.inference_mode():
        w = torch.randn(64, 64, device="cuda").bfloat16()
        lin = ltxq.QuantizedLinear.from_linear(w, mode="nvfp4").set_compute("fp4")
        x = torch.randn(40, 64, device="cuda").bfloat16()
        assert torch.equal(lin(x), lin(ltxq.FP4Tensor.quantize(x, "nvfp4")))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(1, 5000, 512), (3, 2600, 4064), (16, 40, 1056)])
def test_few_rows_of_any_range(cuda, mode, m, n, k):
    """Rows whose values span all of bf16: none is lost beside one many binades larger, whatever the weight has there."""
    g = rng(n)
    lin, w = _weight(g, n, k, mode)
    x = _values(g, (m, k)) * np.exp2(g.integers(-60, 60, (m, k))).astype(np.float32)
    x[:, 0] = 2.0 ** 100  # alone decides the result, except where the weight is zero
    x[0, 1:k // 2] = 0.0
    x[m - 1, 5] = 2.0 ** -130
    lin.scales[: n // 2, 0] = 0 if mode == "nvfp4" else 104  # (almost) nothing of the largest value
    sc = lin.scales.cpu().numpy()
    w = of.dequantize(of.unpack(lin.weight.cpu().view(torch.uint8).numpy()), sc, mode)
    out = lin(_bf16(x))
    exact = x.astype(np.float64) @ w.T
    size = np.abs(x).astype(np.float64) @ np.abs(w).T
    err = np.abs(from_dev_bf16(out).astype(np.float64) - exact)
    assert (err <= 2.0 ** -8 * np.abs(exact) + k * 2.0 ** -23 * size + 2.0 ** -126).all()
    # a row with an infinity: where its weight is not zero, infinite or NaN; the other rows as they were
    x[0, 3] = np.inf
    again = from_dev_bf16(lin(_bf16(x)))
    assert np.array_equal(again[1:], from_dev_bf16(out)[1:])
    assert (~np.isfinite(again[0][w[:, 3] != 0])).all()
