"""Rotary positions on the GPU against the definition in 64 bits.

Tolerance of a rotated element: one rounding to the output type (2^-8 of the
value for bf16, 2^-24 for fp32), plus scale * (|u| + |v|) times the error of an
fp32 rotation: 2^-24 each for the fp32 angle, cos and sin (two roundings),
their scaling, the products and the sum, at most 2^-21 in all, and the angle's
own 2^-46 of its size (two fp32 parts of position and frequency, 2^-48 each;
2^-51 in fp64).  bf16 results are formed with the hardware's cos and sin, each
within 2^-20.9: 2^-19.9 for both, and 2^-19.5 with the roundings above.
"""

import numpy as np
import pytest
import torch

from helpers import rng

pytestmark = pytest.mark.gpu


def _exact(x, pos, freqs, axes, layout, scale, inverse, eps=2.0 ** -21):
    """x (B, T, H, D) float64; pos (B, A, T); freqs, axes (H, R/2): rotated values and tolerance sizes."""
    half = freqs.shape[1]
    ang = np.zeros(x.shape[:3] + (half,))
    for h in range(freqs.shape[0]):
        for i in range(half):
            ang[:, :, h, i] = pos[:, axes[h, i], :] * freqs[h, i]
    c, s = scale * np.cos(ang), scale * np.sin(ang) * (-1 if inverse else 1)
    lo, hi = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y, size = x.copy(), np.zeros_like(x)
    u, v = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
    e = abs(scale) * (np.abs(u) + np.abs(v)) * (eps + 2.0 ** -46 * np.abs(ang))
    size[..., lo], size[..., hi] = e, e
    return y, size


def _run(b, t, heads, d, r, layout, dtype, *, per_head=False, n_axes=1, pos_type=torch.int64, far=1000, scale=1.0,
         inverse=False, form="rows", seed=0):
    import ltxq

    g = rng(seed)
    half = r // 2
    x = torch.from_numpy(g.standard_normal((b, t, heads, d)).astype(np.float32)).to(dtype)
    freqs = 10000.0 ** (-np.arange(half * (heads if per_head else 1)) / max(1, half)) if half else np.zeros(0)
    freqs = freqs.reshape((heads, half) if per_head else (half,))
    axes = g.integers(0, n_axes, freqs.shape).astype(np.int32)
    pos = g.integers(-far, far + 1, (b, n_axes, t)).astype(np.float64)
    if pos_type.is_floating_point:
        pos += g.integers(0, 4, pos.shape) / 4
    p = torch.from_numpy(pos).to(pos_type).cuda()
    xc = x.cuda()
    if form == "rows":
        xin = xc.view(b, t, heads * d)
    elif form == "slice":
        wide = torch.zeros(b, t, heads * d * 2 + 8, dtype=dtype, device="cuda")
        xin = wide[..., 8:8 + heads * d]
        xin.copy_(xc.view(b, t, heads * d))
    elif form == "odd":  # off the 16-byte grid
        wide = torch.zeros(b, t, heads * d + 3, dtype=dtype, device="cuda")
        xin = wide[..., 1:1 + heads * d]
        xin.copy_(xc.view(b, t, heads * d))
    else:  # (B, heads, T, D) seen as (B, T, heads, D)
        xin = xc.transpose(1, 2).contiguous().transpose(1, 2)
    before = xin.clone()
    out = ltxq.rotary(xin, p if n_axes > 1 else p[:, 0], torch.from_numpy(freqs).cuda(), heads, layout=layout,
                      axes=torch.from_numpy(axes).cuda() if n_axes > 1 else None, scale=scale, inverse=inverse)
    assert out.shape == xin.shape and out.dtype == dtype and out.is_contiguous() and torch.equal(xin, before)
    y, size = _exact(x.double().numpy(), p.double().cpu().numpy(), np.broadcast_to(freqs, (heads, half)),
                     np.broadcast_to(axes, (heads, half)), layout, scale, inverse,
                     2.0 ** -19.5 if dtype == torch.bfloat16 else 2.0 ** -21)
    tol = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) * np.abs(y) + size
    err = np.abs(out.double().cpu().numpy().reshape(y.shape) - y)
    err[..., r:] = np.where(out.double().cpu().numpy().reshape(y.shape)[..., r:] == y[..., r:], 0, np.inf)  # untouched
    assert (err <= tol).all(), (np.max(err - tol), np.unravel_index(np.argmax(err - tol), err.shape))


SHAPES = [(1, 1, 1, 2, 2), (1, 1, 32, 128, 128), (2, 5, 3, 64, 32), (1, 33, 7, 80, 36), (3, 17, 4, 48, 16),
          (2, 130, 8, 64, 64), (1, 9, 2, 96, 0), (1, 3, 5, 33, 20), (1, 700, 32, 128, 64), (1, 2, 1, 4096, 4096)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(cuda, layout, dtype, shape):
    _run(*shape, layout, dtype, seed=1)
    _run(*shape, layout, dtype, seed=2, inverse=True, scale=1.25)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["slice", "odd", "heads"])
def test_strides(cuda, layout, dtype, form):
    _run(2, 37, 6, 64, 48, layout, dtype, form=form)
    _run(2, 37, 6, 64, 64, layout, dtype, form=form, per_head=True, n_axes=3, pos_type=torch.float32)


@pytest.mark.parametrize("pos_type", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("n_axes", [1, 3])
def test_positions(cuda, pos_type, per_head, n_axes):
    _run(2, 50, 4, 64, 64, "half", torch.float32, per_head=per_head, n_axes=n_axes, pos_type=pos_type, far=1 << 20)
    _run(1, 50, 4, 32, 24, "interleaved", torch.bfloat16, per_head=per_head, n_axes=n_axes, pos_type=pos_type, far=60)


def test_far_positions(cuda):
    """Angles of 2^24 radians and of 2^40: the fp64 product's own error is all that grows."""
    _run(1, 64, 2, 64, 64, "half", torch.float32, far=1 << 24)
    _run(1, 64, 2, 64, 64, "half", torch.float32, far=1 << 24, pos_type=torch.float64, per_head=True)
    import ltxq

    f = torch.full((4,), 0.7, dtype=torch.float64, device="cuda")
    x = torch.zeros(1, 3, 8, device="cuda")
    x[..., :4] = 1
    p = torch.tensor([1 << 40, -(1 << 40), (1 << 51)], device="cuda")
    y = ltxq.rotary(x, p, f, 1).double().cpu().numpy()[0]
    a = p.cpu().numpy().astype(np.float64) * 0.7
    tol = 2.0 ** -21 + 2.0 ** -51 * np.abs(a)
    assert (np.abs(y[:, 0] - np.cos(a)) <= tol).all() and (np.abs(y[:, 4] - np.sin(a)) <= tol).all()


def test_inverse_undoes_and_is_the_gradient(cuda):
    """R' R = scale^2, and <R x, y> = <x, R' y> against differences of the fp64 definition."""
    import ltxq

    g = rng(3)
    x, y = (torch.from_numpy(g.standard_normal((2, 19, 3 * 40))).float().cuda() for _ in range(2))
    p = torch.from_numpy(g.integers(0, 5000, (2, 19))).cuda()
    f = torch.from_numpy(10000.0 ** (-np.arange(16) / 16)).cuda()
    for layout in ("half", "interleaved"):
        fw = ltxq.rotary(x, p, f, 3, layout=layout, scale=1.5)
        back = ltxq.rotary(fw, p, f, 3, layout=layout, scale=1.5, inverse=True).view(2, 19, 3, 40)
        xs = x.view(2, 19, 3, 40)
        assert (back[..., :32] - 2.25 * xs[..., :32]).abs().max() <= 2.25 * 2 * 5 * 2.0 ** -20
        assert torch.equal(back[..., 32:], xs[..., 32:])
        grad = ltxq.rotary(y, p, f, 3, layout=layout, scale=1.5, inverse=True).double()
        # loss <R x, y> is linear in x: its difference along a direction is the gradient's product with it
        dx = torch.from_numpy(g.standard_normal(tuple(x.shape))).cuda()
        one = np.zeros((3, 16), np.int32)
        fr = np.broadcast_to(f.cpu().numpy(), (3, 16))
        dy, _ = _exact(dx.cpu().numpy().reshape(2, 19, 3, 40), p.double().cpu().numpy()[:, None], fr, one, layout, 1.5, False)
        want = float((torch.from_numpy(dy).reshape(y.shape).cuda() * y.double()).sum())
        size = float((dx.abs() * y.double().abs()).sum()) * 3
        assert abs(float((grad * dx).sum()) - want) <= 2.0 ** -20 * size


def test_in_place_out_and_broadcast_positions(cuda):
    import ltxq

    x = torch.randn(2, 21, 4 * 64, device="cuda").bfloat16()
    f = torch.from_numpy(10000.0 ** (-np.arange(32) / 32)).cuda()
    p = torch.arange(21, device="cuda")
    want = ltxq.rotary(x, p, f, 4)
    assert torch.equal(ltxq.rotary(x, p[None].expand(2, -1), f, 4), want)
    assert torch.equal(ltxq.rotary(x.view(2, 21, 4, 64), p, f, 4).view(2, 21, 256), want)
    assert torch.equal(ltxq.rotary(x, p[None, None].expand(2, 3, -1), f, 4, axes=torch.zeros(32, dtype=torch.int32, device="cuda")), want)
    qkv = torch.zeros(2, 21, 3 * 256, dtype=torch.bfloat16, device="cuda")
    qkv[..., 256:512] = x
    k = qkv[..., 256:512]
    assert ltxq.rotary(k, p, f, 4, out=k) is k and torch.equal(k, want)
    assert (qkv[..., :256] == 0).all() and (qkv[..., 512:] == 0).all()
    assert ltxq.rotary(x[:, :0], p[:0], f, 4).shape == (2, 0, 256)


def test_bad_axis_and_position_give_nan(cuda):
    import ltxq

    x = torch.randn(1, 3, 2 * 8, device="cuda")
    f = torch.ones(4, dtype=torch.float64, device="cuda")
    ax = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device="cuda")
    p = torch.ones(2, 3, device="cuda")
    for freqs, axes in ((f, ax), (f.expand(2, 4), ax.expand(2, 4))):
        y = ltxq.rotary(x, p, freqs, 2, axes=axes).view(3, 2, 8)
        assert torch.equal(y.isnan()[0, 0], torch.tensor([0, 1, 1, 0] * 2, device="cuda").bool())
    p[0, 1] = float("inf")
    y = ltxq.rotary(x, p[0], f, 2)
    assert y.isnan()[0, 1].all() and y.isnan().sum() == 16


def test_refusals(cuda):
    import ltxq

    x = torch.randn(2, 3, 32, device="cuda")
    f = torch.ones(8, dtype=torch.float64, device="cuda")
    p = torch.arange(3, device="cuda")
    ok = lambda *a, **k: ltxq.rotary(*a, **k)  # noqa: E731
    ok(x, p, f, 2)
    for bad in ((x, p, f.float(), 2), (x, p, f, 3), (x, p, f, 0), (x.half(), p, f, 2), (x, p[:2], f, 2), (x, p.half(), f, 2),
                (x[0], p, f, 2), (x, p[None, None], f, 2), (x, p, f.expand(3, 8), 2), (x, p, torch.ones(9, dtype=torch.float64, device="cuda"), 2),
                (x, p, f.cpu(), 2), (x, p.cpu(), f, 2)):
        with pytest.raises(ValueError):
            ok(*bad)
    ax = torch.zeros(8, dtype=torch.int32, device="cuda")
    for kw in (dict(layout="split"), dict(axes=ax.long()), dict(axes=ax[:4]), dict(axes=ax), dict(out=x[:, :2]),
               dict(out=x.bfloat16()), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            ok(x, p, f, 2, **kw)


def test_captured_and_replayed(cuda):
    import ltxq

    x = torch.randn(1, 40, 256, device="cuda").bfloat16()
    f = torch.from_numpy(10000.0 ** (-np.arange(32) / 32)).cuda()
    p = torch.arange(40, device="cuda")
    want = [ltxq.rotary(x, p + i, f, 4) for i in range(3)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    q = p.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        out = ltxq.rotary(x, q, f, 4)
    for i in (1, 2, 0):
        q.copy_(p + i)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


@pytest.mark.parametrize("mode", ["mxfp4", "nvfp4"])
def test_projection_rotary_attention_run(cuda, mode):
    """The operators as they are used together: one quantized input serves the
    Q, K and V projections, Q and K are rotated in place by the model's grid
    positions, attention follows -- against the same run in 64 bits."""
    import ltxq
    from ltxq import kernels
    from ltxq.rope import grid_rotary, video_positions
    from oracle import fp4 as of

    heads, d, t, c = 4, 64, 2 * 6 * 5, 256
    g = rng(9)
    x = torch.from_numpy(g.standard_normal((1, t, c)).astype(np.float32)).bfloat16()
    lin, wv = [], []
    for _ in range(3):
        w = torch.from_numpy((g.standard_normal((heads * d, c)) * 0.06).astype(np.float32)).bfloat16()
        lin.append(ltxq.QuantizedLinear.from_linear(w.cuda(), mode=mode).set_compute("fp4"))
        wv.append(of.dequantize(*of.quantize(w.float().numpy(), mode), mode))
    pos, freqs, axes = grid_rotary(video_positions(1, 2, 6, 5, 24.0, device="cuda"), heads * d,
                                   use_middle_indices_grid=True, num_attention_heads=heads)
    xt = ltxq.FP4Tensor.quantize(x.cuda(), mode)
    q, k, v = (p(xt) for p in lin)
    for y in (q, k):
        ltxq.rotary(y, pos, freqs, heads, axes=axes, out=y)
    out = kernels.attention(q, k, v, heads).double().cpu().numpy()

    xe = of.dequantize(*of.quantize(x[0].float().numpy(), mode), mode)
    qe, ke, ve = (torch.from_numpy(xe @ w.T).bfloat16().double().numpy().reshape(1, t, heads, d) for w in wv)
    args = (pos.cpu().numpy(), freqs.cpu().numpy(), axes.cpu().numpy(), "half", 1.0, False)
    qe, ke = (torch.from_numpy(_exact(y, *args)[0]).bfloat16().double().numpy()[0] for y in (qe, ke))
    s = np.einsum("qhd,khd->hqk", qe, ke) / np.sqrt(d)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    want = np.einsum("hqk,khd->qhd", w, ve[0]).reshape(1, t, heads * d)
    # q, k, v and the weights each carry a bf16 rounding: a score is off by at most 2 * 2^-8 |q||k| / sqrt(d), which
    # changes the softmax by that much again, relative; V, P and the result add 2^-8 each, relative to max |v|
    ds = 2 * 2.0 ** -8 * np.max(np.linalg.norm(qe, axis=-1)) * np.max(np.linalg.norm(ke, axis=-1)) / np.sqrt(d)
    assert np.abs(out - want).max() <= np.abs(ve).max() * (2 * ds + 4 * 2.0 ** -8)
