"""CPU checks of the 4-bit floating point and rotary entry points: the oracle's
own definitions, refusals before any CUDA call, and the frequency tables."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import fp4 as of


@pytest.fixture(scope="module")
def lib():
    from ltxq import _lib

    return _lib.load()


# ---------------------------------------------------------------- formats


def test_e4m3_table_is_the_format():
    assert of.E4M3[0] == 0 and of.E4M3[1] == 2.0 ** -9 and of.E4M3[8] == 2.0 ** -6 and of.E4M3[126] == 448
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, of.E4M3)


def test_ties_go_to_the_even_code():
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    assert of.nearest(v, of.E2M1).tolist() == [0, 2, 2, 4, 4, 6, 6, 7]


@pytest.mark.parametrize("mode", ["mxfp4", "nvfp4"])
def test_round_trip_of_representable_values(mode):
    codes = np.arange(16, dtype=np.uint8).repeat(4).reshape(1, 64).copy()
    codes[0, :] = np.random.default_rng(0).permutation(codes[0])
    codes[0, ::16] = 7  # every group holds its largest magnitude
    s = np.full((1, 64 // of.GROUP[mode]), 130 if mode == "mxfp4" else 0x38, np.uint8)
    x = of.dequantize(codes, s, mode)
    c2, s2 = of.quantize(x, mode)
    assert np.array_equal(s, s2)
    assert np.array_equal(of.dequantize(c2, s2, mode), x)


def test_non_finite_groups_read_back_as_nan():
    for mode in of.GROUP:
        for bad in (np.inf, -np.inf, np.nan):
            x = np.ones((1, 64))
            x[0, 3] = bad
            v = of.dequantize(*of.quantize(x, mode), mode)
            g = of.GROUP[mode]
            assert np.isnan(v[0, :g]).all() and np.isfinite(v[0, g:]).all()


def test_sizes_match_the_layout(lib):
    from ltxq import _lib

    for mode, name in ((_lib.MXFP4, "mxfp4"), (_lib.NVFP4, "nvfp4")):
        for rows, k in ((1, 32), (127, 256), (128, 288), (129, 4096), (9216, 16384)):
            c, s = ctypes.c_size_t(0), ctypes.c_size_t(0)
            assert lib.ltxq_fp4_sizes(rows, k, mode, ctypes.byref(c), ctypes.byref(s)) == -(-rows // 128)
            assert c.value == rows * k // 2
            if rows <= 129:
                assert s.value == of.scale_atoms(np.zeros((rows, k // of.GROUP[name]), np.uint8), rows, k, name).size
    assert lib.ltxq_fp4_sizes(4, 48, _lib.NVFP4, None, None) == 0
    assert lib.ltxq_fp4_sizes(4, 64, _lib.MXFP8, None, None) == 0
    assert lib.ltxq_fp4_sizes(0, 64, _lib.NVFP4, None, None) == 0


# ---------------------------------------------------------------- refusals (fake pointers: nothing is launched)


def test_fp4_refusals(lib):
    from ltxq import _lib

    act = _lib.Fp4Act(16, 16, _lib.NVFP4, 1.0)
    q = lambda *a: lib.ltxq_fp4_quantize(*a)  # noqa: E731
    assert q(None, 4, 64, 64, ctypes.byref(act), None) == _lib.ERR_INVALID
    assert q(16, 4, 64, 64, None, None) == _lib.ERR_INVALID
    assert q(16, -1, 64, 64, ctypes.byref(act), None) == _lib.ERR_INVALID
    assert q(16, 4, 48, 48, ctypes.byref(act), None) == _lib.ERR_UNSUPPORTED
    assert q(16, 4, 64, 32, ctypes.byref(act), None) == _lib.ERR_INVALID
    assert q(16, 4, 64, 68, ctypes.byref(act), None) == _lib.ERR_UNSUPPORTED
    assert q(24, 4, 64, 64, ctypes.byref(act), None) == _lib.ERR_UNSUPPORTED
    assert q(16, 4, 1 << 31, 1 << 31, ctypes.byref(act), None) == _lib.ERR_UNSUPPORTED
    for bad in (_lib.Fp4Act(16, 16, _lib.MXFP8, 1.0), _lib.Fp4Act(16, 16, _lib.MXFP4, 2.0),
                _lib.Fp4Act(16, 16, _lib.NVFP4, -1.0), _lib.Fp4Act(16, 16, _lib.NVFP4, float("nan")),
                _lib.Fp4Act(16, 16, _lib.NVFP4, 1e30), _lib.Fp4Act(None, 16, _lib.NVFP4, 1.0)):
        assert q(16, 4, 64, 64, ctypes.byref(bad), None) == _lib.ERR_INVALID
    assert q(16, 4, 64, 64, ctypes.byref(_lib.Fp4Act(24, 16, _lib.NVFP4, 1.0)), None) == _lib.ERR_UNSUPPORTED
    assert q(16, 0, 64, 64, ctypes.byref(act), None) == _lib.OK
    assert lib.ltxq_fp4_dequantize(ctypes.byref(act), 4, 64, None, None) == _lib.ERR_INVALID
    assert lib.ltxq_fp4_dequantize(ctypes.byref(act), 4, 64, 24, None) == _lib.ERR_UNSUPPORTED


def test_fp4_weight_refusals(lib):
    from ltxq import _lib

    def w(mode=_lib.NVFP4, bits=4, gs=16, n=64, k=64, layout=0, compute=0, scales=16, weight=16, mx=None, g=0.0):
        return ctypes.byref(_lib.QWeight(weight, scales, None, None, n, k, mode, bits, gs, layout, 0, compute, mx, g))

    deq = lambda q: lib.ltxq_dequantize(q, 16, None)  # noqa: E731
    assert deq(w(bits=8)) == _lib.ERR_UNSUPPORTED
    assert deq(w(gs=32)) == _lib.ERR_UNSUPPORTED
    assert deq(w(mode=_lib.MXFP4, gs=16)) == _lib.ERR_UNSUPPORTED
    assert deq(w(mode=4)) == _lib.ERR_UNSUPPORTED
    assert deq(w(k=72)) == _lib.ERR_UNSUPPORTED
    assert deq(w(mode=_lib.MXFP4, gs=32, g=2.0)) == _lib.ERR_INVALID
    assert deq(w(g=-1.0)) == _lib.ERR_INVALID
    assert deq(w(weight=24)) == _lib.ERR_UNSUPPORTED
    assert lib.ltxq_quantize(24, w(), None) == _lib.ERR_UNSUPPORTED
    lin = lambda q, m=4, x=16, out=16: lib.ltxq_qlinear(x, m, q, None, out, None, 0, None)  # noqa: E731
    assert lin(w(k=48)) == _lib.ERR_UNSUPPORTED
    assert lin(w(n=60)) == _lib.ERR_UNSUPPORTED
    assert lin(w(layout=_lib.LAYOUT_PRETRANSPOSED)) == _lib.ERR_UNSUPPORTED
    assert lin(w(weight=24)) == _lib.ERR_UNSUPPORTED
    assert lin(w(), x=8) == _lib.ERR_UNSUPPORTED
    assert lin(w(), m=-1) == _lib.ERR_INVALID
    assert lib.ltxq_fp4_weight_scales_size(w(mode=_lib.MXFP8, bits=8, gs=32)) == 0
    assert lib.ltxq_fp4_weight_scales_size(w(layout=_lib.LAYOUT_PRETRANSPOSED)) == 0
    assert lib.ltxq_fp4_pack_weight_scales(w(k=48), 16, None) == _lib.ERR_UNSUPPORTED
    assert lib.ltxq_fp4_pack_weight_scales(w(), 24, None) == _lib.ERR_UNSUPPORTED
    act = _lib.Fp4Act(16, 16, _lib.NVFP4, 1.0)
    f4 = lambda a, q, m=4, out=16: lib.ltxq_qlinear_fp4(a, m, q, None, out, None)  # noqa: E731
    assert f4(None, w()) == _lib.ERR_INVALID
    assert f4(ctypes.byref(act), w(), m=-1) == _lib.ERR_INVALID
    assert f4(ctypes.byref(act), w(mode=_lib.MXFP8, bits=8, gs=32)) == _lib.ERR_UNSUPPORTED
    assert f4(ctypes.byref(act), w(), out=None) == _lib.ERR_INVALID


def test_fp4_workspace_sizes(lib):
    from ltxq import _lib

    q = _lib.QWeight(16, 16, None, None, 4096, 2080, _lib.NVFP4, 4, 16, 0, 0, _lib.COMPUTE_FP4, 16, 1.0)
    need = lib.ltxq_qlinear_workspace_size(40, ctypes.byref(q))
    assert need >= 40 * 2080 // 2 + 9 * 4 * 512
    assert lib.ltxq_adaln_qlinear_workspace_size(40, ctypes.byref(q)) >= need + 40 * 2080 * 2
    assert lib.ltxq_qlinear_workspace_size(9, ctypes.byref(q)) == 0  # a few rows are quantized as they are read
    q.compute = _lib.COMPUTE_DEQUANT
    assert lib.ltxq_qlinear_workspace_size(2048, ctypes.byref(q)) >= 4096 * 2080 * 2
    assert lib.ltxq_qlinear_workspace_size(0, ctypes.byref(q)) == 0


def _rotary_args(**kw):
    from ltxq import _lib

    st = _lib.RotaryArgs(x=16, out=16, dtype=_lib.BF16, layout=_lib.ROTARY_HALF, batch=1, tokens=4, heads=2,
                         head_dim=64, rotary_dim=64, positions=16, pos_dtype=_lib.POS_I64, n_axes=1, freqs=16, scale=1.0)
    st.x_stride[:] = (512, 128, 64)
    st.out_stride[:] = (512, 128, 64)
    st.pos_stride[:] = (4, 0, 1)
    for k, v in kw.items():
        setattr(st, k, v)
    return ctypes.byref(st)


def test_rotary_refusals(lib):
    from ltxq import _lib

    call = lambda **kw: lib.ltxq_rotary(_rotary_args(**kw), None)  # noqa: E731
    assert lib.ltxq_rotary(None, None) == _lib.ERR_INVALID
    for kw in (dict(rotary_dim=63), dict(rotary_dim=66), dict(heads=0), dict(head_dim=0), dict(tokens=-1),
               dict(layout=2), dict(pos_dtype=4), dict(n_axes=0), dict(n_axes=2), dict(x=None), dict(freqs=None),
               dict(positions=None), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(**kw) == _lib.ERR_INVALID, kw
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED
    assert call(x=17) == _lib.ERR_UNSUPPORTED
    assert call(head_dim=8192, rotary_dim=4098) == _lib.ERR_UNSUPPORTED
    assert call(tokens=0) == _lib.OK
    assert call(batch=0) == _lib.OK


def test_python_refuses_cpu_tensors():
    import ltxq

    with pytest.raises(ValueError, match="CUDA"):
        ltxq.FP4Tensor.quantize(torch.zeros(4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        ltxq.rotary(torch.zeros(1, 4, 64), torch.arange(4), torch.ones(32, dtype=torch.float64), 1)


def test_fp4_tensor_arguments():
    import ltxq

    for kw in (dict(K=48), dict(K=0), dict(mode="fp4"), dict(mode="mxfp4", global_scale=2.0), dict(global_scale=0.0),
               dict(global_scale=float("nan"))):
        a = dict(K=64, mode="nvfp4", global_scale=1.0, **{}) | kw
        with pytest.raises(ValueError):
            ltxq.FP4Tensor((4,), a["K"], a["mode"], "cpu", a["global_scale"])
    t = ltxq.FP4Tensor((3, 5), 288, "nvfp4", "cpu")
    c, s = t.tensors()
    assert t.shape == (3, 5, 288) and c.shape == (15, 144) and s.numel() == 2 * 4 * 512


# ---------------------------------------------------------------- frequencies


def test_rotary_frequencies():
    from ltxq.rope import rotary_frequencies

    f, s = rotary_frequencies(64, 10000.0)
    assert s == 1.0 and f.dtype == torch.float64 and f[0] == 1 and math.isclose(float(f[-1]), 10000.0 ** (-62 / 64))
    lin, _ = rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4)
    ntk, _ = rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    y, s = rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    f = rotary_frequencies(128)[0]
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 32], f[turns > 32])
    assert torch.allclose(y[turns < 1], f[turns < 1] / 8, rtol=1e-15)
    assert (y <= f).all() and (y >= f / 8 * (1 - 1e-15)).all() and math.isclose(s, 0.1 * math.log(8) + 1)
    for kw in (dict(rotary_dim=63), dict(rotary_dim=64, scaling="other"), dict(rotary_dim=64, factor=2.0),
               dict(rotary_dim=64, scaling="yarn", factor=2.0), dict(rotary_dim=2, scaling="ntk", factor=2.0),
               dict(rotary_dim=64, scaling="linear", factor=0.5)):
        with pytest.raises(ValueError):
            rotary_frequencies(**kw)


@pytest.mark.parametrize("dim,heads", [(256, 4), (128, 2)])
def test_grid_rotary_matches_the_tables(dim, heads):
    """position * frequency reproduces the fp32 tables' angles: they are
    rounded to fp32 at up to theta * pi / 2 radians, 2^-24 relative in each of
    the grid, the scaled position (twice) and the product."""
    from ltxq.rope import THETA, grid_rotary, precompute_freqs_cis, video_positions

    grid = video_positions(2, 2, 3, 2, 24.0)
    cos, sin = precompute_freqs_cis(grid, dim, use_middle_indices_grid=True, num_attention_heads=heads)
    pos, freqs, axes = grid_rotary(grid, dim, use_middle_indices_grid=True, num_attention_heads=heads)
    a = torch.gather(pos, 1, axes.reshape(1, -1, 1).expand(2, -1, pos.shape[2]).long())  # (B, dim/2, T)
    a = (a * freqs.reshape(1, -1, 1)).view(2, heads, -1, pos.shape[2]).transpose(2, 3)
    tol = THETA * math.pi / 2 * 5 * 2.0 ** -24 + 2.0 ** -23
    assert (torch.cos(a) - cos.double()).abs().max() <= tol
    assert (torch.sin(a) - sin.double()).abs().max() <= tol
