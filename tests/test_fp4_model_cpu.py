"""CPU checks of 4-bit floating point weights in blocks and caches: what is refused."""

from types import SimpleNamespace

import pytest
import torch


def test_cache_builder_refuses_unknown_or_mixed_formats(tmp_path):
    from ltxq import cache_build as CB

    for kw in (dict(mode="off", fp4="fp4"), dict(mode="off", fp4="mxfp4", affine=(8, 64)), dict(fp4="nvfp4")):
        with pytest.raises(ValueError, match="fp4"):
            CB.build_transformer_cache(tmp_path / "none.safetensors", tmp_path / "c" / "t.safetensors", **kw)


def test_cache_reader_refuses_scales_of_no_format():
    from ltxq import cache as C

    arrs = {"weight": torch.zeros(8, 16, dtype=torch.uint32), "scales": torch.zeros(8, 3, dtype=torch.uint8)}
    with pytest.raises(ValueError, match="3 scales for 128 values"):
        C.quantized_linears_from_state({"quant": {"a": arrs}, "bias": {}}, {"a": 128})


def test_fused_projections_need_one_tensor_scale():
    from ltxq.block import _cat_linears

    with pytest.raises(ValueError, match="global_scale"):
        _cat_linears([SimpleNamespace(global_scale=1.0), SimpleNamespace(global_scale=0.5)])


def test_microbench_knows_the_formats():
    from ltxq import microbench as mb
    from ltxq.quantized_linear import COMPUTE, quant_defaults

    for name in ("mxfp4", "nvfp4", "mxfp4_fp4", "nvfp4_fp4"):
        mode, bits, compute = mb.MODES[name]
        assert quant_defaults(mode, None, None)[1] == bits and compute in COMPUTE


def _layer(weight, scales, bias=None, mode="nvfp4", n=16, k=96, bits=4, group=16):
    from ltxq.quantized_linear import QuantizedLinear

    lin = object.__new__(QuantizedLinear)  # the constructor wants a GPU's tensors
    lin.weight, lin.scales, lin.bias, lin.mode, lin.pretransposed = weight, scales, bias, mode, False
    lin.out_features, lin.in_features, lin.bits, lin.group_size = n, k, bits, group
    return lin


def test_arrays_must_fit_the_layer():
    w, s = torch.zeros(16, 12, dtype=torch.uint32), torch.zeros(16, 6, dtype=torch.uint8)
    b = torch.zeros(16, dtype=torch.bfloat16)
    _layer(w, s)._check_fp4()
    _layer(w, s, b)._check_fp4()
    _layer(w, s[:, :3].contiguous(), mode="mxfp4", group=32)._check_fp4()
    for bad in (_layer(w, s[:, :5]), _layer(w, s[:, :5].contiguous()), _layer(w, s[:15]), _layer(w[:15], s),
                _layer(w, s.short()), _layer(w.view(torch.uint8).view(16, 48), s), _layer(w, s, b[:8]),
                _layer(w, s, b.float()), _layer(w, s, k=128), _layer(w, s, n=17), _layer(w, s, group=32),
                _layer(w, s, bits=8), _layer(w, s, mode="mxfp4")):
        with pytest.raises(ValueError):
            bad._check_fp4()


def _descriptors(mode, gw, gx, n=16, k=64):
    from ltxq import _lib

    group = 16 if mode == _lib.NVFP4 else 32
    w = _lib.QWeight(0x1000, 0x2000, None, None, n, k, mode, 4, group, _lib.LAYOUT_STD, global_scale=gw)
    return w, _lib.Fp4Act(0x3000, 0x4000, mode, gx)


@pytest.mark.parametrize("gw,gx", [(2.0 ** 60, 2.0 ** 60), (2.0 ** -50, 2.0 ** -50)])
def test_product_of_tensor_scales_is_bounded(gw, gx):
    import ctypes

    from ltxq import _lib

    w, x = _descriptors(_lib.NVFP4, gw, gx)
    lib = _lib.load()
    assert lib.ltxq_qlinear_fp4(ctypes.byref(x), 1, ctypes.byref(w), None, 0x5000, None) == _lib.ERR_UNSUPPORTED
    assert b"global scales" in lib.ltxq_last_error()


def test_dequantize_wants_an_aligned_output():
    import ctypes

    from ltxq import _lib

    w, _ = _descriptors(_lib.MXFP4, 1.0, 1.0)
    lib = _lib.load()
    assert lib.ltxq_dequantize(ctypes.byref(w), 0x5008, None) == _lib.ERR_UNSUPPORTED
    assert b"aligned" in lib.ltxq_last_error()


def test_unsplit_workspace():
    """The part of the workspace that a product needs to run the same kernels unsplit."""
    import ctypes

    from ltxq import _lib

    lib = _lib.load()
    for mode in (_lib.MXFP4, _lib.NVFP4):
        w, _ = _descriptors(mode, 1.0, 1.0, n=5120, k=544)
        q = ctypes.byref(w)
        both = lambda m: (lib.ltxq_qlinear_unsplit_workspace_size(m, q), lib.ltxq_qlinear_workspace_size(m, q))  # noqa: E731
        assert both(0) == (0, 0) and both(16) == (0, 0)
        assert both(200)[0] == 0  # the fused kernels
        assert both(767)[0] == 0
        assert both(768)[0] == 5120 * 544 * 2 <= both(768)[1]
        w.compute, w.mx_scales = _lib.COMPUTE_FP4, 0x6000
        assert both(200)[0] == both(200)[1] > 0 and both(2000)[0] == both(2000)[1] > both(200)[0]
        assert both(16) == (0, 0)
    assert lib.ltxq_qlinear_unsplit_workspace_size(4, None) == 0


def test_quantized_tensor_describes_what_it_holds():
    import copy

    import ltxq

    t = ltxq.FP4Tensor((3, 5), 288, "nvfp4", "cpu", 0.5)
    st = t.struct()
    codes, scales = t.tensors()
    assert (st.codes, st.scales, st.global_scale) == (codes.data_ptr(), scales.data_ptr(), 0.5)
    t.buffer = t.buffer.clone()
    codes, scales = t.tensors()
    st = t.struct()
    assert (st.codes, st.scales) == (codes.data_ptr(), scales.data_ptr())
    t.global_scale = 0.25
    assert t.struct().global_scale == 0.25
    other = copy.deepcopy(t)
    st = other.struct()
    assert st.codes == other.buffer.data_ptr() != t.buffer.data_ptr()
    for bad in (t.buffer[:-1], t.buffer[1:], t.buffer[::2], t.buffer.view(torch.int16)):
        other.buffer = bad
        with pytest.raises(ValueError, match="buffer"):
            other.struct()


def test_operands_on_another_device_are_refused(monkeypatch):
    """A product's residual, gate and prologue vectors lie on its own device (stand-ins for tensors of two GPUs)."""
    from ltxq import quantized_linear as Q

    class On(SimpleNamespace):
        def get_device(self):
            return self.device.index

        def new_empty(self, *a, **k):
            return self

    def on(i, *shape):
        return On(device=torch.device("cuda", i), shape=shape, dtype=torch.bfloat16, numel=lambda: 4 * 96, is_cuda=True)

    monkeypatch.setattr(Q, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(Q, "_device", lambda: 0)
    lin = _layer(on(0, 16, 12), None)
    lin.compute = "dequant"
    for kw in (dict(residual=on(1, 4, 16), gate=on(0, 16)), dict(residual=on(0, 4, 16), gate=on(1, 16)),
               dict(adaln=(on(1, 96), on(0, 96), 1e-6)), dict(adaln=(on(0, 96), on(1, 96), 1e-6))):
        with pytest.raises(ValueError, match="cuda:1"):
            lin(on(0, 4, 96), **kw)


def test_arrays_of_another_type_of_the_same_size_are_refused():
    w, s = torch.zeros(16, 12, dtype=torch.uint32), torch.zeros(16, 6, dtype=torch.uint8)
    b = torch.zeros(16, dtype=torch.bfloat16)
    s32 = s[:, :3].contiguous()
    for ok in (_layer(w.view(torch.int32), s, b), _layer(w, s.view(torch.float8_e4m3fn)), _layer(w, s.view(torch.int8)),
               _layer(w, s32.view(torch.float8_e8m0fnu), mode="mxfp4", group=32)):
        ok._check_fp4()
    for bad in (_layer(w, s, b.half()), _layer(w, s, b.view(torch.int16)), _layer(w.view(torch.float32), s),
                _layer(w, s.view(torch.float8_e5m2)), _layer(w, s.view(torch.float8_e8m0fnu)), _layer(w, s.bool()),
                _layer(w, s32.view(torch.float8_e4m3fn), mode="mxfp4", group=32)):
        with pytest.raises(ValueError, match="must be"):
            bad._check_fp4()
