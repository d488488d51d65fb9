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
