"""4-bit floating point weights where the model has them: caches, fused
projections, blocks; and weights that change after their scales were packed.
Every comparison is of bits: the same weights through the same kernels."""

import pytest
import torch

pytestmark = pytest.mark.gpu

MODES = ["mxfp4", "nvfp4"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).bfloat16()


def _checkpoint_name(base):
    for ours, theirs in (("audio_ff.project_in.proj", "audio_ff.net.0.proj"), ("audio_ff.project_out", "audio_ff.net.2"),
                         ("ff.project_in.proj", "ff.net.0.proj"), ("ff.project_out", "ff.net.2")):
        if base == ours:
            return theirs
    return base.replace(".to_out", ".to_out.0")


@pytest.mark.parametrize("mode", MODES)
def test_cache_round_trip_and_block(cuda, tmp_path, mode):
    """A block built into a cache and read back gives the bits of the block
    quantized directly, in both computes, eager and from a graph."""
    from ltxq import cache as C
    from ltxq import cache_build as CB
    from ltxq.block import BasicAVTransformerBlock, StreamConfig, TransformerArgs, linear_specs, table_specs
    from ltxq.quantized_linear import QuantizedLinear

    video, audio = StreamConfig(1024, 8, 128, 1024), StreamConfig(512, 8, 64, 512)
    gen = _gen(3)
    ckpt, lin, tabs = {}, {}, {}
    for base, (n, k) in linear_specs(video, audio).items():
        w, b = _randn(gen, n, k, std=0.02), _randn(gen, n, std=0.01)
        key = f"model.diffusion_model.transformer_blocks.0.{_checkpoint_name(base)}"
        ckpt[f"{key}.weight"], ckpt[f"{key}.bias"] = w, b
        lin[base] = QuantizedLinear.from_linear(w, b, mode=mode)
    for name, shape in table_specs(video, audio).items():
        t = torch.randn(*shape, generator=gen, device="cuda") * 0.1
        tabs[name] = 1.0 + t if name.endswith("norm.weight") else t
        ckpt[f"model.diffusion_model.transformer_blocks.0.{name}"] = tabs[name]
    direct = BasicAVTransformerBlock(lin, tabs, video, audio)
    C.save_safetensors(tmp_path / "ckpt.safetensors", ckpt)
    cache_file = tmp_path / "cache" / "transformer.safetensors"
    payload = CB.build_transformer_cache(tmp_path / "ckpt.safetensors", cache_file, mode="off", fp4=mode)
    assert payload["block_linear_quantize"] == mode
    loaded = C.blocks_from_cache(cache_file, "cuda", video, audio)[0]
    assert all(q.mode == mode for q in loaded.quantized_modules())

    def rope(heads, t, d):
        ang = torch.rand(1, heads, t, d // 2, generator=gen, device="cuda") * 6.28
        return torch.cos(ang), torch.sin(ang)

    def args(cfg, t):
        f32 = lambda n, std: torch.randn(1, 1, n, cfg.dim, generator=gen, device="cuda") * std
        return TransformerArgs(x=_randn(gen, 1, t, cfg.dim), context=_randn(gen, 1, 24, cfg.context_dim),
                               timesteps=f32(9, 0.1), positional_embeddings=rope(cfg.heads, t, cfg.d_head),
                               cross_positional_embeddings=rope(audio.heads, t, audio.d_head),
                               cross_scale_shift_timestep=f32(4, 0.1), cross_gate_timestep=f32(1, 0.1),
                               prompt_timestep=f32(2, 0.1))

    v, a = args(video, 64), args(audio, 9)
    outs = {}
    for compute in ("dequant", "fp4"):
        outs[compute] = [blk.set_compute(compute)(v, a)[0].x.clone() for blk in (direct, loaded)]
        assert torch.isfinite(outs[compute][0]).all()
        assert torch.equal(*outs[compute])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = loaded(v, a)[0].x
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, outs[compute][0])
    assert not torch.equal(outs["dequant"][0], outs["fp4"][0])  # the activations are quantized in one of them


@pytest.mark.parametrize("mode,gs", [("mxfp4", 1.0), ("nvfp4", 1.0), ("nvfp4", 0.25)])
def test_fused_projections_keep_their_rows(cuda, mode, gs):
    from ltxq.block import _cat_linears
    from ltxq.quantized_linear import QuantizedLinear

    gen = _gen(5)
    parts = [QuantizedLinear.from_linear(_randn(gen, n, 96, std=0.1), None, mode=mode, global_scale=gs)
             for n in (64, 8, 136)]
    cat = _cat_linears(parts)
    assert cat.global_scale == gs
    assert torch.equal(cat.dequantize(), torch.cat([p.dequantize() for p in parts]))


@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
@pytest.mark.parametrize("change", ["in place", "replaced", "inference"])
def test_changed_scales_are_used(cuda, m, compute, change):
    from ltxq.quantized_linear import QuantizedLinear

    gen = _gen(7)
    with torch.inference_mode(change == "inference"):
        w, x = _randn(gen, 128, 256), _randn(gen, m, 256)
        lin = QuantizedLinear.from_linear(w, mode="nvfp4").set_compute(compute)
        twice = QuantizedLinear.from_linear(w * 2, mode="nvfp4").set_compute(compute)
        before = lin(x)
        if change == "replaced":
            lin.scales = twice.scales.clone()
        else:
            lin.scales.copy_(twice.scales)
        if change == "inference":
            lin.set_compute(compute)
        got, want = lin(x), twice(x)
        assert torch.equal(lin.weight, twice.weight)  # a power of two moves into the scales alone
        assert torch.equal(got, want) and not torch.equal(got, before)


def test_captured_product_follows_scales_that_are_packed_again(cuda):
    from ltxq.quantized_linear import QuantizedLinear

    gen = _gen(8)
    w, x = _randn(gen, 128, 256), _randn(gen, 40, 256)
    lin = QuantizedLinear.from_linear(w, mode="nvfp4").set_compute("fp4")
    twice = QuantizedLinear.from_linear(w * 2, mode="nvfp4").set_compute("fp4")
    lin(x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = lin(x)
    lin.set_compute("dequant")  # what the graph reads stays
    spoil = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (512, 2048, 4096, 8192)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, lin.set_compute("fp4")(x))
    lin.scales.copy_(twice.scales)
    lin.set_compute("fp4")
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, twice(x))
    del spoil


def test_microbench_modes(cuda, capsys):
    import json

    from ltxq import microbench

    microbench.main(["--shapes", "64x256x256", "--modes", "mxfp4,nvfp4,mxfp4_fp4,nvfp4_fp4", "--iters", "2", "--warmup",
                     "1", "--graph"])
    row = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert all(row[m]["ms"] > 0 for m in ("mxfp4", "nvfp4", "mxfp4_fp4", "nvfp4_fp4"))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("compute", ["dequant", "fp4"])
def test_long_feed_forward_runs_its_parts(cuda, mode, compute):
    """Enough rows that the weight is dequantized once: the prologue's and the
    feed-forward's workspaces hold that too."""
    import ltxq

    gen = _gen(9)
    ff = ltxq.FeedForward.from_linear(_randn(gen, 2048, 256, std=0.05), None, _randn(gen, 2048, 2048, std=0.02), None,
                                      mode=mode)
    ff.project_in.set_compute(compute)
    ff.project_out.set_compute(compute)
    x = _randn(gen, 1, 1550, 256)
    scale, shift = (torch.randn(1, 1, 256, generator=gen, device="cuda") * 0.1 for _ in range(2))
    h = ltxq.adaln_modulate(x, scale, shift, 1e-6)
    want = ff.project_in(h, gelu=True)
    assert torch.equal(ff.project_in(x, adaln=(scale, shift, 1e-6), gelu=True), want)
    assert torch.equal(ff(h), ff.project_out(want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_head", [False, True])
def test_rotary_positions_past_fp32(cuda, dtype, per_head):
    """Frequency 0 turns by nothing, wherever the token is."""
    import ltxq

    x = torch.randn(1, 3, 2, 64, device="cuda").to(dtype)
    pos = torch.tensor([1e300, -1e39, 5.0], dtype=torch.float64, device="cuda")
    freqs = torch.zeros(2, 32, dtype=torch.float64, device="cuda")
    assert torch.equal(ltxq.rotary(x, pos, freqs if per_head else freqs[0], 2), x)


def test_rotary_output_refusals(cuda):
    import ltxq

    x = torch.randn(2, 3, 64, device="cuda")
    pos, freqs = torch.arange(3, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError, match="memory of its own"):
        ltxq.rotary(x, pos, freqs, 1, out=x[:1].expand(2, 3, 64))
    for scale in (float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="finite"):
            ltxq.rotary(x, pos, freqs, 1, scale=scale)


@pytest.mark.parametrize("compute,m", [("fp4", 40), ("fp4", 700), ("dequant", 1600)])
def test_calls_in_a_row_share_the_workspace(cuda, compute, m):
    """Two launches per call, the second set up while the first still runs,
    and the next call writes the same workspace: eager and as one graph, the
    results are those of calls that were waited for."""
    import ltxq

    gen = _gen(11)
    lins = [ltxq.QuantizedLinear.from_linear(_randn(gen, 2048, 512, std=0.05), mode="mxfp4").set_compute(compute)
            for _ in range(2)]
    xs = [_randn(gen, m, 512) for _ in range(6)]
    want = []
    for i, x in enumerate(xs):
        want.append(lins[i % 2](x))
        torch.cuda.synchronize()

    def run():
        return [lins[i % 2](x) for i, x in enumerate(xs)]

    for _ in range(5):
        for got, w in zip(run(), want):
            assert torch.equal(got, w)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = run()
    for _ in range(5):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
