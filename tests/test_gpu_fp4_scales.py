"""Scales of an fp4 weight that change between calls: the product always uses
the ones the weight has, whoever packed them last.  Every comparison is of bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(seed=21, n=128, k=256):
    """A weight whose compute is "fp4", and one of twice its values: the same codes, other scales."""
    from ltxq.quantized_linear import QuantizedLinear

    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(n, k, generator=gen, device="cuda").bfloat16()
    one, two = (QuantizedLinear.from_linear(v, mode="nvfp4").set_compute("fp4") for v in (w, w * 2))
    assert torch.equal(one.weight, two.weight)
    return one, two, gen


@pytest.mark.parametrize("m", [3, 40, 700])
def test_scales_swapped_back_after_another_reader_packed(cuda, m):
    import ltxq

    lin, twice, gen = _weights()
    x = torch.randn(m, 256, generator=gen, device="cuda").bfloat16()
    want, other = lin(x), twice(x)
    ff = ltxq.FeedForward(lin, ltxq.QuantizedLinear.from_linear(torch.randn(64, 128, device="cuda").bfloat16(), mode="nvfp4"))
    a, b = lin.scales, twice.scales.clone()
    for reader in (lin.dequantize, lin.qweight, lin.mx_scales, lambda: ff(x), lambda: lin(x)):
        lin.scales = b
        reader()
        lin.scales = a
        assert torch.equal(lin(x), want)
        lin.scales = b
        assert torch.equal(lin(x), other)
        lin.scales = a
        assert torch.equal(lin(x), want)


@pytest.mark.parametrize("change", ["in place", "replaced", "never packed"])
def test_capture_before_any_call_sees_a_change(cuda, change):
    """The packing goes into the graph; calls outside do not count on it, before the first replay or after."""
    lin, twice, gen = _weights()
    x = torch.randn(40, 256, generator=gen, device="cuda").bfloat16()
    old, want = lin(x), twice(x)
    if change == "in place":
        lin.scales.copy_(twice.scales)
    elif change == "replaced":
        lin.scales = twice.scales.clone()
    else:
        lin, want = type(lin)(lin.weight, lin.scales, group_size=16, bits=4, mode="nvfp4"), old
        lin.compute = "fp4"
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = lin(x)
        second = lin(x)
    assert torch.equal(lin(x), want)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(second, want) and torch.equal(lin(x), want)
    if change == "in place":
        lin.scales.fill_(0)
        assert not lin(x).any()
        graph.replay()
        torch.cuda.synchronize()
        assert not out.any()


def test_compute_set_inside_a_capture(cuda):
    lin, twice, gen = _weights()
    x = torch.randn(40, 256, generator=gen, device="cuda").bfloat16()
    want = twice(x)
    lin.scales.copy_(twice.scales)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = lin.set_compute("fp4")(x)
    assert torch.equal(lin(x), want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_changed_scales_on_two_streams(cuda):
    """Both streams wait for the change; the first call packs, behind a delay
    of its stream, and the second finds the scales packed.  Then the other way
    round: a delayed product still reads what the next change packs over."""
    lin, twice, gen = _weights()
    x = torch.randn(40, 256, generator=gen, device="cuda").bfloat16()
    one, two = lin(x), twice(x)
    sets = [lin.scales.clone(), twice.scales.clone()]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(6):
        want, scales = ((two, one)[i % 2], sets[1 - i % 2])
        lin.scales.copy_(scales)
        for s in (a, b):
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(a):
            torch.cuda._sleep(20_000_000)  # about 10 ms
            first = lin(x)
        with torch.cuda.stream(b):
            second = lin(x)
            torch.cuda._sleep(20_000_000)
            third = lin(x)
        torch.cuda.current_stream().wait_stream(a)  # the next change waits for a alone
        lin.scales.copy_(sets[i % 2])
        fourth = lin(x)
        torch.cuda.synchronize()
        for got in (first, second, third):
            assert torch.equal(got, want)
        assert torch.equal(fourth, (one, two)[i % 2])


@pytest.mark.parametrize("m", [40, 300])
def test_feed_forward_captured_before_any_call_sees_a_change(cuda, m):
    """Its descriptors keep the graph's own packed scales until the launch, beside a workspace of the same pool."""
    import ltxq

    def pair():
        one, two, gen = _weights(n=512)
        out1, out2, _ = _weights(seed=22, n=256, k=512)
        return ltxq.FeedForward(one, out1), ltxq.FeedForward(two, out2), gen

    ff, want_ff, gen = pair()
    x = torch.randn(m, 256, generator=gen, device="cuda").bfloat16()
    want, old = want_ff(x), ff(x)
    ff.project_in.scales.copy_(want_ff.project_in.scales)
    ff.project_out.scales = want_ff.project_out.scales.clone()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = ff(x)
    assert torch.equal(ff(x), want) and not torch.equal(old, want)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_copies_keep_their_scales_apart(cuda):
    import copy

    lin, twice, gen = _weights()
    x = torch.randn(40, 256, generator=gen, device="cuda").bfloat16()
    one, two = lin(x), twice(x)
    for other in (copy.copy(lin), copy.deepcopy(lin)):
        assert torch.equal(other(x), one)
        other.scales = twice.scales.clone()
        assert torch.equal(other(x), two) and torch.equal(lin(x), one)
