"""The packed scales of an fp4 weight and the descriptor that points at them,
on the CPU: a fake library that copies scale bytes stands for the packing
kernel, and the pointers of the descriptor are read as host memory."""

import contextlib
import ctypes

import pytest
import torch

from ltxq import quantized_linear as Q


class FakeLibrary:
    """Packing is a copy, now or, where it is only recorded (``recording``), later."""

    def __init__(self):
        self.log, self.recording, self.recorded = [], False, []

    def ltxq_fp4_weight_scales_size(self, q):
        return self._q(q).n_out * self._q(q).k_in // 16

    def ltxq_fp4_pack_weight_scales(self, q, out, stream):
        self.log.append("pack")
        job = (out, self._q(q).scales, self.ltxq_fp4_weight_scales_size(q))
        if self.recording:
            self.recorded.append(job)
        else:
            ctypes.memmove(*job)
        return 0

    def ltxq_dequantize(self, q, out, stream):
        return 0

    @staticmethod
    def _q(q):
        return getattr(q, "_obj", q)


@pytest.fixture
def lib(monkeypatch):
    fake = FakeLibrary()
    monkeypatch.setattr(Q._lib, "load", lambda: fake)
    monkeypatch.setattr(Q, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(Q, "_stream", lambda: 0)
    monkeypatch.setattr(Q, "_capturing", lambda: fake.recording, raising=False)
    monkeypatch.setattr(Q, "_wait_device", lambda dev: fake.log.append("device"), raising=False)
    monkeypatch.setattr(Q, "_wait_stream", lambda: fake.log.append("stream"), raising=False)
    return fake


def _scales(fill, n=16, k=96):
    return torch.full((n, k // 16), fill, dtype=torch.uint8)


def _linear(n=16, k=96):
    lin = object.__new__(Q.QuantizedLinear)  # the constructor wants a GPU's tensors
    lin.weight, lin.scales = torch.zeros(n, k // 8, dtype=torch.uint32), _scales(1, n, k)
    lin.biases = lin.bias = None
    lin.mode, lin.pretransposed, lin.bits, lin.group_size = "nvfp4", False, 4, 16
    lin.out_features, lin.in_features, lin.global_scale = n, k, 1.0
    return lin.set_compute("fp4")


def _read(q, n=16, k=96):
    """The packed bytes a product with this descriptor reads: one value in these tests."""
    got = set(ctypes.string_at(q.mx_scales, n * k // 16))
    assert len(got) == 1
    return got.pop()


def test_descriptor_follows_what_other_readers_pack(lib):
    """Scales swapped, packed by another reader, and swapped back."""
    lin = _linear()
    a, b = lin.scales, _scales(2)
    for other in (lin.mx_scales, lin.qweight, lin.dequantize, lambda: lin.set_compute("fp4")):
        assert _read(lin._qweight4()) == 1
        lin.scales = b
        other()
        lin.scales = a
        assert _read(lin._qweight4()) == 1
        assert _read(lin.qweight()) == 1


def test_reading_a_weight_back_packs_nothing(lib):
    lin = _linear()
    lin.scales = _scales(2)
    del lib.log[:]
    lin.dequantize()
    assert "pack" not in lib.log


def test_packing_that_is_only_recorded_counts_for_nothing_else(lib):
    """In a capture the packing is part of the graph: a call outside before its
    first replay packs for itself, and the graph leaves that memory alone."""
    lin = _linear()
    for change in ("in place", "replaced"):
        before = lin.mx_scales()
        if change == "in place":
            lin.scales.fill_(5)
        else:
            lin.scales = _scales(6)
        want = 5 if change == "in place" else 6
        lib.recording = True
        q = lin._qweight4()
        assert lib.recorded and all(job[0] != before.data_ptr() for job in lib.recorded)
        lib.recording = False
        assert _read(lin._qweight4()) == want
        assert lin.mx_scales() is before
        for job in lib.recorded:  # the replay
            ctypes.memmove(*job)
        assert _read(q) == want and _read(lin._qweight4()) == want
        del lib.recorded[:]


def test_packed_before_a_capture_nothing_is_recorded(lib):
    lin = _linear()
    lin.mx_scales()
    lib.recording = True
    q = lin._qweight4()
    assert not lib.recorded and _read(q) == 1


def test_recorded_packing_keeps_its_memory_while_the_descriptor_lives(lib):
    lin = _linear()
    lin.scales = _scales(3)
    del lin._fp4_packed  # never packed before
    lib.recording = True
    assert lin._qweight4().mx_scales
    first, second = lin.qweight(), lin.qweight()
    assert first.mx_scales != second.mx_scales
    lin.set_compute("fp4")
    lib.recording = False
    assert _read(lin._qweight4()) == 3


def test_packing_is_ordered_against_every_stream(lib):
    """Memory that other streams may still read is waited for before it is
    packed again, and every packing is finished before a call on another
    stream can find it; neither inside a capture."""
    lin = _linear()
    assert lib.log == ["pack", "stream"]  # memory of its own: nothing reads it yet
    lin._qweight4(), lin.mx_scales()
    assert lib.log == ["pack", "stream"]
    del lib.log[:]
    lin.scales.fill_(4)
    lin._qweight4()
    assert lib.log == ["device", "pack", "stream"]
    del lib.log[:]
    lin.set_compute("fp4")
    assert lib.log == ["device", "pack", "stream"]
    del lib.log[:]
    lin.scales.fill_(5)
    lib.recording = True
    lin._qweight4()
    assert lib.log == ["pack"]


def _same_place(t, *shape, stride=None):
    """Another array at t's address."""
    return t.as_strided(shape, stride or torch.empty(shape, dtype=torch.uint8).stride())


@pytest.mark.parametrize("name,other", [
    ("weight", lambda lin: _same_place(lin.weight, 8, 12)), ("weight", lambda lin: _same_place(lin.weight, 16, 6)),
    ("weight", lambda lin: _same_place(lin.weight, 16, 12, stride=(6, 1))),
    ("weight", lambda lin: lin.weight.view(torch.uint8)), ("scales", lambda lin: _same_place(lin.scales, 8, 6)),
    ("scales", lambda lin: _same_place(lin.scales, 16, 6, stride=(1, 1))),
    ("bias", lambda lin: _same_place(lin.bias, 8)), ("bias", lambda lin: _same_place(lin.bias, 16, stride=(0,))),
    ("bias", lambda lin: lin.bias.float()),
])
def test_array_at_the_same_address_is_checked(lib, name, other):
    """A descriptor is kept for arrays, not for addresses: another array there is looked at anew."""
    lin = _linear()
    lin.set_compute("dequant")
    lin.bias = torch.zeros(16, dtype=torch.bfloat16)
    lin._qweight4()
    setattr(lin, name, other(lin))
    with pytest.raises(ValueError, match=name):
        lin._qweight4()


def test_layer_of_other_sizes_is_checked(lib):
    for name, value in (("in_features", 192), ("out_features", 32), ("group_size", 32), ("bits", 8), ("mode", "mxfp4")):
        lin = _linear()
        lin.set_compute("dequant")
        lin._qweight4()
        setattr(lin, name, value)
        with pytest.raises(ValueError):
            lin._qweight4()


def test_array_changed_under_its_object_is_checked(lib):
    lin = _linear()
    lin.set_compute("dequant")
    lin._qweight4()
    lin.weight.data = lin.weight[:8]
    with pytest.raises(ValueError, match="weight"):
        lin._qweight4()


def test_scales_are_checked_before_they_are_packed(lib):
    lin = _linear()
    del lib.log[:]
    for reader in (lin.mx_scales, lin.qweight, lin._qweight4, lambda: lin.set_compute("fp4")):
        lin.scales = torch.zeros(16, 3, dtype=torch.uint8)
        with pytest.raises(ValueError, match="scales"):
            reader()
    assert lib.log == []


def test_copies_have_descriptors_and_packed_scales_of_their_own(lib):
    import copy

    lin = _linear()
    lin._qweight4()
    for other in (copy.deepcopy(lin), copy.copy(lin)):
        assert _read(other._qweight4()) == 1
        other.scales = _scales(9)
        assert _read(other._qweight4()) == 9 and _read(lin._qweight4()) == 1
        assert other._qweight4().weight == other.weight.data_ptr()


def test_arrays_are_checked_before_they_are_read_back(lib):
    lin = _linear()
    lin.scales = torch.zeros(16, 3, dtype=torch.uint8)
    with pytest.raises(ValueError, match="scales"):
        lin.dequantize()
