"""What rotary takes and refuses at its two interfaces, on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _args(x, out, heads, rotary_dim, **kw):
    from ltxq import _lib

    b, t = x.shape[0], x.shape[1]
    d = x.shape[2] // heads
    st = _lib.RotaryArgs(x=x.data_ptr(), out=out.data_ptr(), dtype=_lib.F32 if x.dtype == torch.float32 else _lib.BF16,
                         batch=b, tokens=t, heads=heads, head_dim=d, rotary_dim=rotary_dim, pos_dtype=_lib.POS_I64,
                         n_axes=1, scale=1.0)
    st.x_stride[:] = (x.stride(0), x.stride(1), d)
    st.out_stride[:] = (out.stride(0), out.stride(1), d)
    st.pos_stride[:] = (0, 0, 1)
    for k, v in kw.items():
        setattr(st, k, v)
    return st


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_head", [0, 1])
@pytest.mark.parametrize("positions", [True, False])
def test_nothing_rotated_is_a_copy(cuda, dtype, per_head, positions):
    import ctypes

    from ltxq import _lib

    x = torch.randn(2, 37, 3 * 40, device="cuda").to(dtype)
    out = torch.zeros_like(x)
    p = torch.arange(37, device="cuda")
    st = _args(x, out, 3, 0, freqs_per_head=per_head, positions=p.data_ptr() if positions else None)
    torch.cuda.synchronize()
    assert _lib.load().ltxq_rotary(ctypes.byref(st), None) == _lib.OK
    torch.cuda.synchronize()
    assert torch.equal(out, x)


@pytest.mark.parametrize("n_axes", [1, 3])
def test_no_frequencies_for_each_head(cuda, n_axes):
    import ltxq

    x = torch.randn(2, 37, 3 * 40, device="cuda").bfloat16()
    f = torch.zeros(3, 0, dtype=torch.float64, device="cuda")
    p = torch.zeros(2, n_axes, 37, device="cuda")
    axes = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    got = ltxq.rotary(x, p, f, 3, axes=axes) if n_axes > 1 else ltxq.rotary(x, p[:, 0], f, 3)
    assert torch.equal(got, x)


@pytest.mark.parametrize("per_head", [False, True])
def test_quadrants_of_far_positions(cuda, per_head):
    """The fp64 value of pi / 2 times the kernel's 1 / (2 pi) is exactly a quarter turn, and a quarter times an integer
    below 2^53 is exact: position n is turned by n quarters, whatever its size.  2^-21: an fp32 rotation."""
    import math

    import numpy as np

    import ltxq

    n = np.array([2 ** 51 + 1, 2 ** 51 - 1, 2400000000000001, 2400000000000003, -2400000000000001, -2400000000000002,
                  -2 ** 51 - 3, 4000000000000001, -4000000000000001, 2 ** 53 - 1, 1 - 2 ** 53, 4 * 262144 + 3], np.int64)
    assert (math.pi / 2) * 0.15915494309189535 == 0.25
    x = torch.zeros(1, len(n), 8, device="cuda")
    x[..., :4] = 1
    f = torch.full((1, 4) if per_head else (4,), math.pi / 2, dtype=torch.float64, device="cuda")
    for inverse in (False, True):
        y = ltxq.rotary(x, torch.from_numpy(n).cuda(), f, 1, inverse=inverse).double().cpu().numpy()[0]
        q = (-n if inverse else n) % 4
        assert np.abs(y[:, 0] - np.array([1, 0, -1, 0])[q]).max() <= 2.0 ** -21
        assert np.abs(y[:, 4] - np.array([0, 1, 0, -1])[q]).max() <= 2.0 ** -21


def _freqs(n):
    return 10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n)


def test_outputs_beside_the_input(cuda):
    """Everything that shares no element with x is written, whatever memory lies between."""
    import ltxq

    p, f = torch.arange(21, device="cuda"), _freqs(32)
    buf = torch.randn(2, 21, 3, 4, 64, device="cuda").bfloat16()
    rows = buf.view(2, 21, 768)
    want = ltxq.rotary(rows[..., :256].clone(), p, f, 4)
    for out in (rows[..., 256:512], rows[..., 512:]):  # columns of the same rows
        before = rows.clone()
        assert ltxq.rotary(rows[..., :256], p, f, 4, out=out) is out and torch.equal(out, want)
        out.copy_(before[..., out.storage_offset() % 768:][..., :256])
        assert torch.equal(rows, before)
    flat = torch.zeros(4 * 2 * 21 * 256, device="cuda").bfloat16()
    x = flat[:2 * 21 * 256].view(2, 21, 256)
    x.copy_(rows[..., :256])
    for i in (1, 3):  # behind one another
        out = flat[i * 2 * 21 * 256:][:2 * 21 * 256].view(2, 21, 256)
        assert torch.equal(ltxq.rotary(x, p, f, 4, out=out), want)
    both = torch.zeros(2, 21, 8, 64, device="cuda").bfloat16()  # alternate heads
    both[:, :, ::2] = rows[..., :256].view(2, 21, 4, 64)
    ltxq.rotary(both[:, :, ::2], p, f, 4, out=both[:, :, 1::2])
    assert torch.equal(both[:, :, 1::2].reshape(2, 21, 256), want)
    turned = torch.zeros(2, 4, 21, 64, device="cuda").bfloat16().transpose(1, 2)
    assert torch.equal(ltxq.rotary(rows[..., :256].view(2, 21, 4, 64), p, f, 4, out=turned).reshape(2, 21, 256), want)
    view = x.view(2, 21, 256)  # another tensor object over x itself
    assert torch.equal(ltxq.rotary(x, p, f, 4, out=view), want) and torch.equal(x, want)
    one = torch.randn(1, 1, 256, device="cuda").bfloat16()
    assert torch.equal(ltxq.rotary(one, p[:1], f, 4, out=one.expand(1, 1, 256)), one)


def test_outputs_that_share_elements_are_refused(cuda):
    import ltxq

    p, f = torch.arange(3, device="cuda"), _freqs(32)
    flat = torch.zeros(2000, device="cuda").bfloat16()
    x = flat[:2 * 3 * 64].view(2, 3, 64)
    for out in (flat[8:][:384].view(2, 3, 64), flat[64:][:384].view(2, 3, 64), flat[1:][:384].view(2, 3, 64),
                flat.as_strided((2, 3, 64), (64, 128, 1))):
        with pytest.raises(ValueError, match="x itself"):
            ltxq.rotary(x, p, f, 1, out=out)
    for rows in (flat[:64].expand(2, 3, 64), flat[:192].view(1, 3, 64).expand(2, 3, 64), flat.as_strided((2, 3, 64), (192, 32, 1))):
        with pytest.raises(ValueError, match="memory of its own"):
            ltxq.rotary(rows, p, f, 1, out=rows)
        with pytest.raises(ValueError, match="memory of its own"):
            ltxq.rotary(x.clone(), p, f, 1, out=rows)
        assert torch.equal(ltxq.rotary(rows, p, f, 1), ltxq.rotary(rows.clone(), p, f, 1))  # read only: fine
    assert not flat.any()
