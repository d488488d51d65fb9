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
