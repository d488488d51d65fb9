"""What rotary refuses before any CUDA call (made-up addresses: nothing is launched)."""

import ctypes

import pytest


def _status(**kw):
    from ltxq import _lib

    st = _lib.RotaryArgs(x=1 << 20, out=1 << 30, dtype=_lib.BF16, layout=_lib.ROTARY_HALF, batch=3, tokens=4, heads=2,
                         head_dim=64, rotary_dim=64, positions=16, pos_dtype=_lib.POS_I64, n_axes=1, freqs=16, scale=1.0)
    st.x_stride[:] = st.out_stride[:] = (512, 128, 64)
    st.pos_stride[:] = (4, 0, 1)
    for k, v in kw.items():
        if k.endswith("stride"):
            getattr(st, k)[:] = v
        else:
            setattr(st, k, v)
    lib = _lib.load()
    status = lib.ltxq_rotary(ctypes.byref(st), None)
    return {_lib.ERR_INVALID: "invalid", _lib.ERR_UNSUPPORTED: "unsupported"}.get(status), lib.ltxq_last_error().decode()


X = 1 << 20


@pytest.mark.parametrize("kw", [
    dict(out_stride=(0, 128, 64)), dict(out_stride=(512, 0, 64)), dict(out_stride=(512, 128, 0)),
    dict(out_stride=(512, 64, 64)), dict(out_stride=(512, 128, 32)), dict(out_stride=(510, 128, 64)),
    dict(out_stride=(512, -64, 64)), dict(out_stride=(1, 1, 1)),
    dict(x=X, out=X, x_stride=(0, 128, 64), out_stride=(0, 128, 64)),  # in place on rows that share memory
    dict(x=X, out=X, x_stride=(512, 64, 64), out_stride=(512, 64, 64)),
])
def test_out_with_shared_elements(kw):
    status, text = _status(**kw)
    assert status == "invalid" and "memory of its own" in text


@pytest.mark.parametrize("kw", [
    dict(x=X, out=X + 2), dict(x=X, out=X - 2), dict(x=X, out=X + 1, dtype=0), dict(x=X + 64, out=X),
    dict(x=X, out=X + 128), dict(x=X, out=X + 256), dict(x=X, out=X + 256 * 3), dict(x=X, out=X + 1024 * 2 + 256),
    dict(x=X, out=X - 1024 + 128),
    dict(x=X, out=X, out_stride=(512, 64, 256)),  # the same memory in another order
    dict(x=X, out=X + 4, x_stride=(0, 128, 64)),
    dict(x=X, out=X + 127 * 2, batch=1, tokens=1, x_stride=(0, 0, 64), out_stride=(0, 0, 64)),
    dict(x=X, out=X + 2, batch=1, tokens=2, heads=1, x_stride=(9, 64, 9), out_stride=(7, 64, 7)),
])
def test_out_that_overlaps_x(kw):
    status, text = _status(**kw)
    assert (status == "invalid" and "x itself" in text) or (kw["out"] % 2 and status == "unsupported")


def test_extents_past_64_bits():
    big = (1 << 62) - 8
    assert _status(batch=1 << 30, out_stride=(big, 128, 64), x_stride=(0, 128, 64))[0] in ("invalid", "unsupported")


@pytest.mark.parametrize("kw", [dict(positions=20), dict(positions=18, pos_dtype=0), dict(positions=17, pos_dtype=2),
                                dict(positions=20, pos_dtype=3), dict(freqs=20), dict(axis=18), dict(axis=17, n_axes=3),
                                dict(freqs=12, freqs_per_head=1)])
def test_unaligned_positions_and_frequencies(kw):
    status, text = _status(**kw)
    assert status == "unsupported" and "aligned to their elements" in text
