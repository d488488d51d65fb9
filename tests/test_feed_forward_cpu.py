"""Where a feed-forward runs: on its input's device, which is its weights' (stand-ins for tensors of two GPUs)."""

import contextlib
from types import SimpleNamespace

import pytest
import torch


class On(SimpleNamespace):
    def get_device(self):
        return self.device.index


def _on(i):
    return On(device=torch.device("cuda", i), dtype=torch.bfloat16, shape=(4, 64), is_cuda=True)


def _layer(i):
    return SimpleNamespace(in_features=64, out_features=64, weight=_on(i))


def test_runs_on_the_input_s_device(monkeypatch):
    from ltxq import feed_forward as F

    entered = []

    @contextlib.contextmanager
    def device(dev):
        entered.append(dev)
        monkeypatch.setattr(F, "_device", lambda: dev)
        yield

    class Reached(Exception):
        pass

    def contiguous():
        raise Reached

    monkeypatch.setattr(F, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(F, "_device", lambda: 0, raising=False)
    monkeypatch.setattr(F.torch.cuda, "device", device)
    x = _on(1)
    x.contiguous = contiguous
    with pytest.raises(Reached):
        F.FeedForward(_layer(1), _layer(1))(x)
    assert entered == [1]
    for layers in ((_layer(0), _layer(1)), (_layer(1), _layer(0))):
        with pytest.raises(ValueError, match="cuda:1"):
            F.FeedForward(*layers)(x)
