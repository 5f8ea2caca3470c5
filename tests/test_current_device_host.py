"""Tensors of another device than the current one, without a GPU: a launch for them is refused before a
stream handle is taken, and the 8-bit checkpoints' Linears enter the tensor's device."""
from types import SimpleNamespace

import pytest
import torch

from visionseg import _lib as L, linear


class _Device:
    current = 0

    def __init__(self, d):
        self.index = torch.device(d).index

    def __enter__(self):
        self.before, _Device.current = _Device.current, self.index

    def __exit__(self, *exc):
        _Device.current = self.before


@pytest.fixture
def two_devices(monkeypatch):
    """torch.cuda's idea of the current device; every default stream has the handle 0."""
    _Device.current = 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: _Device.current)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=0))
    monkeypatch.setattr(torch.cuda, "device", _Device)


def _on(index, **kw):
    return SimpleNamespace(device=torch.device("cuda", index), is_cuda=True, **kw)


def test_stream_of_another_device_is_refused(two_devices):
    assert not L.stream(_on(0)).value and not L.stream().value
    with pytest.raises(RuntimeError, match="cuda:1 while the current device is cuda:0"):
        L.stream(_on(1))
    with L.on_device_of(_on(1)):
        assert not L.stream(_on(1)).value
        with pytest.raises(RuntimeError, match="cuda:0 while"):
            L.stream(_on(0))
    assert _Device.current == 0


def test_act8_linears_enter_the_device(two_devices, monkeypatch):
    seen = []
    monkeypatch.setattr(linear._LinearAct8Fn, "apply", lambda *a: seen.append(_Device.current))
    monkeypatch.setattr(linear._MlpAct8Fn, "apply", lambda *a: seen.append(_Device.current))
    t = _on(1, dtype=torch.float32, numel=lambda: 4, requires_grad=True)
    linear.linear_act8(t, t, None)
    linear.mlp_act8(t, t, None, t, None)
    assert seen == [1, 1] and _Device.current == 0
