"""Operators of 4-bit weights on tensors of a device that is not the current one (which device is, and the kernels, are stand-ins)."""
import contextlib

import torch

from gcore_b200.ops import _lib, quant


def test_weights_are_quantised_on_their_own_device(monkeypatch):
    state = {"inside": 0, "calls": 0}

    @contextlib.contextmanager
    def device(d):
        assert d == torch.device("cpu")
        state["inside"] += 1
        yield
        state["inside"] -= 1

    quantise = quant.quant_fp4_1x32

    def on_its_device(w):
        assert state["inside"] == 1, "launched on another device's stream"
        state["calls"] += 1
        with monkeypatch.context() as m:
            m.setattr(_lib, "use_native", lambda t: False)
            return quantise(w)

    monkeypatch.setattr(_lib, "use_native", lambda t: True)
    monkeypatch.setattr(_lib, "is_current", lambda t: state["inside"] > 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(quant, "quant_fp4_1x32", on_its_device)
    w = torch.randn(8, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    W = quant.Fp4Weight.of(w)
    assert state == {"inside": 0, "calls": 1} and W.shape == (8, 64)
