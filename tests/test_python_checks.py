"""Checks of the Python layer that need no GPU: tensors of another device than the
current one, whose stream would run the kernels."""
import pytest
import torch

from molot_amd import attn


def on(device):
    """A tensor that says it lies on this device."""
    class Placed(torch.Tensor):
        device = property(lambda self: torch.device(device))
        get_device = lambda self: -1 if self.device.type == "cpu" else self.device.index  # noqa: E731

    return torch.zeros(8).as_subclass(Placed)


def test_tensors_of_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(attn, "_device", lambda: 1)
    attn._need(on("cuda:1"), "q", torch.float32, 8)
    with pytest.raises(ValueError, match="q.*cuda:0.*cuda:1"):
        attn._need(on("cuda:0"), "q", torch.float32, 8)
    with pytest.raises(ValueError, match="device tensor"):
        attn._need(on("cpu"), "q", torch.float32, 8)
