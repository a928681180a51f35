"""pico_amd.kernels with a torch that lacks the private names it takes for their speed
(host logic, no GPU)."""
import importlib.util

import torch

from pico_amd import kernels


def test_without_torchs_private_names(monkeypatch):
    names = ("_cuda_getDevice", "_cuda_getCurrentRawStream")
    for name in names:
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("pico_amd.kernels_elsewhere", kernels.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device: type("Stream", (), {"cuda_stream": 100 + device}))
    assert module._raw_stream(3) == 103
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    assert module._stream() == 105


def test_with_them():
    if hasattr(torch._C, "_cuda_getDevice"):
        assert kernels._device is torch._C._cuda_getDevice
    if hasattr(torch._C, "_cuda_getCurrentRawStream"):
        assert kernels._raw_stream is torch._C._cuda_getCurrentRawStream
