"""The binding's stream handle where torch does not offer the direct way to it (CPU)."""
import torch

import dramamoe as D


def test_without_the_direct_call(monkeypatch):
    class Stream:
        cuda_stream = 0x1234

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(D, "_raw_stream", None, raising=False)
    assert D.stream_ptr() == 0x1234


def test_direct_call(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x1000 + device, raising=False)
    monkeypatch.setattr(D, "_raw_stream", None, raising=False)
    assert D.stream_ptr() == 0x1003
