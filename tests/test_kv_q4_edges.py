"""4-bit KV cache and windowed attention without a GPU: what their launch path and their formats promise."""

import types

import torch

from test_stateful_b200 import _lib


def test_raw_stream_without_torchs_private_call(monkeypatch):
    """A torch that lacks the call still gives the current stream's handle."""
    seen = []
    monkeypatch.setattr(_lib, "_current_raw_stream", None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: seen.append(d) or types.SimpleNamespace(cuda_stream=77))
    assert _lib.raw_stream(2) == 77 and _lib.stream_ptr() == 77 and seen == [2, 3]
    monkeypatch.setattr(_lib, "_current_raw_stream", lambda d: 100 + d)
    assert _lib.raw_stream(2) == 102 and _lib.stream_ptr() == 103
    assert _lib.stream_ptr(types.SimpleNamespace(cuda_stream=5)) == 5
