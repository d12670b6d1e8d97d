"""4-bit KV cache and windowed attention without a GPU: what their launch path and their formats promise."""

import types

import numpy as np
import torch

from oracle import kv_q4 as O
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


def test_what_four_bits_keep_of_a_normal_key():
    """Groups of 64 normal values read back with about 21 dB, some 2 dB above 4-bit floats (0, .5, 1, 1.5, 2, 3, 4, 6 with
    a sign) of the same 4.25 to 4.5 bits, a power-of-two scale for each 32 that keeps the largest within 6."""
    x = np.random.default_rng(3).standard_normal((4000, 64)).astype(np.float32)
    snr = lambda y: 10 * np.log10((x.astype(np.float64) ** 2).sum() / ((x - y) ** 2).sum())  # noqa: E731
    ours = snr(O.values(*O.quantise(x)))
    g = x.reshape(-1, 32).astype(np.float64)
    scale = 2.0 ** np.ceil(np.log2(np.abs(g).max(-1, keepdims=True) / 6))
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    near = grid[np.abs(np.abs(g / scale)[..., None] - grid).argmin(-1)]
    floats = snr((np.sign(g) * near * scale).reshape(x.shape))
    assert 20.5 < ours < 21.5 and 1.5 < ours - floats < 3.5, (ours, floats)


def test_pairs_of_a_four_bit_value():
    """The chunk tiles' operands, step for step: high parts exact in fp16 for every code, and high + low within 2^-18 of
    the group's largest value (2^-23 where that is below 2^-5).  Groups from 1e-9 to all of fp16, with offsets."""
    rng = np.random.default_rng(0)
    f32, f16 = np.float32, np.float16
    n = 40000
    size, off = 10.0 ** rng.uniform(-9, 5, (n, 1)), 10.0 ** rng.uniform(-9, 4.8, (n, 1)) * rng.choice([-1, 0, 1], (n, 1))
    x = np.clip(rng.standard_normal((n, 64)) * size + off, -65504, 65504).astype(f32)
    x[0], x[1] = 0, 0
    x[1, :2] = 65504, -65504
    _, s, z = O.quantise(x)
    s, z = s[:, 0].astype(f32), z[:, 0].astype(f32)
    top = np.maximum(np.abs(z), np.abs(f32(15) * s + z)).astype(f32)
    e = np.maximum((top.view(np.uint32) >> 23).astype(np.int64), 113)
    magic = (((e + 14) << 23) | 0x400000).astype(np.uint32).view(f32)
    s0, z0 = (s + magic) - magic, (z + magic) - magic
    sh, sl, zh, zl = (a.astype(f16).astype(np.float64)[:, None] for a in (s0, s - s0, f32(0.5) * z0, f32(0.5) * (z - z0)))
    c = np.arange(16) / 2
    high, low = c * sh + zh, (c * sl + zl).astype(f16).astype(np.float64)
    np.testing.assert_array_equal(high.astype(f16), high)
    value = 2 * c * s.astype(np.float64)[:, None] + z.astype(np.float64)[:, None]
    err = np.abs(2 * (high + low) - value).max(1)
    # (2^-18 is half a step of the low part; its operands' own rounding is far below)
    assert (err <= np.maximum(1.001 * 2.0 ** -18 * top.astype(np.float64), 2.0 ** -23)).all()
