"""CPU oracle of the 4-bit KV cache and of paged attention with a window and sinks (numpy float64,
except the fp32 / fp16 steps that the cache's definition names)."""

from __future__ import annotations

import numpy as np

GROUP = 64
BLOCK = 16


def quantise(x: np.ndarray):
    """fp32 rows ``[..., D]`` -> codes ``[..., G, 64]`` (int), scale and zero fp16 ``[..., G]``."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    nan = np.isnan(g).any(-1)
    c = np.clip(np.where(np.isnan(g), np.float32(0), g), np.float32(-65504), np.float32(65504))
    lo, hi = c.min(-1) + np.float32(0), c.max(-1)  # a zero is +0 whatever the signs of the group's zeros
    zero = lo.astype(np.float16)
    scale = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
    d = (c - zero.astype(np.float32)[..., None]).astype(np.float64)
    s = scale.astype(np.float64)[..., None]
    code = np.where(s == 0, 0, np.clip(np.rint(d / np.where(s == 0, 1, s)), 0, 15)).astype(np.int64)
    code[nan] = 0
    return code, np.where(nan, np.float16(0), scale), np.where(nan, np.float16(np.nan), zero)


def values(code, scale, zero) -> np.ndarray:
    v = code.astype(np.float64) * scale.astype(np.float64)[..., None] + zero.astype(np.float64)[..., None]
    return v.reshape(*v.shape[:-2], -1)


def pack(code, scale, zero) -> np.ndarray:
    """Codes ``[..., 16, G, 64]`` and parameters ``[..., 16, G]`` of whole chunks -> bytes ``[..., 9 D]``."""
    G = code.shape[-2]
    lead = code.shape[:-3]
    out = np.zeros((*lead, 9 * G * GROUP), np.uint8)
    for g in range(G):
        for i in range(8):
            word = sum(code[..., g, 8 * i + n].astype(np.uint64) << np.uint64(4 * n) for n in range(8))
            for b in range(4):
                at = (G * i + g) * 4 + b
                out[..., np.arange(BLOCK) * (G * 32) + at] = (word >> np.uint64(8 * b)) & np.uint64(255)
        for j, prm in enumerate((scale, zero)):
            raw = np.ascontiguousarray(prm[..., g]).view(np.uint16)
            at = BLOCK * G * 32 + g * 64 + np.arange(BLOCK) * 4 + 2 * j
            out[..., at], out[..., at + 1] = raw & 255, raw >> 8
    return out


def unpack(raw: np.ndarray) -> np.ndarray:
    """Bytes ``[..., 9 D]`` -> values ``[..., 16, D]`` (float64)."""
    D = raw.shape[-1] // 9
    G = D // GROUP
    out = np.empty((*raw.shape[:-1], BLOCK, D))
    tok = np.arange(BLOCK)
    for g in range(G):
        at = BLOCK * G * 32 + g * 64 + tok * 4
        scale = (raw[..., at].astype(np.uint16) | raw[..., at + 1].astype(np.uint16) << 8).view(np.float16)
        zero = (raw[..., at + 2].astype(np.uint16) | raw[..., at + 3].astype(np.uint16) << 8).view(np.float16)
        for c in range(GROUP):
            byte = raw[..., tok * (G * 32) + (G * (c // 8) + g) * 4 + (c % 8) // 2]
            out[..., 64 * g + c] = ((byte >> (4 * (c % 2))) & 15) * scale.astype(np.float64) + zero.astype(np.float64)
    return out


def visible(ctx: int, n_keys: int, window: int, sinks: int) -> np.ndarray:
    j = np.arange(n_keys)
    return (j < ctx) & ((j >= ctx - window) | (j < sinks) | (window == 0))


def attention(q, keys, vals, ctx: int, window: int = 0, sinks: int = 0) -> np.ndarray:
    """One row: ``q [Hq, D]`` over ``keys``, ``vals [Hkv, n, D]`` -> float64 ``[Hq * D]``; keys that the
    row does not see are left out before any arithmetic."""
    Hq, D = q.shape
    Hkv = keys.shape[0]
    see = visible(ctx, keys.shape[1], window, sinks)
    out = np.zeros((Hq, D))
    if see.any():
        for h in range(Hq):
            k, v = keys[h // (Hq // Hkv)][see], vals[h // (Hq // Hkv)][see]
            s = k.astype(np.float64) @ q[h].astype(np.float64) / np.sqrt(D)
            p = np.exp(s - s.max())
            out[h] = (p @ v.astype(np.float64)) / p.sum()
    return out.reshape(-1)
