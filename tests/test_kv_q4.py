"""4-bit KV cache and windowed attention without a GPU: the oracle's own properties, and the
refusals of the C entry points and of their Python wrappers."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from test_stateful_b200 import _lib, ops
from test_stateful_b200.config import tiny_engine_config
from test_stateful_b200.runtime.model import PagedPoolTensors

I3 = (C.c_int64 * 3)(0, 0, 0)
ALIGNED = 1 << 20  # stands for a device address; every call below is refused before it is used


@pytest.mark.parametrize("D", [64, 128])
def test_oracle_pack_roundtrip_and_error_bound(D):
    rng = np.random.default_rng(D)
    x = rng.standard_normal((3, 16, D)).astype(np.float32) * 4
    code, scale, zero = O.quantise(x)
    assert code.min() == 0 and code.max() == 15
    raw = O.pack(code, scale, zero)
    assert raw.shape == (3, 9 * D)
    back = O.unpack(raw)
    np.testing.assert_array_equal(back, O.values(code, scale, zero))
    # half a step, plus what rounding moved the zero (2^-11 of it) and 15 steps (2^-11 each)
    step = np.repeat(scale.astype(np.float64), 64, -1)
    base = np.repeat(np.abs(zero.astype(np.float64)), 64, -1)
    assert (np.abs(back - x) <= 0.5 * step + 2.0 ** -11 * (base + 15 * step) + 1e-7).all()


def test_oracle_special_groups():
    x = np.zeros((5, 64), np.float32)
    x[0] = 3.0                                  # constant: scale 0
    x[1, 5] = np.nan                            # NaN: the group reads back as NaN
    x[2, :2] = np.inf, -np.inf                  # saturates
    x[3] = np.arange(64) % 16                   # exact integers
    x[4] = np.where(np.arange(64) % 2, 1e30, -1e30)
    code, scale, zero = O.quantise(x)
    v = O.values(code, scale, zero)
    np.testing.assert_array_equal(v[0], 3.0)
    assert np.isnan(v[1]).all() and scale[1] == 0
    assert code[2, 0, 0] == 15 and code[2, 0, 1] == 0 and zero[2] == np.float16(-65504)
    np.testing.assert_array_equal(v[3], x[3])
    assert set(code[4].ravel()) == {0, 15}


def _write(**kw):
    a = dict(cache=ALIGNED, nb=4, L=2, H=2, D=128, k=ALIGNED, v=ALIGNED, dt=_lib.DT_F16, ks=I3, vs=I3, first=0, nl=1,
             m=ALIGNED, n=3)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("bad", [dict(D=32), dict(D=96), dict(nb=0), dict(L=0), dict(H=0), dict(dt=3), dict(dt=-1),
                                 dict(first=2), dict(first=-1), dict(nl=0), dict(nl=3), dict(first=1, nl=2),
                                 dict(n=-1), dict(cache=None), dict(k=None), dict(v=None), dict(m=None),
                                 dict(ks=None), dict(cache=ALIGNED + 8), dict(k=ALIGNED + 1), dict(m=ALIGNED + 2),
                                 dict(dt=_lib.DT_F32, v=ALIGNED + 2)])
def test_cache_entries_refuse(bad):
    lib = _lib.load()
    for fn in (lib.qtts_kv_write_q4, lib.qtts_kv_read_q4):
        assert fn(*_write(**bad), None) == _lib.ERR_INVALID
        assert "q4" in _lib.last_error()
    assert lib.qtts_kv_write_q4(*_write(n=0, k=None), None) == _lib.OK


def test_gather_entry_refuses():
    lib = _lib.load()
    good = [ALIGNED, 4, 2, 2, 128, ALIGNED, 5, ALIGNED]
    for i, v in [(0, None), (0, ALIGNED + 4), (1, 0), (2, 0), (3, -1), (4, 256), (5, None), (5, ALIGNED + 1), (6, -1),
                 (7, None), (7, ALIGNED + 1)]:
        a = list(good)
        a[i] = v
        assert lib.qtts_kv_gather_q4(*a, None) == _lib.ERR_INVALID, (i, v)
    good[6] = 0
    assert lib.qtts_kv_gather_q4(*good, None) == _lib.OK


def _attn(**kw):
    a = dict(q=ALIGNED, R=4, S=1, Hq=16, Hkv=8, D=128, kv=ALIGNED, layer=0, L=2, bs=16, nb=9, table=ALIGNED, slots=4,
             mbps=8, row_slot=ALIGNED, row_ctx=ALIGNED, max_ctx=128, window=16, sinks=4, out=ALIGNED, out_lo=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("bad", [dict(R=-1), dict(S=0), dict(S=3), dict(Hq=15), dict(Hq=0), dict(Hkv=0), dict(D=32),
                                 dict(D=256), dict(layer=2), dict(layer=-1), dict(L=0), dict(bs=32), dict(nb=0),
                                 dict(slots=0), dict(mbps=0), dict(max_ctx=0), dict(max_ctx=129), dict(window=-1),
                                 dict(sinks=-1), dict(q=None), dict(kv=None), dict(table=None), dict(row_slot=None),
                                 dict(row_ctx=None), dict(out=None), dict(q=ALIGNED + 4), dict(kv=ALIGNED + 8)])
def test_attention_entries_refuse(bad):
    lib = _lib.load()
    for fn in (lib.qtts_paged_attention_window, lib.qtts_paged_attention_q4):
        assert fn(*_attn(**bad), None) == _lib.ERR_INVALID
        assert fn(*_attn(R=0, q=None), None) == _lib.OK


def test_wrappers_take_cuda_tensors_only():
    cache = torch.zeros(2, 1, 2, 2, 9 * 64, dtype=torch.uint8)
    rows = torch.zeros(3, 2, 64)
    m = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(1, 4, 64)
    t = torch.zeros(1, 2, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(2, 1, 2, 2, 16, 64, dtype=torch.float16)
    for call in (lambda: ops.kv_write_q4(cache, rows, rows, m), lambda: ops.kv_read_q4(cache, m),
                 lambda: ops.kv_gather_q4(cache, m, 3),
                 lambda: ops.paged_attention_q4(q, cache, 0, t, one, one, 32),
                 lambda: ops.paged_attention_window(q, pool, 0, t, one, one, 32, 8)):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


def test_pool_formats():
    cfg = tiny_engine_config()
    with pytest.raises(ValueError, match="kv_format"):
        PagedPoolTensors(cfg, "cpu", kv_format="int4")
    fp16, q4 = PagedPoolTensors(cfg, "cpu"), PagedPoolTensors(cfg, "cpu", kv_format="q4")
    t = cfg.talker
    assert q4.kv.shape == (cfg.pool.num_blocks, t.num_layers, 2, t.kv_heads, 9 * t.head_dim)
    assert fp16.block_elems == t.num_layers * 2 * t.kv_heads * 16 * t.head_dim
    assert q4.block_elems * 2 == q4.kv[0].numel() and q4.block_elems % 8 == 0
    cfg.talker.head_dim = 32
    with pytest.raises(ValueError, match="head_dim"):
        PagedPoolTensors(cfg, "cpu", kv_format="q4")
