"""4-bit KV cache and windowed paged attention on the GPU against the float64 oracle.

Tolerances.  The cache: codes and parameters bit for bit; values read back are one rounding (half a
unit) of the stored value.  Attention, out + out_lo: fp32 score sums, ex2.approx (2^-22), probabilities
in two halves of 16 bits together (2^-16, the 4-bit pool) or 22 (fp16 pool), the output in two bf16
halves (2^-17): without q's own rounding a score is off by less than 2^-14 for the norms drawn here
(D <= 128 fp32 terms), so an output, a mean of values, by at most (2^-13 + 2^-15) max|v| < 2^-12 max|v|.
q is two fp16 halves (2^-22, covered by that) over the fp16 pool.  Over the 4-bit pool it is a 16-bit
fixed-point number, each channel off by at most max|q| / 65278 (half a unit): a score by at most
d = max|q| / 65278 sum|k| / sqrt(D), a probability by a factor within exp(+-2 d) (numerator and sum), an
output by (exp(2 d) - 1) max|v| more.
Chunks of rows go through fp16 tiles: q and P round to fp16 (2^-11), and so do 4-bit values: d = 2^-11
sum|q k| / sqrt(D) (twice that at 4 bits), and 2^-11 max|v| for P (once more at 4 bits).  Those bounds let all
roundings conspire; as they are independent, the root mean square over a row is held to twice its
expectation's bound as well: (d2 + 2^-11) rms(v) with d2 = 2^-11 |q| max|k| / D (times sqrt 2 at 4 bits)."""


import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import kv_q4 as O  # noqa: E402
from test_stateful_b200 import _lib, ops  # noqa: E402
from test_stateful_b200.config import EngineConfig, PagedPoolConfig, TalkerConfig  # noqa: E402

DEV = "cuda"
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _new_cache(nb, L, H, D):
    return torch.zeros(nb, L, 2, H, 9 * D, dtype=torch.uint8, device=DEV)


def _expect(cache_shape, k, v, mapping, layer):
    """Bytes of a zero-filled cache after the write, and the values of the written rows [n, nl, 2, H, D]."""
    nb, L, _, H, chunk = cache_shape
    D = chunk // 9
    kv = torch.stack([k, v], 2).float().cpu().numpy()
    code, scale, zero = O.quantise(kv)
    codes = np.zeros((nb, L, 2, H, 16, D // 64, 64), np.int64)
    sc, zr = np.zeros((2, nb, L, 2, H, 16, D // 64), np.float16)
    for i, m in enumerate(mapping):
        if 0 <= m < nb * 16:
            for arr, src in ((codes, code), (sc, scale), (zr, zero)):
                arr[m // 16, layer:layer + kv.shape[1], :, :, m % 16] = src[i]
    return O.pack(codes, sc, zr), O.values(code, scale, zero)


def _same_bytes(got, want, D):
    """Bit equality; NaN zeros compare as NaN (their payload is not defined)."""
    n = 8 * D
    np.testing.assert_array_equal(got[..., :n], want[..., :n])
    g, w = (np.ascontiguousarray(a[..., n:]).view(np.float16) for a in (got, want))
    np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
    np.testing.assert_array_equal(g[~np.isnan(g)].view(np.uint16), w[~np.isnan(w)].view(np.uint16))


def _close_values(got, want, dtype):
    got = got.double().cpu().numpy()
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    # one rounding of the exact value; bf16 and fp16 may round the fp32 value again (2^-24)
    assert (np.abs(got - want)[~nan] <= (EPS[dtype] + 2.0 ** -24) * np.abs(want)[~nan] + tiny).all()


# ------------------------------------------------------------------------------ the cache
@pytest.mark.parametrize("D,H,L,layer,nl", [(128, 8, 1, 0, 1), (64, 2, 3, 1, 2), (128, 1, 2, 1, 1), (64, 3, 2, 0, 2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 15, 16, 37])
def test_write_and_read(D, H, L, layer, nl, dtype, n):
    g = _gen(n)
    k, v = (torch.randn(n, nl, H, D, generator=g) * 3).to(dtype), (torch.randn(n, nl, H, D, generator=g)).to(dtype)
    cache = _new_cache(6, L, H, D)
    m = torch.randperm(96, generator=g)[:n].to(torch.int32)
    ops.kv_write_q4(cache, k.to(DEV), v.to(DEV), m.to(DEV), layer=layer)
    want, vals = _expect(cache.shape, k, v, m.tolist(), layer)
    _same_bytes(cache.cpu().numpy(), want, D)
    for out in (dtype, torch.float16):
        rk, rv = ops.kv_read_q4(cache, m.to(DEV), layer=layer, n_layers=nl, dtype=out)
        _close_values(rk, vals[:, :, 0], out)
        _close_values(rv, vals[:, :, 1], out)


def test_write_special_groups():
    """Constant, tied, saturating, subnormal, NaN and infinite groups, bit for bit."""
    x = torch.zeros(10, 1, 1, 64)
    x[0] = 7.25
    x[1] = torch.arange(64) % 16 + 0.5 * (torch.arange(64) % 2)       # ties between codes
    x[1, 0, 0, 0], x[1, 0, 0, 1] = 0, 15
    x[2, 0, 0, 3] = float("nan")
    x[3, 0, 0, :2] = torch.tensor([float("inf"), float("-inf")])
    x[4] = torch.where(torch.arange(64) % 2 == 0, 1e30, -1e30)
    x[5] = torch.randn(64, generator=_gen(1)) * 1e-8                  # scale underflows to 0
    x[6] = torch.randn(64, generator=_gen(2)) * 3e-7                  # subnormal scale
    x[7] = 1000.0 + torch.randn(64, generator=_gen(3)) * 0.01         # range far below the offset
    x[8] = -torch.rand(64, generator=_gen(4)) * 65504
    # borders: k + 1/2 steps of a scale of 1, one fp32 step to either side
    b = torch.arange(15) + 0.5
    x[9, 0, 0, :15], x[9, 0, 0, 15:30], x[9, 0, 0, 30:45] = b, torch.nextafter(b, b + 1), torch.nextafter(b, b - 1)
    x[9, 0, 0, 45:] = 15
    x[9, 0, 0, 63] = 0
    m = torch.arange(10, dtype=torch.int32)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        cache = _new_cache(1, 1, 1, 64)
        k = x.to(dtype)
        ops.kv_write_q4(cache, k.to(DEV), (-k).to(DEV), m.to(DEV))
        want, vals = _expect(cache.shape, k, -k, m.tolist(), 0)
        _same_bytes(cache.cpu().numpy(), want, 64)
        rk, rv = ops.kv_read_q4(cache, m.to(DEV), dtype=torch.float32)
        _close_values(rk, vals[:, :, 0], torch.float32)
        _close_values(rv, vals[:, :, 1], torch.float32)


@pytest.mark.parametrize("D", [64, 128])
def test_groups_across_all_of_fp16_stay_finite(D):
    """(65504 + 65504) / 15 rounds up to a scale of 8736, and 15 of it on -65504 is 65536: 65504 in fp16, read back,
    gathered, and in either form of attention (half a step of 2^-11, which chunk tolerances count for a 4-bit value)."""
    n = 80
    k = torch.randn(n, 1, 1, D, generator=_gen(31))
    k[:, :, :, 0], k[:, :, :, 1] = 65504, -65504
    k[3, 0, 0, 2] = float("inf")
    cache, m = _new_cache(5, 1, 1, D), torch.arange(n, dtype=torch.int32)
    ops.kv_write_q4(cache, k.to(DEV), k.to(DEV), m.to(DEV))
    want, vals = _expect(cache.shape, k, k, m.tolist(), 0)
    _same_bytes(cache.cpu().numpy(), want, D)
    assert vals.max() == 65536
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        rk, _ = ops.kv_read_q4(cache, m.to(DEV), dtype=dtype)
        _close_values(rk, np.minimum(vals[:, :, 0], 65504) if dtype == torch.float16 else vals[:, :, 0], dtype)
    flat = ops.kv_gather_q4(cache, torch.arange(5, dtype=torch.int32, device=DEV), n)
    assert torch.isfinite(flat).all()
    # queries small enough for scores of order one (0: every key counts the same)
    S, kv = 64, vals[:, 0].transpose(1, 2, 0, 3)
    table, ctx = torch.arange(5, dtype=torch.int32).view(1, 5), torch.arange(n - S, n, dtype=torch.int32) + 1
    for qscale in (0.0, 1e-6):
        q = torch.randn(S, 2, D, generator=_gen(32)) * qscale
        for s in (1, S):
            out = ops.paged_attention_q4(q.to(DEV), cache, 0, table.to(DEV), torch.zeros(S, dtype=torch.int32, device=DEV),
                                         ctx.to(DEV), n, rows_per_stream=s).double().cpu().numpy()
            for r in range(S):
                w = O.attention(q[r].numpy(), kv[0], kv[1], int(ctx[r]))
                tol = _tolerance("q4", q[r].numpy(), kv, s > 1)
                assert (np.abs(out[r] - w) <= 2.0 ** -8 * np.abs(w) + tol).all(), (qscale, s, r)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_queries_of_zero(fmt):
    """Every visible key counts the same, hidden ones nothing, in either form."""
    for S in (1, 90):
        _run_case(fmt, 4, 2, 128, [100, 95], S, 40, 3, qscale=0.0)


def test_write_many_random_borders():
    """Values drawn next to code borders, where a rounded quotient would decide wrongly."""
    g = _gen(9)
    n = 512
    scale = (torch.rand(n, 1, generator=g) + 0.5).half().float()
    x = (torch.randint(0, 15, (n, 128), generator=g) + 0.5) * scale
    x = torch.nextafter(x, torch.where(torch.rand(n, 128, generator=g) < 0.5, 1e9, -1e9))
    x[:, 0::64], x[:, 1::64] = 0, 15 * scale
    k = x.view(n, 1, 1, 128)
    cache = _new_cache(n // 16, 1, 1, 128)
    m = torch.arange(n, dtype=torch.int32)
    ops.kv_write_q4(cache, k.to(DEV), (k + scale.view(n, 1, 1, 1)).to(DEV), m.to(DEV))
    want, _ = _expect(cache.shape, k, k + scale.view(n, 1, 1, 1), m.tolist(), 0)
    _same_bytes(cache.cpu().numpy(), want, 128)


@pytest.mark.parametrize("offset", [0, 1])
def test_strided_and_unaligned_rows(offset):
    """K and V as views: of a QKV output, heads before tokens, broadcast over heads, off by one element."""
    g = _gen(3)
    n, H, D = 21, 4, 128
    buf = torch.randn(n * 16 * D + 8, generator=g).to(torch.bfloat16).to(DEV)
    qkv = buf[offset:offset + n * 16 * D].view(n, 16, D)
    hf = torch.randn(H, n, D, generator=g).to(torch.bfloat16).to(DEV).transpose(0, 1)
    one = torch.randn(n, 1, D, generator=g).to(torch.bfloat16).to(DEV).expand(n, H, D)
    m = torch.arange(n, dtype=torch.int32).flip(0).contiguous()
    for k, v in ((qkv[:, 8:12], qkv[:, 12:]), (hf, one), (qkv[:, 0:8:2], hf)):
        cache = _new_cache(2, 1, H, D)
        ops.kv_write_q4(cache, k, v, m.to(DEV))
        want, vals = _expect(cache.shape, k.unsqueeze(1), v.unsqueeze(1), m.tolist(), 0)
        _same_bytes(cache.cpu().numpy(), want, D)
        out = torch.full((n, 3 * H * D + 2), 5.0, device=DEV, dtype=torch.float32)
        ko = out[:, offset:offset + H * D].view(n, H, D)
        vo = out[:, 2 * H * D + offset:3 * H * D + offset].view(n, H, D)
        ops.kv_read_q4(cache, m.to(DEV), k=ko, v=vo)
        _close_values(ko, vals[:, 0, 0], torch.float32)
        _close_values(vo, vals[:, 0, 1], torch.float32)
        assert (out[:, H * D + offset:2 * H * D + offset] == 5).all()  # nothing past the rows


def test_positions_outside_the_pool():
    g = _gen(4)
    k = torch.randn(5, 2, 64, generator=g)
    cache = _new_cache(2, 1, 2, 64)
    m = torch.tensor([-1, 31, 32, -16, 7], dtype=torch.int32)
    ops.kv_write_q4(cache, k.to(DEV), k.to(DEV), m.to(DEV))
    want, vals = _expect(cache.shape, k.unsqueeze(1), k.unsqueeze(1), m.tolist(), 0)
    _same_bytes(cache.cpu().numpy(), want, 64)
    rk, _ = ops.kv_read_q4(cache, m.to(DEV), dtype=torch.float32)
    vals = vals[:, :, 0].copy()
    vals[[0, 2, 3]] = 0
    _close_values(rk, vals, torch.float32)
    # a position's neighbours keep what they hold
    ops.kv_write_q4(cache, k[:1].to(DEV), k[:1].to(DEV), m[3 + 1:].to(DEV))
    again, _ = ops.kv_read_q4(cache, torch.tensor([31], dtype=torch.int32, device=DEV), dtype=torch.float32)
    assert torch.equal(again[0], rk[1])


def test_empty_calls():
    cache = _new_cache(1, 1, 2, 64)
    e = torch.empty(0, 2, 64, device=DEV)
    m = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.kv_write_q4(cache, e, e, m)
    assert ops.kv_read_q4(cache, m)[0].shape == (0, 1, 2, 64)
    assert ops.kv_gather_q4(cache, m, 0).shape == (2, 2, 0, 64)
    q = torch.empty(0, 4, 64, device=DEV)
    t = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    assert ops.paged_attention_q4(q, cache, 0, t, m, m, 16).shape == (0, 256)
    assert int(cache.sum()) == 0


@pytest.mark.parametrize("D,n", [(128, 1), (128, 16), (128, 53), (64, 100)])
def test_gather(D, n):
    H, L, nb = 3, 2, 9
    raw = torch.from_numpy(np.random.default_rng(n).integers(0, 256, (nb, L, 2, H, 9 * D), dtype=np.uint8))
    prm = torch.randn(nb, L, 2, H, D // 2, generator=_gen(n)).half()   # finite scales and zeros
    raw[..., 8 * D:] = prm.view(torch.uint8)
    blocks = torch.randperm(nb, generator=_gen(n)).to(torch.int32)
    blocks[1] = -1
    blocks[2] = nb
    got = ops.kv_gather_q4(raw.to(DEV), blocks.to(DEV), n)
    vals = O.unpack(raw.numpy())
    want = np.zeros((L, 2, H, n, D))
    for t in range(n):
        b = int(blocks[t // 16])
        if 0 <= b < nb:
            want[:, :, :, t] = vals[b, :, :, :, t % 16]
    _close_values(got, want.reshape(2 * L, H, n, D), torch.float16)


def test_wrapper_refusals_on_device():
    cache = _new_cache(2, 2, 2, 64)
    rows = torch.zeros(3, 2, 64, device=DEV)
    m = torch.arange(3, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, device=DEV)
    t = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    bad = [lambda: ops.kv_write_q4(cache, rows, rows[:2], m), lambda: ops.kv_write_q4(cache, rows, rows.half(), m),
           lambda: ops.kv_write_q4(cache, rows.double(), rows.double(), m),
           lambda: ops.kv_write_q4(cache, rows, rows, m.long()), lambda: ops.kv_write_q4(cache, rows, rows, m, layer=2),
           lambda: ops.kv_write_q4(cache.float(), rows, rows, m),
           lambda: ops.kv_write_q4(cache, rows.transpose(1, 2), rows.transpose(1, 2), m),
           lambda: ops.kv_write_q4(cache[..., :500], rows, rows, m),
           lambda: ops.kv_read_q4(cache, m, n_layers=3), lambda: ops.kv_read_q4(cache, m, layer=-1),
           lambda: ops.kv_read_q4(cache, m, dtype=torch.int8), lambda: ops.kv_gather_q4(cache, two, 33),
           lambda: ops.kv_gather_q4(cache, two, -1),
           lambda: ops.paged_attention_q4(q.half(), cache, 0, t, two, two, 32),
           lambda: ops.paged_attention_q4(q, cache, 2, t, two, two, 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 33),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two[:1], two, 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t.long(), two, two, 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 32, window=-1),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 32, window=(1 << 32) + 5),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 32, window=8, sinks=1 << 31),
           lambda: ops.paged_attention_q4(q, cache, 1 << 32, t, two, two, 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, (1 << 32) + 16),
           lambda: ops.paged_attention_q4(torch.zeros(2 * 4 * 64 + 1, device=DEV)[1:].view(2, 4, 64), cache, 0, t, two,
                                          two, 32),
           lambda: ops.kv_read_q4(cache, m, k=torch.zeros(1, 2, 64, device=DEV).expand(3, 2, 64),
                                  v=torch.zeros(3, 2, 64, device=DEV)),
           lambda: ops.kv_write_q4(cache, rows, rows, m, layer=1 << 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 32, rows_per_stream=3),
           lambda: ops.paged_attention_q4(q[:, :3], cache, 0, t, two, two, 32),
           lambda: ops.paged_attention_q4(q, cache, 0, t, two, two, 32, out=torch.empty(2, 255, device=DEV)),
           lambda: ops.paged_attention_window(q, cache, 0, t, two, two, 32, 4)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------------------ attention
def _pool(fmt, nb, L, H, D, seed, scale=1.0):
    """A pool of ``fmt`` filled with random K/V, and its values [nb, L, 2, H, 16, D] (float64)."""
    x = torch.randn(nb, L, 2, H, 16, D, generator=_gen(seed)) * scale
    x[..., : D // 16] *= 3.0
    if fmt == "fp16":
        x = x.half()
        return x.to(DEV), x.double().numpy()
    raw = O.pack(*O.quantise(x.half().float().numpy()))
    return torch.from_numpy(raw).to(DEV), O.unpack(raw)


def _attend(fmt, *a, window=0, sinks=0, **kw):
    if fmt == "fp16":
        return ops.paged_attention_window(*a, window, sinks, **kw)
    return ops.paged_attention_q4(*a, window=window, sinks=sinks, **kw)


def _is_chunk(S, Hq, H):
    """Whether rows may go through fp16 tiles."""
    forced = os.environ.get("QTTS_WINDOW_TILES")
    return S > 1 and forced != "0" and (forced == "1" or S * Hq // H >= 64)


def _tolerance(fmt, q, kv, chunk=False):
    """Absolute tolerance of out + out_lo for one row (see the module's docstring)."""
    if not kv.size:
        return 0.0
    top = np.abs(kv[1]).max()
    group, D = len(q) // len(kv[0]), q.shape[-1]
    if chunk:
        q4 = fmt == "q4"
        d = 2.0 ** -11 * (1 + q4) * max((np.abs(kv[0][h // group]) @ np.abs(q[h])).max() for h in range(len(q))) / np.sqrt(D)
        return (2.0 ** -12 + np.expm1(2 * d) + 2.0 ** -11 * (1 + q4)) * top
    d = np.abs(q).max() / 65278 * np.abs(kv[0]).sum(-1).max() / np.sqrt(D) if fmt == "q4" else 0.0
    return (2.0 ** -12 + np.expm1(2 * d)) * top


def _rms_tolerance(fmt, q, kv):
    """Root mean square over a row of a chunk (see the module's docstring)."""
    if not kv.size:
        return 0.0
    d2 = 2.0 ** -11 * np.linalg.norm(q, axis=-1).max() * np.linalg.norm(kv[0], axis=-1).max() / q.shape[-1]
    return 2 * (d2 * (np.sqrt(2) if fmt == "q4" else 1) + 2.0 ** -11) * np.sqrt((kv[1] ** 2).mean())


def _run_case(fmt, Hq, H, D, ctxs, S, window, sinks, seed=0, max_ctx=None, poison=None, qscale=1.0):
    """``ctxs``: each stream's last row's context.  Returns nothing; asserts against the oracle."""
    n = len(ctxs)
    width = max(1, -(-max(max(ctxs), 1) // 16)) + 1
    nb, L, layer = n * width + 2, 2, 1
    pool, vals = _pool(fmt, nb, L, H, D, seed)
    perm = torch.randperm(nb, generator=_gen(seed + 1)).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32)
    for b, c in enumerate(ctxs):
        have = -(-max(c, 0) // 16)
        table[b, :have] = perm[b * width:b * width + have]
    if poison is not None:
        pool = poison(pool, table, perm)
    q = torch.randn(n * S, Hq, D, generator=_gen(seed + 2)) * qscale
    row_slot = torch.arange(n).repeat_interleave(S).to(torch.int32)
    row_ctx = torch.tensor([c - S + 1 + t for c in ctxs for t in range(S)], dtype=torch.int32)
    out_lo = torch.full((n * S, Hq * D), 9.0, device=DEV, dtype=torch.bfloat16)
    limit = max_ctx or width * 16
    out = _attend(fmt, q.to(DEV), pool, layer, table.to(DEV), row_slot.to(DEV), row_ctx.to(DEV), limit, window=window,
                  sinks=sinks, rows_per_stream=S, out_lo=out_lo)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    got = (out.double() + out_lo.double()).cpu().numpy()
    for b, c in enumerate(ctxs):
        blocks = table[b, :-(-max(c, 0) // 16)].long().numpy()
        kv = vals[blocks, layer].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
        for t in range(S):
            r = b * S + t
            want = O.attention(q[r].numpy(), kv[0], kv[1], min(int(row_ctx[r]), limit), window, sinks)
            tol = _tolerance(fmt, q[r].numpy(), kv, _is_chunk(S, Hq, H))
            assert np.abs(got[r] - want).max() <= tol, (r, np.abs(got[r] - want).max(), tol)
            if _is_chunk(S, Hq, H):
                assert np.sqrt(((got[r] - want) ** 2).mean()) <= _rms_tolerance(fmt, q[r].numpy(), kv), r
    return out


HEADS = [(16, 8, 128), (4, 2, 64), (8, 8, 64), (16, 4, 128), (16, 2, 128), (6, 2, 64), (12, 1, 128), (5, 1, 64)]


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("Hq,H,D", HEADS)
def test_decode_rows(fmt, Hq, H, D):
    _run_case(fmt, Hq, H, D, [1, 2, 15, 16, 17, 31, 33, 100, 255, 257, 700, 0, -3], 1, 0, 0)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (16, 16), (17, 4), (72, 4), (100, 33), (300, 5),
                                          (5, 1000), (100000, 3)])
def test_decode_window_and_sinks(fmt, window, sinks):
    for Hq, H, D in HEADS[:2]:
        _run_case(fmt, Hq, H, D, [1, 4, 16, 17, 40, 73, 77, 200, 411, 0], 1, window, sinks, seed=window)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("S,ctxs", [(2, [2, 40, 33]), (5, [5, 18, 100]), (21, [21, 58, 321, 26]), (70, [70, 150]),
                                    (7, [3, 0])])
@pytest.mark.parametrize("Hq,H,D", [HEADS[0], HEADS[1], HEADS[5], HEADS[6]])
def test_chunks(fmt, S, ctxs, Hq, H, D):
    """Streams of S rows; the last two begin before the first key (rows without keys, as a padded chunk has)."""
    for window, sinks in ((0, 0), (9, 2), (64, 20)):
        _run_case(fmt, Hq, H, D, ctxs, S, window, sinks, seed=S)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("ctx", [4096, 9001])
def test_long_rows_split_over_a_cluster(fmt, ctx):
    _run_case(fmt, 4, 2, 128, [ctx], 1, 0, 0)
    _run_case(fmt, 4, 2, 64, [ctx, 17], 1, 3000, 4)


def test_long_rows_are_unbiased():
    """Nearly uniform attention over zero-mean values: 4-bit values are code * scale + zero, two sums of some 7.5
    scales that cancel to a few hundredths, so a rounding of p * scale in one direction would show.  To
    nearest, a term is off by 2^-17 of at most 15 scale / n, 9001 of them at random 15 * 2^-17 / sqrt(3 n) =
    7e-7 scale; fp32 sums of some 10 blocks a warp, 10 * 2^-24 * 7.5 = 4.5e-6 scale at most; the output
    2^-17 of itself: together below 2^-16 scale in the root mean square (cutting p off: 6e-5)."""
    H, D, ctx = 2, 128, 9001
    nb = -(-ctx // 16)
    x = torch.randn(nb, 1, 2, H, 16, D, generator=_gen(3)).half().float().numpy()
    raw = O.pack(*O.quantise(x))
    scale = O.quantise(x[:, 0, 1])[1].astype(np.float64).max()
    vals = O.unpack(raw)[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
    q = torch.randn(1, 4, D, generator=_gen(4)) * 0.01
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    lo = torch.empty(1, 4 * D, device=DEV, dtype=torch.bfloat16)
    out = ops.paged_attention_q4(q.to(DEV), torch.from_numpy(raw).to(DEV), 0,
                                 torch.arange(nb, dtype=torch.int32, device=DEV).view(1, nb), zero, zero + ctx, nb * 16,
                                 out_lo=lo)
    err = (out.double() + lo.double()).cpu().numpy()[0] - O.attention(q[0].numpy(), vals[0], vals[1], ctx)
    assert np.sqrt((err ** 2).mean()) < 2.0 ** -16 * scale


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("S", [100, 300])
def test_long_chunks(fmt, S):
    _run_case(fmt, 4, 2, 128, [S + 37, S], S, 0, 0, seed=S)
    _run_case(fmt, 4, 2, 128, [S + 203], S, 65, 7, seed=S)
    _run_case(fmt, 8, 2, 64, [S + 9], S, 0, 0, seed=S)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_many_chunks(fmt):
    """Enough rows for the tile kernel by its own rule, several CTAs a tile and one."""
    _run_case(fmt, 16, 8, 128, [300, 150], 150, 0, 0)
    _run_case(fmt, 16, 8, 128, [1300], 100, 0, 0)
    _run_case(fmt, 16, 8, 128, [400, 210, 333, 205, 50], 200, 100, 20)


@pytest.mark.skipif(os.environ.get("QTTS_WINDOW_TILES") is not None, reason="already a forced run")
@pytest.mark.parametrize("form", ["0", "1"])
def test_both_chunk_forms(form):
    """Chunks go through 8-row or 128-row tiles by a rule on their sizes (QTTS_WINDOW_TILES forces one, read
    once per process): rerun every chunk case in a child process with each."""
    import subprocess
    import sys

    env = dict(os.environ, QTTS_WINDOW_TILES=form)
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-k",
                        "chunk or reach or finite or zero or garbage or bad or repeats", os.path.abspath(__file__)], env=env, capture_output=True, text=True,
                       timeout=900)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_row_ctx_is_capped_at_max_ctx(fmt):
    _run_case(fmt, 4, 2, 64, [90, 40], 1, 0, 0, max_ctx=50)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("qscale", [1e-6, 1e-3, 8.0])
def test_query_magnitudes(fmt, qscale):
    """Scores near 0 and up to some tens (fp32 sums of 8 times larger terms: below 2^-11 in the worst case of
    all roundings aligned, 2^-15 at their spread, which 2^-12 max|v| covers for a mean over few values)."""
    _run_case(fmt, 4, 2, 64, [50, 130], 1, 0, 0, qscale=qscale)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("S,ctx,window,sinks", [(1, 37, 0, 0), (1, 100, 20, 3), (9, 45, 12, 2), (70, 90, 0, 0),
                                                (130, 170, 33, 5)])
def test_what_a_row_does_not_see_does_not_reach_it(fmt, S, ctx, window, sinks):
    """Everything outside the stream's keys, and the keys between sinks and the first row's window, hold NaN
    or infinity."""
    def poison(pool, table, perm):
        used = set(int(b) for b in table.flatten() if b >= 0)
        for b in range(pool.shape[0]):
            if b not in used:
                pool[b] = 255 if fmt == "q4" else float("nan")
        hide = list(range(ctx, -(-ctx // 16) * 16))
        if window:
            hide += list(range(sinks, max(sinks, ctx - S + 1 - window)))
        for j in hide:
            b, o = int(table[0, j // 16]), j % 16
            if fmt == "fp16":
                pool[b, :, :, :, o] = float("nan") if j % 2 else float("inf")
            else:
                D = pool.shape[-1] // 9
                pool[b, :, :, :, o * D // 2:(o + 1) * D // 2] = 255
                for g in range(D // 64):
                    at = 8 * D + g * 64 + o * 4
                    pool[b, :, :, :, at:at + 4] = torch.tensor([0, 124, 0, 254] if j % 2 else [255, 255, 0, 124],
                                                               dtype=torch.uint8)
        return pool

    for Hq, H, D in (HEADS[0], HEADS[1]):
        _run_case(fmt, Hq, H, D, [ctx], S, window, sinks, poison=poison)


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("S", [20, 140])
def test_nan_key_inside_a_chunk_reaches_later_rows_only(fmt, S):
    H, D, ctx, bad = 2, 128, S + 10, S // 2
    nb = -(-ctx // 16)
    pool, vals = _pool(fmt, nb, 1, H, D, 5)
    table = torch.arange(nb, dtype=torch.int32).view(1, nb)
    if fmt == "fp16":
        pool[bad // 16, 0, 1, 0, bad % 16, 3] = float("nan")
    else:
        at = 8 * D + (bad % 16) * 4
        pool[bad // 16, 0, 1, 0, at + 3] = 0x7e   # the zero of V's first group
    q = torch.randn(S, 4, D, generator=_gen(6))
    ctxs = torch.arange(ctx - S + 1, ctx + 1, dtype=torch.int32)
    out = _attend(fmt, q.to(DEV), pool, 0, table.to(DEV), torch.zeros(S, dtype=torch.int32, device=DEV),
                  ctxs.to(DEV), ctx, rows_per_stream=S).float().cpu().view(S, 4, D)
    for r in range(S):
        sees = int(ctxs[r]) > bad
        assert bool(torch.isnan(out[r, :2, 3]).all()) == sees, r       # the two heads of the poisoned KV head
        assert torch.isfinite(out[r, 2:]).all()
        if not sees:
            kv = vals[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
            want = O.attention(q[r].numpy(), kv[0], kv[1], int(ctxs[r]))
            # bf16 output alone: half a unit (2^-8 of the value), then the tolerance of the pair
            err = np.abs(out[r].double().numpy().reshape(-1) - want)
            assert (err <= 2.0 ** -8 * np.abs(want) + _tolerance(fmt, q[r].numpy(), kv, _is_chunk(S, 4, H))).all()


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_bad_slots_and_blocks_are_reported(fmt):
    H, D, nb = 2, 64, 4
    pool, vals = _pool(fmt, nb, 1, H, D, 5)
    table = torch.tensor([[0, 1], [2, 99], [-1, 3]], dtype=torch.int32)
    q = torch.randn(5, 4, D, generator=_gen(6))
    slots = torch.tensor([0, -1, 3, 1, 2], dtype=torch.int32)
    ctx = torch.full((5,), 32, dtype=torch.int32)
    _lib.device_error()
    out = _attend(fmt, q.to(DEV), pool, 0, table.to(DEV), slots.to(DEV), ctx.to(DEV), 32).double().cpu().numpy()
    assert _lib.device_error() == 8   # an attention kernel met an index outside its buffers
    assert _lib.device_error() == 0
    assert not out[1].any() and not out[2].any()
    for r, blocks in ((0, [0, 1]), (3, [2]), (4, [3])):   # an id outside the pool hides its keys
        kv = vals[blocks, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
        want = O.attention(q[r].numpy(), kv[0], kv[1], kv.shape[2])
        assert (np.abs(out[r] - want) <= 2.0 ** -8 * np.abs(want) + _tolerance(fmt, q[r].numpy(), kv)).all()


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_graph_streams_and_repeats(fmt):
    """Captured, replayed on new data, on a side stream, twice at once: the same bits each time."""
    H, D, ctx = 8, 128, 2100
    nb = -(-ctx // 16)
    pool, _ = _pool(fmt, nb, 1, H, D, 7)
    table = torch.randperm(nb, generator=_gen(1)).to(torch.int32).view(1, nb).to(DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    qs = [torch.randn(1, 16, D, generator=_gen(i)).to(DEV) for i in range(3)]
    c = torch.full((1,), ctx, dtype=torch.int32, device=DEV)

    def call(q, out=None):
        return _attend(fmt, q, pool, 0, table, zero, c, ctx, window=2000, sinks=4, out=out)

    want = [call(q) for q in qs]
    for q, w in zip(qs, want):
        assert torch.equal(call(q), w)
    q_in, out = qs[0].clone(), torch.empty_like(want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(q_in, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call(q_in, out)
        for q, w in zip(qs, want):
            q_in.copy_(q)
            graph.replay()
            s.synchronize()
            assert torch.equal(out, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(5):
        for st, q in zip(streams, qs):
            with torch.cuda.stream(st):
                outs.append(call(q))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 3])


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_chunks_with_bad_ids_captured_and_at_once(fmt):
    """Eight chunks of 64 rows (128-row tiles): a slot and a block id outside their ranges, then captured, replayed
    on new data, and two launches on two streams at once."""
    H, D, S, n = 8, 64, 64, 8
    pool, vals = _pool(fmt, 64, 1, H, D, 15)
    table = torch.randperm(64, generator=_gen(16)).to(torch.int32).view(n, 8)
    table[3, 1], table[4, 2] = 64, -7
    q = torch.randn(n * S, 16, D, generator=_gen(17))
    slots = torch.arange(n).repeat_interleave(S).to(torch.int32)
    slots[5 * S:6 * S], slots[6 * S:7 * S] = -1, n
    ctx = (torch.arange(S) + 40).repeat(n).to(torch.int32)
    args = (pool, 0, table.to(DEV), slots.to(DEV), ctx.to(DEV), 128)
    qd = q.to(DEV)
    _lib.device_error()
    out = _attend(fmt, qd, *args, window=50, sinks=3, rows_per_stream=S)
    got = out.double().cpu().numpy()
    assert _lib.device_error() == 8
    assert not got[5 * S:7 * S].any()
    for b in (0, 3, 4, 7):
        ids = table[b].long()
        kv = vals[ids.clamp(0, 63), 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
        there = ((ids >= 0) & (ids < 64)).repeat_interleave(16).numpy()
        for t in (0, 1, 20, S - 1):
            r, c = b * S + t, int(ctx[t])
            see = O.visible(c, 128, 50, 3) & there
            want = O.attention(q[r].numpy(), kv[0][:, see], kv[1][:, see], int(see.sum()))
            assert (np.abs(got[r] - want) <= 2.0 ** -8 * np.abs(want) + _tolerance(fmt, q[r].numpy(), kv, True)).all()
    kw = dict(window=50, sinks=3, rows_per_stream=S)
    other = torch.randn(n * S, 16, D, generator=_gen(18)).to(DEV)
    want = [out.clone(), _attend(fmt, other, *args, **kw)]
    torch.cuda.synchronize()
    s, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            res = _attend(fmt, qd, *args, **kw)
        for data, w in ((other.clone(), want[1]), (q.to(DEV), want[0])):
            qd.copy_(data)
            graph.replay()
            s.synchronize()
            assert torch.equal(res, w)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            a = _attend(fmt, qd, *args, **kw)
        with torch.cuda.stream(s2):
            b = _attend(fmt, other, *args, **kw)
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert _lib.device_error() == 8


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_garbage_queries_of_padded_rows(fmt):
    """Rows without keys whose q holds NaN and infinity, among rows that have keys."""
    H, D, S = 2, 128, 40
    pool, vals = _pool(fmt, 4, 1, H, D, 5)
    table = torch.arange(4, dtype=torch.int32).view(1, 4)
    q = torch.randn(S, 4, D, generator=_gen(6))
    q[:S // 2:2], q[1:S // 2:2] = float("nan"), float("inf")
    ctx = torch.arange(S, dtype=torch.int32) - S // 2 + 1
    ctx[:S // 2] = 0
    slots = torch.zeros(S, dtype=torch.int32, device=DEV)
    for s in (1, S):
        out = _attend(fmt, q.to(DEV), pool, 0, table.to(DEV), slots, ctx.to(DEV), 64, rows_per_stream=s)
        out = out.double().cpu().numpy()
        assert not out[:S // 2].any()
        for r in range(S // 2, S):
            kv = vals[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
            want = O.attention(q[r].numpy(), kv[0], kv[1], int(ctx[r]))
            assert (np.abs(out[r] - want) <= 2.0 ** -8 * np.abs(want) + _tolerance(fmt, q[r].numpy(), kv, True)).all()


def test_first_call_inside_a_capture():
    """A process whose first calls are captured: the graph replays what eager calls give."""
    import subprocess
    import sys

    code = """
import torch
from test_stateful_b200 import ops
cache = torch.zeros(8, 1, 2, 2, 9 * 64, dtype=torch.uint8, device="cuda")
k = torch.randn(100, 2, 64, device="cuda"); m = torch.arange(100, dtype=torch.int32, device="cuda")
q = torch.randn(100, 4, 64, device="cuda"); t = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
z = torch.zeros(100, dtype=torch.int32, device="cuda"); c = m + 1
def step(s):
    ops.kv_write_q4(cache, k, -k, m)
    return ops.kv_read_q4(cache, m)[0], ops.paged_attention_q4(q, cache, 0, t, z, c, 128, 30, 2, rows_per_stream=s)
torch.cuda.synchronize()
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a = step(1) + step(100)
    g.replay()
    s.synchronize()
for x, y in zip(a, step(1) + step(100)):
    assert torch.equal(x, y)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
def test_pool_offsets_past_32_bits(fmt):
    """A pool of more than 2^32 bytes (and fp16 elements): its last blocks are written, read and attended."""
    H, D, L = 8, 128, 28
    per = L * 2 * H * (9 * D if fmt == "q4" else 16 * D * 2)
    nb = (2 ** 33 + 2 ** 30) // per
    if fmt == "q4":
        pool = torch.zeros(nb, L, 2, H, 9 * D, dtype=torch.uint8, device=DEV)
    else:
        pool = torch.zeros(nb, L, 2, H, 16, D, dtype=torch.float16, device=DEV)
    blocks = torch.tensor([nb - 1, nb - 3, nb // 2], dtype=torch.int32)
    ctx = 41
    x = torch.randn(3, 2, H, 16, D, generator=_gen(1)).half()
    if fmt == "q4":
        m = (blocks.repeat_interleave(16) * 16 + torch.arange(16).repeat(3)).to(torch.int32).to(DEV)
        rows = x.permute(0, 3, 1, 2, 4).reshape(48, 2, H, D).to(DEV)
        ops.kv_write_q4(pool, rows[:, 0], rows[:, 1], m, layer=L - 1)
        vals = O.values(*O.quantise(x.float().numpy()))
        rk, rv = ops.kv_read_q4(pool, m, layer=L - 1)
        want = vals.transpose(0, 3, 1, 2, 4).reshape(48, 2, H, D)
        _close_values(rk[:, 0], want[:, 0], torch.float16)
        _close_values(rv[:, 0], want[:, 1], torch.float16)
    else:
        pool[blocks.long().to(DEV), L - 1] = x.to(DEV)
        vals = x.double().numpy()
    q = torch.randn(1, 16, D, generator=_gen(2))
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = _attend(fmt, q.to(DEV), pool, L - 1, blocks.view(1, 3).to(DEV), one, one + ctx, 48).double().cpu().numpy()
    kv = vals.transpose(1, 2, 0, 3, 4).reshape(2, H, 48, D)
    want = O.attention(q[0].numpy(), kv[0], kv[1], ctx)
    assert (np.abs(out[0] - want) <= 2.0 ** -8 * np.abs(want) + _tolerance(fmt, q[0].numpy(), kv)).all()


# ------------------------------------------------------------------------------ as a server uses them
def test_streams_on_a_q4_pool():
    """The paged allocator over a 4-bit pool: prompts written, a prefix shared with copy-on-write, decode
    steps that append and attend (full, and windowed with sinks), and the slot read back."""
    from test_stateful_b200.runtime.model import PagedPoolTensors
    t = TalkerConfig(num_layers=2, hidden_size=256, num_heads=4, kv_heads=2, head_dim=64, intermediate_size=512)
    cfg = EngineConfig(talker=t, pool=PagedPoolConfig(block_size=16, num_blocks=64, max_slots=4, max_seq_len=256))
    pool = PagedPoolTensors(cfg, DEV, kv_format="q4")
    pool.init()
    sch = ops.Sched(pool)
    g = _gen(8)
    held = {0: [], 1: []}  # slot -> rows [n, 2L, H, D] written, as values

    def write(slot, rows, mapping):
        sch.scatter(rows.to(DEV), mapping)
        held[slot].append(O.values(*O.quantise(rows.float().numpy())))

    one = lambda s: torch.tensor([s], dtype=torch.int32, device=DEV)  # noqa: E731
    rows = torch.randn(23, 4, 2, 64, generator=g).half()
    m, *_ = sch.append(one(0), 23)
    write(0, rows, m)
    entry = sch.make_entry(0, 20)                 # a prefix that ends inside a block
    sch.share_prefix(1, entry, 20)
    held[1] = [np.concatenate(held[0])[:20]]
    both = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for step in range(30):
        m, ctx, _, cs, cd = sch.append(both, 1)
        sch.copy_blocks(cs, cd)                   # slot 1's first write into the shared block
        rows = torch.randn(2, 4, 2, 64, generator=g).half()
        for layer in range(2):                    # a decode step writes layer by layer
            ops.kv_write_q4(pool.kv, rows[:, 2 * layer].to(DEV), rows[:, 2 * layer + 1].to(DEV), m, layer=layer)
        for s in (0, 1):
            held[s].append(O.values(*O.quantise(rows[s:s + 1].float().numpy())))
        if step % 7:
            continue
        for layer, window, sinks in ((0, 0, 0), (1, 10, 3)):
            q = torch.randn(2, 4, 64, generator=g)
            lo = torch.empty(2, 256, device=DEV, dtype=torch.bfloat16)
            out = ops.paged_attention_q4(q.to(DEV), pool.kv, layer, pool.block_table, both, ctx, 256, window, sinks,
                                         out_lo=lo)
            out = (out.double() + lo.double()).cpu().numpy()
            for s in (0, 1):
                kv = np.concatenate(held[s])[:, 2 * layer:2 * layer + 2].transpose(1, 2, 0, 3)
                want = O.attention(q[s].numpy(), kv[0], kv[1], kv.shape[2], window, sinks)
                assert np.abs(out[s] - want).max() <= _tolerance("q4", q[s].numpy(), kv)
    for s in (0, 1):
        n = sum(len(h) for h in held[s])
        _close_values(sch.gather(s, n), np.concatenate(held[s]).transpose(1, 2, 0, 3), torch.float16)
    assert _lib.device_error() == 0 and int(sch.status.item()) == 0
