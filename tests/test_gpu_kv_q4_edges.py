"""Corners of the 4-bit KV cache and of windowed paged attention, against the float64 oracle.

Tolerances are those of ``test_gpu_kv_q4`` (derived there) unless a test derives its own."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import kv_q4 as O  # noqa: E402
from test_stateful_b200 import _lib, ops  # noqa: E402
from tests.test_gpu_kv_q4 import DEV, _attend, _expect, _gen, _new_cache, _pool, _same_bytes, _tolerance  # noqa: E402

FORCED = os.environ.get("QTTS_WINDOW_TILES")


# ------------------------------------------------------------------------------ rows without keys
@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("S,pad,last", [(38, 5, 100), (38, 5, 1500), (90, 27, 200), (90, 27, 520)])
@pytest.mark.parametrize("Hq,H,D", [(4, 2, 128), (8, 2, 64)])
def test_padded_rows_beside_whole_blocks(fmt, S, pad, last, Hq, H, D):
    """The last rows of a chunk are padding (context 0) whose q holds what memory held: finite numbers whose scores
    overflow, one infinite channel, NaN.  The other rows of their tile see whole blocks, so that no mask is
    applied there; keys of the long ones are shared by CTAs of a cluster."""
    nb = -(-last // 16)
    # keys of one sign, so that a huge q's scores overflow to +infinity over 4 bits too (zeros near 0)
    x = (torch.randn(nb, 1, 2, H, 16, D, generator=_gen(5)).abs() * 4).half()
    raw = x.numpy() if fmt == "fp16" else O.pack(*O.quantise(x.float().numpy()))
    pool, vals = torch.from_numpy(raw).to(DEV), x.double().numpy() if fmt == "fp16" else O.unpack(raw)
    table = torch.arange(nb, dtype=torch.int32).view(1, nb)
    q = torch.randn(S, Hq, D, generator=_gen(6)) / 4
    real = S - pad
    ctx = torch.zeros(S, dtype=torch.int32)
    ctx[:real] = torch.arange(last - real + 1, last + 1)
    fills = [lambda x: x[:, 3].fill_(3e38), lambda x: x.fill_(3e38), lambda x: x[:, 3].fill_(float("inf")),
             lambda x: x.mul_(1e38), lambda x: x.fill_(float("nan")), lambda x: x.fill_(float("inf"))]
    for r in range(real, S):
        fills[(r - real) % len(fills)](q[r])
    lo = torch.full((S, Hq * D), 9.0, device=DEV, dtype=torch.bfloat16)
    out = _attend(fmt, q.to(DEV), pool, 0, table.to(DEV), torch.zeros(S, dtype=torch.int32, device=DEV), ctx.to(DEV), last,
                  rows_per_stream=S, out_lo=lo)
    assert _lib.device_error() == 0
    assert not out[real:].any() and not lo[real:].any()
    got = (out.double() + lo.double()).cpu().numpy()
    kv = vals[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
    for r in range(0, real, 7):
        want = O.attention(q[r].numpy(), kv[0], kv[1], int(ctx[r]))
        assert np.abs(got[r] - want).max() <= _tolerance(fmt, q[r].numpy(), kv, True), r


# ------------------------------------------------------------------------------ small probabilities
def _dominant(fmt, n, at, D, fall):
    """A pool of one KV head and n keys, key ``at`` of value 0 scoring ``fall`` (nats) above all others for q = 8 e_0; the
    others' values lie in [4, 12].  Returns pool, keys and values [2, 1, n, D]."""
    nb = -(-n // 16)
    x = torch.zeros(nb * 16, 2, D)
    x[at, 0, 0] = fall * D ** 0.5 / 8
    x[:, 1] = 4 + 8 * torch.rand(nb * 16, D, generator=_gen(at))
    x[at, 1] = 0
    x = x.view(nb, 16, 2, 1, D).permute(0, 2, 3, 1, 4).unsqueeze(1).contiguous().half()
    raw = x.numpy() if fmt == "fp16" else O.pack(*O.quantise(x.float().numpy()))
    vals = x.double().numpy() if fmt == "fp16" else O.unpack(raw)
    return torch.from_numpy(raw).to(DEV), vals[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, 1, -1, D)[:, :, :n]


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [0, 17000, 32000])
@pytest.mark.parametrize("S", [1, 300])
def test_many_small_probabilities_beside_a_dominant_key(fmt, D, at, S):
    """32000 keys below 2^-25 of the largest probability are 1e-3 of the sum: they count in the output as they do there.
    Tolerance: a probability's fp16 halves end at 2^-32 of the maximum (half of 2^-31), n of them; relative errors of
    scores (27 in log2 units x 2^-22), ex2 (2^-22), probabilities (2^-16), sums and output (2^-17) below 2^-14."""
    n, rows = 32001, 300  # more tiles than CTAs fit at once: keys are not split, a warp walks thousands of them
    pool, kv = _dominant(fmt, n, at, D, 18.3)
    q = torch.zeros(rows, 2, D)
    q[:, :, 0] = 8
    zero = torch.zeros(rows, dtype=torch.int32, device=DEV)
    lo = torch.empty(rows, 2 * D, device=DEV, dtype=torch.bfloat16)
    out = _attend(fmt, q.to(DEV), pool, 0, torch.arange(pool.shape[0], dtype=torch.int32, device=DEV).view(1, -1), zero,
                  zero + n, n, rows_per_stream=S, out_lo=lo)
    got = (out.double() + lo.double()).cpu().numpy()
    want = O.attention(q[0].numpy(), kv[0], kv[1], n)
    assert want.min() > 1e-3
    assert (np.abs(got - want) <= n * 2.0 ** -32 * 12 + 2.0 ** -14 * want).all()


# ------------------------------------------------------------------------------ precision of chunks
def _chunk(fmt, S, past, Hq, H, D, qscale, seed=0):
    """Out + out_lo, the oracle's and the values' root mean square of every ninth row of a chunk of S after ``past`` keys."""
    n = S + past
    nb = -(-n // 16)
    pool, vals = _pool(fmt, nb, 1, H, D, seed + 11)
    q = torch.randn(S, Hq, D, generator=_gen(seed + 12)) * qscale
    zero = torch.zeros(S, dtype=torch.int32, device=DEV)
    ctx = torch.arange(past + 1, n + 1, dtype=torch.int32)
    lo = torch.empty(S, Hq * D, device=DEV, dtype=torch.bfloat16)
    out = _attend(fmt, q.to(DEV), pool, 0, torch.arange(nb, dtype=torch.int32, device=DEV).view(1, nb), zero, ctx.to(DEV), n,
                  rows_per_stream=S, out_lo=lo)
    got = (out.double() + lo.double()).cpu().numpy()
    kv = vals[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
    rows = range(0, S, 9)
    want = np.stack([O.attention(q[r].numpy(), kv[0], kv[1], past + 1 + r) for r in rows])
    return got[list(rows)], want, np.sqrt((kv[1] ** 2).mean())


@pytest.mark.parametrize("fmt", ["q4", "fp16"])
@pytest.mark.parametrize("Hq,H,D", [(4, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("S,past,qscale", [(150, 3, 1.0), (150, 100, 4.0), (70, 900, 2.0)])
def test_chunks_keep_sixteen_bits(fmt, Hq, H, D, S, past, qscale):
    """Out + out_lo of a chunk, root mean square over a row, whichever form the call goes through.  The output's halves
    leave 2^-17 of it, a probability's pair 2^-17 or less of it (its errors at random over the keys, and no more than
    one key's); q is held to 2^-20 of its largest channel or better, below 2^-20 * 3 qscale |k| / sqrt(D) <= 2^-17 qscale
    of a score, products and their fp32 sums less.  A probability moves by twice a score's error: together 2^-16 (1 +
    qscale) of the values, which rounding at random stays well below."""
    got, want, rms_v = _chunk(fmt, S, past, Hq, H, D, qscale)
    err = np.sqrt(((got - want) ** 2).mean(-1))
    assert err.max() <= 2.0 ** -16 * (1 + qscale) * rms_v, err.max() / rms_v


@pytest.mark.parametrize("Hq,H,D", [(16, 8, 128), (16, 4, 128), (16, 2, 128), (6, 2, 64), (4, 1, 64)])
@pytest.mark.parametrize("ctx,qscale", [(9, 1.0), (300, 4.0), (2000, 2.0)])
def test_decode_rows_keep_sixteen_bits_over_4_bits(Hq, H, D, ctx, qscale):
    """Decode rows whose q has a channel 30 times as loud as the rest, against the bound of the test above: the loud
    channel is 30 qscale, so that q is off by 2^-22 * 30 qscale a channel, 2^-17 qscale |k| / sqrt(D) of a score at the very
    most.  Its scores alone are large, so its K channel is 1/16 of the others'."""
    rows, nb = 5, -(-ctx // 16)
    x = torch.randn(nb, 1, 2, H, 16, D, generator=_gen(21))
    x[:, :, 0, :, :, 5] /= 16
    raw = O.pack(*O.quantise(x.half().float().numpy()))
    kv = O.unpack(raw)[:, 0].transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)
    q = torch.randn(rows, Hq, D, generator=_gen(22)) * qscale
    q[:, :, 5] = 30 * qscale
    zero = torch.zeros(rows, dtype=torch.int32, device=DEV)
    lo = torch.empty(rows, Hq * D, device=DEV, dtype=torch.bfloat16)
    out = ops.paged_attention_q4(q.to(DEV), torch.from_numpy(raw).to(DEV), 0,
                                 torch.arange(nb, dtype=torch.int32, device=DEV).view(1, nb), zero, zero + ctx, ctx,
                                 out_lo=lo)
    got = (out.double() + lo.double()).cpu().numpy()
    rms_v = np.sqrt((kv[1] ** 2).mean())
    for r in range(rows):
        want = O.attention(q[r].numpy(), kv[0], kv[1], ctx)
        assert np.sqrt(((got[r] - want) ** 2).mean()) <= 2.0 ** -16 * (1 + qscale) * rms_v, r


# ------------------------------------------------------------------------------ the cache
def test_write_groups_that_saturate_near_the_top():
    """fp32 values past 65504 are 65504 before they are coded, also where the group's zero is near 65504 itself (fp16(min)
    may round up, so that (65504 - zero) / scale is far from 15)."""
    g = _gen(41)
    n = 400
    lo = 65504 - torch.rand(n, 1, 1, 1, generator=g) * 10.0 ** (torch.rand(n, 1, 1, 1, generator=g) * 3.5 - 0.5)
    x = lo + (65504 - lo) * torch.rand(n, 1, 1, 128, generator=g)
    far = torch.rand(n, 1, 1, 128, generator=g) < 0.05
    x[far] = 65504 + 10.0 ** (torch.rand(int(far.sum()), generator=g) * 30)
    x[0], x[0, :, :, 7] = 65400.0, 1e6
    x[1], x[1, :, :, 7] = 65495.0, 1e6
    x[2], x[2, :, :, 7] = 65457.0, float("inf")
    x[3], x[3, :, :, :] = 65504.0, 70000.0
    assert (O.quantise(x[:2].numpy())[0][:, 0, 0, 0, 7] == [14, 0]).all()
    m = torch.arange(n, dtype=torch.int32)
    cache = _new_cache(n // 16, 1, 1, 128)
    ops.kv_write_q4(cache, x.to(DEV), (-x).to(DEV), m.to(DEV))
    want, _ = _expect(cache.shape, x, -x, m.tolist(), 0)
    _same_bytes(cache.cpu().numpy(), want, 128)


def test_outputs_that_are_one_memory_are_refused():
    """Both outputs in one tensor would be a mixture of the two."""
    cache = _new_cache(2, 1, 2, 64)
    m = torch.arange(3, dtype=torch.int32, device=DEV)
    rows = torch.zeros(3, 2, 64, device=DEV)
    q = torch.zeros(3, 4, 64, device=DEV)
    t = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    out = torch.zeros(3, 256, dtype=torch.bfloat16, device=DEV)
    pool = torch.zeros(2, 1, 2, 2, 16, 64, dtype=torch.float16, device=DEV)
    for call in (lambda: ops.kv_read_q4(cache, m, k=rows, v=rows),
                 lambda: ops.paged_attention_q4(q, cache, 0, t, m, m, 32, out=out, out_lo=out),
                 lambda: ops.paged_attention_window(q, pool, 0, t, m, m, 32, 8, out=out, out_lo=out.view(-1))):
        with pytest.raises(ValueError, match="same memory"):
            call()


def test_first_chunk_of_a_process_inside_a_capture():
    """The split of a tile's keys asks the card what it holds: also when the first call is captured."""
    code = """
import torch
from test_stateful_b200 import ops
pools = [torch.zeros(100, 1, 2, 2, 9 * 128, dtype=torch.uint8, device="cuda"),
         torch.randn(100, 1, 2, 2, 16, 128, device="cuda").half()]
k = torch.randn(1600, 2, 128, device="cuda"); m = torch.arange(1600, dtype=torch.int32, device="cuda")
q = torch.randn(200, 4, 128, device="cuda"); t = torch.arange(100, dtype=torch.int32, device="cuda").view(1, 100)
z = torch.zeros(200, dtype=torch.int32, device="cuda"); c = torch.arange(1401, 1601, dtype=torch.int32, device="cuda")
def step():
    ops.kv_write_q4(pools[0], k, -k, m)
    return (ops.paged_attention_q4(q, pools[0], 0, t, z, c, 1600, rows_per_stream=200),
            ops.paged_attention_window(q, pools[1], 0, t, z, c, 1600, 0, rows_per_stream=200))
torch.cuda.synchronize()
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a = step()
    g.replay()
    s.synchronize()
for x, y in zip(a, step()):
    assert torch.isfinite(x).all() and torch.equal(x, y)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for form in ("1", None):
        env = {k: v for k, v in os.environ.items() if k != "QTTS_WINDOW_TILES"}
        r = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(env, QTTS_WINDOW_TILES=form) if form else env,
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.skipif(FORCED is not None, reason="already a forced run")
@pytest.mark.parametrize("form", ["0", "1"])
def test_both_chunk_forms(form):
    """The chunk cases of this file through 8-row and 128-row tiles (QTTS_WINDOW_TILES is read once per process)."""
    env = dict(os.environ, QTTS_WINDOW_TILES=form)
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-k",
                        "padded or chunks or small", os.path.abspath(__file__)], env=env, capture_output=True, text=True, timeout=900,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
