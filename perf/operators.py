"""Measured cases of the 4-bit KV cache and of windowed paged attention.

Three operators of a serving step over the paged KV pool (16-token blocks):

* ``cache`` / ``read``: K/V rows quantised to 4 bits as they are written into the pool, and read
  back (a group is 64 channels of one token and head: fp16 scale and zero, 4-bit codes);
* ``q4``: GQA attention over that pool, decode rows and prompt chunks;
* ``window``: GQA attention over the fp16 pool with a sliding window and a few first tokens that
  stay visible.

``own`` selects the library's kernels; otherwise the plain form runs the same operator with
elementary torch operations in fp32.
"""

import math

import numpy as np
import torch

own = False

BLOCK = 16   # tokens per pool block
GROUP = 64   # channels that share a scale and a zero
LAYERS = 2   # layers of the attention cases' pools; the second one is read


def listed():
    return [
        # one decode step of one layer: 64 streams' new K and V, views of the QKV projection's output
        dict(name="cache_step_64", kind="cache", n=64, layers=1, kv_heads=8, head_dim=128, dtype="bfloat16"),
        # one prompt of 501 tokens, all 28 layers at once
        dict(name="cache_prompt_501", kind="cache", n=501, layers=28, kv_heads=8, head_dim=128, dtype="float16"),
        # a small model's fp32 rows
        dict(name="cache_small_37", kind="cache", n=37, layers=2, kv_heads=2, head_dim=64, dtype="float32"),
        # a cached text prefix of 97 tokens handed to a host as plain fp16, all layers
        dict(name="read_prefix_97", kind="read", n=97, layers=28, kv_heads=8, head_dim=128),
        # a whole session of 1000 tokens moved off the pool
        dict(name="read_session_1000", kind="read", n=1000, layers=28, kv_heads=8, head_dim=128),
        # the 64-stream decode step, ragged contexts around 520
        dict(name="q4_step_64", kind="q4", streams=64, rows=1, heads=16, kv_heads=8, head_dim=128, lo=260, hi=780,
             window=0, sinks=0),
        # one stream with a long context: the keys have to be split
        dict(name="q4_long_1", kind="q4", streams=1, rows=1, heads=16, kv_heads=8, head_dim=128, lo=32749, hi=32749,
             window=0, sinks=0),
        # a small model's step with a padding row (no keys) and four query heads per KV head, windowed
        dict(name="q4_small_5", kind="q4", streams=5, rows=1, heads=8, kv_heads=2, head_dim=64, lo=0, hi=200,
             window=72, sinks=4),
        # one 128-token prompt chunk of 8 streams after 384 cached tokens
        dict(name="q4_chunk_8x128", kind="q4", streams=8, rows=128, heads=16, kv_heads=8, head_dim=128, lo=512,
             hi=512, window=0, sinks=0),
        # the 64-stream decode step with the decoder's window of 72 keys and 4 sinks
        dict(name="window_step_64", kind="window", streams=64, rows=1, heads=16, kv_heads=8, head_dim=128, lo=260,
             hi=780, window=72, sinks=4),
        # long sessions, a wide window
        dict(name="window_long_16", kind="window", streams=16, rows=1, heads=16, kv_heads=4, head_dim=128, lo=2000,
             hi=8000, window=2048, sinks=4),
        # prompt chunks of two streams under a window that is shorter than the chunk
        dict(name="window_chunk_2x500", kind="window", streams=2, rows=500, heads=16, kv_heads=8, head_dim=128,
             lo=537, hi=1200, window=256, sinks=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "read", "q4", "q4", "window", "window"])
    if kind in ("cache", "read"):
        layers, kv_heads, head_dim = rng.choice([(1, 8, 128), (28, 8, 128), (2, 2, 64), (5, 8, 64), (3, 1, 128)])
        n = _log(rng, 1, 1000 if kind == "read" else 501)
        case = dict(kind=kind, n=n, layers=layers, kv_heads=kv_heads, head_dim=head_dim)
        if kind == "cache":
            case["dtype"] = rng.choice(["float16", "bfloat16"] if layers == 28 else ["float16", "bfloat16", "float32"])
        return case
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 4, 128), (8, 2, 64), (16, 2, 128),
                                            (8, 8, 64), (12, 4, 128)])
    case = dict(kind=kind, streams=1, rows=1, heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    if rng.random() < 0.65:   # decode rows
        case["streams"] = _log(rng, 1, 64)
        hi = _log(rng, 16, min(32749, 48000 // case["streams"]))
        case["lo"], case["hi"] = rng.randint(0, hi), hi
    else:                     # prompt chunks
        case["streams"] = _log(rng, 1, 8)
        case["rows"] = _log(rng, 2, 1000 // case["streams"])
        past = rng.choice([0, _log(rng, 1, 700)])
        case["lo"], case["hi"] = case["rows"], case["rows"] + past
    case["window"] = _log(rng, 1, 2048) if kind == "window" or rng.random() < 0.3 else 0
    case["sinks"] = rng.choice([0, 1, 4, 16, 33]) if case["window"] else 0
    return case


# ------------------------------------------------------------------ the pool's layout
# A chunk holds 16 tokens of one (block, layer, k or v, head): 16 rows of head_dim / 2 bytes of
# codes, then head_dim / 64 arrays of 16 (scale, zero) fp16 pairs.  A row's 32-bit words alternate
# between the groups; the low nibble of a word is its first channel.

def chunk_bytes(head_dim):
    return BLOCK * (head_dim // 2 + head_dim // GROUP * 4)


def quantise(x):
    """Rows ``[..., D]`` -> codes uint8 ``[..., D/64, 64]``, scale and zero fp16 ``[..., D/64]``."""
    x = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    zero = lo.half()
    scale = ((hi - lo) * (1.0 / 15.0)).half()
    # the quotient in 64 bits: it decides between two codes next to a border
    quot = (x - zero.float().unsqueeze(-1)).double() / scale.double().unsqueeze(-1)
    code = quot.round().clamp(0, 15)
    return torch.where((scale == 0).unsqueeze(-1), torch.zeros_like(code), code).to(torch.uint8), scale, zero


def dequantise(code, scale, zero):
    return (code.float() * scale.float().unsqueeze(-1) + zero.float().unsqueeze(-1)).flatten(-2)


def pack(code, scale, zero):
    """``[..., 16, D/64, 64]`` codes and ``[..., 16, D/64]`` params -> bytes ``[..., chunk]``."""
    words = code.unflatten(-1, (8, 4, 2)).transpose(-4, -3)         # [..., 16, 8 words, groups, 4, 2]
    codes = (words[..., 0] | (words[..., 1] << 4)).flatten(-4)
    params = torch.stack([scale, zero], -1).transpose(-3, -2).contiguous().view(torch.uint8).flatten(-3)
    return torch.cat([codes, params], -1)


def unpack(chunk, head_dim):
    groups = head_dim // GROUP
    b = chunk[..., :BLOCK * head_dim // 2].unflatten(-1, (BLOCK, 8, groups, 4))
    code = torch.stack([b & 15, b >> 4], -1).transpose(-4, -3).flatten(-3)
    params = chunk[..., BLOCK * head_dim // 2:].contiguous().view(torch.float16).unflatten(-1, (groups, BLOCK, 2))
    params = params.transpose(-3, -2)
    return code, params[..., 0], params[..., 1]


# ------------------------------------------------------------------ inputs

def _rows(gen, dev, shape):
    """K/V-like rows: unit variance with a few loud channels per head."""
    loud = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=gen, device=dev) > 0.94)
    return torch.randn(shape, generator=gen, device=dev) * loud


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    H, D = case["kv_heads"], case["head_dim"]
    if case["kind"] in ("cache", "read"):
        n, L = case["n"], case["layers"]
        blocks = n // BLOCK + 3
        ids = torch.randperm(blocks, generator=gen, device=dev).int()[:-(-n // BLOCK)]
        mapping = (ids.repeat_interleave(BLOCK) * BLOCK + torch.arange(BLOCK, device=dev).repeat(len(ids)))[:n].int()
        if case["kind"] == "cache":
            dt = getattr(torch, case["dtype"])
            if L == 1:   # views of a QKV projection's output, q first
                qkv = _rows(gen, dev, (n, 4 * H, D)).to(dt)
                k, v = qkv[:, 2 * H:3 * H].unsqueeze(1), qkv[:, 3 * H:].unsqueeze(1)
            else:        # [token][layer][k, v][head][channel]
                kv = _rows(gen, dev, (n, L, 2, H, D)).to(dt)
                k, v = kv[:, :, 0], kv[:, :, 1]
            cache = torch.zeros(blocks, L, 2, H, chunk_bytes(D), dtype=torch.uint8, device=dev)
            return dict(case=case, cache=cache, k=k, v=v, mapping=mapping)
        x = _rows(gen, dev, (blocks, L, 2, BLOCK, H, D)).half().transpose(-3, -2)
        return dict(case=case, cache=pack(*quantise(x)), blocks=ids)
    S, n = case["rows"], case["streams"]
    ctx = torch.randint(case["lo"], case["hi"] + 1, (n,), generator=gen, device=dev)
    if n > 1:            # the ends of the range are there
        ctx[0], ctx[-1] = case["hi"], case["lo"]
    width = max(1, -(-case["hi"] // BLOCK))
    have = (ctx + BLOCK - 1) // BLOCK
    used = torch.arange(width, device=dev)[None, :] < have[:, None]
    total = n * width
    table = torch.where(used, torch.randperm(total, generator=gen, device=dev).view(n, width), -1).int()
    q = torch.randn(n * S, case["heads"], D, generator=gen, device=dev)
    row_slot = torch.arange(n, device=dev).repeat_interleave(S).int()
    row_ctx = (ctx[:, None] - S + 1 + torch.arange(S, device=dev)[None, :]).flatten().int()
    x = _rows(gen, dev, (total, LAYERS, 2, BLOCK, H, D)).half().transpose(-3, -2).contiguous()
    return dict(case=case, q=q, table=table, row_slot=row_slot, row_ctx=row_ctx, max_ctx=width * BLOCK,
                kv=x if case["kind"] == "window" else pack(*quantise(x)))


# ------------------------------------------------------------------ one pass

def run(st):
    c = st["case"]
    if own:
        return _run_own(st, c)
    D = c["head_dim"]
    if c["kind"] == "cache":
        m = st["mapping"].long()
        blk, off = m // BLOCK, m % BLOCK
        bytes_of = st["cache"]
        G, half = D // GROUP, D // 2
        rows = bytes_of[..., :BLOCK * half].unflatten(-1, (BLOCK, 8, G, 4))                     # views of the cache
        prm = bytes_of[..., BLOCK * half:].unflatten(-1, (G, BLOCK, 4))
        kv = torch.stack([st["k"], st["v"]], 2)                                                 # [n, L, 2, H, D]
        code, scale, zero = quantise(kv)
        words = code.unflatten(-1, (8, 4, 2)).transpose(-4, -3)
        rows[blk, :, :, :, off] = words[..., 0] | (words[..., 1] << 4)
        pair = torch.stack([scale, zero], -1).view(torch.uint8)
        prm[blk, :, :, :, :, off] = pair
        b = rows[blk, :, :, :, off]
        code = torch.stack([b & 15, b >> 4], -1).transpose(-4, -3).flatten(-3)
        pair = prm[blk, :, :, :, :, off].contiguous().view(torch.float16)
        x = dequantise(code, pair[..., 0], pair[..., 1]).to(st["k"].dtype)
        return x[:, :, 0], x[:, :, 1]
    if c["kind"] == "read":
        code, scale, zero = unpack(st["cache"][st["blocks"].long()], D)                         # [nb, L, 2, H, 16, ..]
        x = dequantise(code, scale, zero).half()
        return x.permute(1, 2, 3, 0, 4, 5).flatten(3, 4)[..., :c["n"], :].flatten(0, 1).contiguous()
    n, S, H, Hq = c["streams"], c["rows"], c["kv_heads"], c["heads"]
    pages = st["kv"][:, LAYERS - 1][st["table"].clamp_min(0).long()]                            # [n, nb, 2, H, ...]
    pages = dequantise(*unpack(pages, D)) if c["kind"] == "q4" else pages.float()               # [n, nb, 2, H, 16, D]
    kv = pages.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)                                          # [2, n, H, keys, D]
    q = st["q"].view(n, S, H, Hq // H, D).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.flatten(2, 3), kv[0].transpose(-1, -2)).unflatten(2, (Hq // H, S)) / math.sqrt(D)
    ctx = st["row_ctx"].view(n, 1, 1, S, 1)
    j = torch.arange(kv.shape[3], device=s.device)
    seen = j < ctx
    if c["window"]:
        seen = seen & ((j >= ctx - c["window"]) | (j < c["sinks"]))
    s = torch.where(seen, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, (s - torch.where(top.isinf(), 0.0, top)).exp(), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.flatten(2, 3), kv[1]).unflatten(2, (Hq // H, S))
    return o.permute(0, 3, 1, 2, 4).reshape(n * S, Hq * D).bfloat16()


def _run_own(st, c):
    from test_stateful_b200 import ops
    if c["kind"] == "cache":
        ops.kv_write_q4(st["cache"], st["k"], st["v"], st["mapping"])
        return ops.kv_read_q4(st["cache"], st["mapping"], n_layers=c["layers"], dtype=st["k"].dtype)
    if c["kind"] == "read":
        return ops.kv_gather_q4(st["cache"], st["blocks"], c["n"])
    attend = ops.paged_attention_q4 if c["kind"] == "q4" else ops.paged_attention_window
    return attend(st["q"], st["kv"], LAYERS - 1, st["table"], st["row_slot"], st["row_ctx"], st["max_ctx"],
                  window=c["window"], sinks=c["sinks"], rows_per_stream=c["rows"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    H, D = case["kv_heads"], case["head_dim"]
    if case["kind"] in ("cache", "read"):
        values = case["n"] * case["layers"] * 2 * H * D
        held = values // 2 + values // GROUP * 4
        if case["kind"] == "read":
            return dict(bytes=held + 2 * values, flops=2 * values)
        return dict(bytes=held + 2 * values * (4 if case["dtype"] == "float32" else 2), flops=6 * values)
    n, S = case["streams"], case["rows"]
    per_key = 2 * H * (D // 2 + D // GROUP * 4 if case["kind"] == "q4" else 2 * D)
    top = 1 << 30
    w, sinks = case["window"] or top, case["sinks"]

    def seen(ctx):
        return min(ctx, w + min(sinks, max(0, ctx - w)))

    # contexts are spread evenly over [lo, hi]: their mean stands for them
    points = [case["lo"] + (case["hi"] - case["lo"]) * i / 8 for i in range(9)] if n > 1 else [case["hi"]]
    keys = sum(min(c, seen(c) + (min(S - 1, max(0, c - seen(c))) if case["window"] else 0)) for c in points) / len(points)
    pairs = sum(sum(seen(max(0, c - S + 1 + t)) for t in range(S)) for c in points) / len(points)
    rows = n * S * case["heads"] * D
    return dict(bytes=int(n * keys * per_key + rows * (4 + 2)), flops=int(4 * D * case["heads"] * n * pairs))


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_values(x):
    """What 4 bits keep of ``x [..., D]`` (float64 holding the inputs), in numpy float64."""
    x = np.clip(x.detach().float().cpu().numpy(), -65504.0, 65504.0)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    zero = lo.astype(np.float16)
    scale = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16).astype(np.float64)
    step = (g - zero.astype(np.float32)).astype(np.float64) / np.where(scale == 0, np.inf, scale)
    return (np.clip(np.rint(step), 0, 15) * scale + zero.astype(np.float64)).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "cache":
        return tuple(torch.from_numpy(_exact_values(st[x])) for x in ("k", "v"))
    D = case["head_dim"]
    if case["kind"] == "read" or case["kind"] == "q4":
        half = BLOCK * D // 2
        raw = st["cache" if case["kind"] == "read" else "kv"].cpu().numpy()
        if case["kind"] == "q4":
            raw = raw[:, LAYERS - 1]
        words = np.ascontiguousarray(raw[..., :half]).view("<u4").astype(np.int64)
        words = words.reshape(*raw.shape[:-1], BLOCK, 8, D // GROUP)
        params = np.ascontiguousarray(raw[..., half:]).view("<f2").astype(np.float64)
        params = params.reshape(*raw.shape[:-1], D // GROUP, BLOCK, 2)
        pool = np.empty((*raw.shape[:-1], BLOCK, D))
        for ch in range(D):
            g, i = ch // GROUP, ch % GROUP
            code = (words[..., :, i // 8, g] >> (4 * (i % 8))) & 15
            pool[..., ch] = code * params[..., g, :, 0] + params[..., g, :, 1]
    else:
        pool = st["kv"][:, LAYERS - 1].cpu().numpy().astype(np.float64)
    if case["kind"] == "read":
        x = pool[st["blocks"].cpu().numpy()]                       # [nb, L, 2, H, 16, D]
        x = np.moveaxis(x, 0, 3).reshape(*x.shape[1:4], -1, D)[:, :, :, :case["n"]]
        return torch.from_numpy(np.ascontiguousarray(x.reshape(-1, *x.shape[2:])))
    dev = st["q"].device
    table, ctx = st["table"].cpu().numpy(), st["row_ctx"].cpu().numpy()
    H, Hq, S = case["kv_heads"], case["heads"], case["rows"]
    q = st["q"].double()
    out = torch.zeros(len(q), Hq, D, dtype=torch.float64, device=dev)
    for b in range(case["streams"]):
        last = int(ctx[b * S + S - 1])
        if last <= 0:
            continue
        blocks = table[b, :-(-last // BLOCK)]
        kv = torch.from_numpy(pool[blocks]).to(dev)                # [nb, 2, H, 16, D]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, H, -1, D)[:, :, :last]
        rows = slice(b * S, b * S + S)
        c = st["row_ctx"][rows].long()[:, None]
        j = torch.arange(last, device=dev)[None, :]
        hide = j >= c
        if case["window"]:
            hide = hide | ((j < c - case["window"]) & (j >= case["sinks"]))
        for h in range(Hq):
            s = (q[rows, h] @ kv[0, h // (Hq // H)].T) / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            out[rows, h] = torch.nan_to_num(p) @ kv[1, h // (Hq // H)]
    return out.reshape(len(q), Hq * D)
