"""Kernel-level Python API over the C ABI (torch tensors in, torch tensors out).

Each function launches one entry point of ``libqtts_b200.so`` on the current
CUDA stream.  Inputs must already be CUDA tensors of the stated dtype; there
is no CPU path.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("libqtts_b200 kernels take CUDA tensors only")


def split_hilo(x: torch.Tensor):
    """fp32 activation -> (hi, lo) bf16 pair with hi + lo ~ x."""
    hi = x.to(torch.bfloat16)
    return hi, (x - hi.float()).to(torch.bfloat16)


def gemm(x: torch.Tensor, w: torch.Tensor, epilogue: int = _lib.EPI_F32, out: Optional[torch.Tensor] = None,
         bias: Optional[torch.Tensor] = None, qkv: Optional[_lib.QkvEpilogue] = None,
         x_lo: Optional[torch.Tensor] = None, out_lo: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x [+ x_lo]) [M,K] bf16 · w [N,K]^T`` with a fused epilogue (see ``_lib.EPI_*``)."""
    _need_cuda(x, w, out, bias, x_lo, out_lo)
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        if epilogue == _lib.EPI_F32:
            out = torch.empty(M, N, device=x.device, dtype=torch.float32)
        elif epilogue == _lib.EPI_BF16:
            out = torch.empty(M, N, device=x.device, dtype=torch.bfloat16)
        elif epilogue == _lib.EPI_SWIGLU:
            out = torch.empty(M, N // 2, device=x.device, dtype=torch.bfloat16)
        else:
            raise ValueError("this epilogue needs an explicit out tensor")
    rc = _lib.load().qtts_gemm(x.data_ptr(), _lib.ptr(x_lo), M, K, w.data_ptr(), N, epilogue, out.data_ptr(),
                               _lib.ptr(out_lo), _lib.ptr(bias), C.byref(qkv) if qkv is not None else None,
                               _lib.stream_ptr())
    _lib.check(rc, "gemm")
    return out


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, rows: Optional[int] = None, ld: Optional[int] = None,
            out: Optional[torch.Tensor] = None, out_lo: Optional[torch.Tensor] = None) -> torch.Tensor:
    _need_cuda(x, w)
    H = w.shape[0]
    M = rows if rows is not None else x.numel() // H
    ld = ld if ld is not None else H
    if out is None:
        out = torch.empty(M, H, device=x.device, dtype=torch.bfloat16)
    _lib.check(_lib.load().qtts_rmsnorm(x.data_ptr(), M, H, ld, w.data_ptr(), eps, out.data_ptr(),
                                        _lib.ptr(out_lo), _lib.stream_ptr()), "rmsnorm")
    return out


def paged_attention(q: torch.Tensor, kv_pool: torch.Tensor, layer: int, block_table: torch.Tensor,
                    row_slot: torch.Tensor, row_ctx: torch.Tensor, max_ctx: int,
                    out: Optional[torch.Tensor] = None, ws_o: Optional[torch.Tensor] = None,
                    ws_ml: Optional[torch.Tensor] = None, out_lo: Optional[torch.Tensor] = None,
                    split_blocks: int = 0) -> torch.Tensor:
    """``q [R, Hq, D]`` fp32 over ``kv_pool [blocks, L, 2, Hkv, 16, D]`` fp16; ``split_blocks``
    KV blocks per split (0: the library default)."""
    _need_cuda(q, kv_pool, block_table, row_slot, row_ctx)
    R, Hq, D = q.shape
    nb, L, _, Hkv, bs, _ = kv_pool.shape
    n_blocks = -(-max_ctx // bs)
    splits = max(1, -(-n_blocks // (split_blocks or _lib.ATTN_SPLIT_BLOCKS)))
    if out is None:
        out = torch.empty(R, Hq * D, device=q.device, dtype=torch.bfloat16)
    if ws_o is None:
        ws_o = torch.empty(R * Hq * splits * D, device=q.device, dtype=torch.float32)
    if ws_ml is None:
        ws_ml = torch.empty(R * Hq * splits * 2, device=q.device, dtype=torch.float32)
    rc = _lib.load().qtts_paged_attention(q.data_ptr(), R, Hq, Hkv, D, kv_pool.data_ptr(), layer, L, bs, nb,
                                          block_table.data_ptr(), block_table.shape[-1], row_slot.data_ptr(),
                                          row_ctx.data_ptr(), max_ctx, split_blocks, ws_o.data_ptr(), ws_ml.data_ptr(),
                                          out.data_ptr(), _lib.ptr(out_lo), _lib.stream_ptr())
    _lib.check(rc, "paged_attention")
    return out


def paged_attention_prefill(q: torch.Tensor, kv_pool: torch.Tensor, layer: int, block_table: torch.Tensor,
                            row_slot: torch.Tensor, row_ctx: torch.Tensor, max_ctx: int, rows_per_stream: int,
                            out: Optional[torch.Tensor] = None, ws_o: Optional[torch.Tensor] = None,
                            ws_ml: Optional[torch.Tensor] = None, out_lo: Optional[torch.Tensor] = None,
                            split_blocks: int = 0) -> torch.Tensor:
    """Chunked-prefill attention (head_dim 128): ``q [R, Hq, D]`` holds ``R / rows_per_stream``
    streams of ``rows_per_stream`` consecutive query rows each (row_ctx causal: past + t + 1);
    the 8-query tiles of a stream share every KV block they read."""
    _need_cuda(q, kv_pool, block_table, row_slot, row_ctx)
    R, Hq, D = q.shape
    nb, L, _, Hkv, bs, _ = kv_pool.shape
    n_blocks = -(-max_ctx // bs)
    splits = max(1, -(-n_blocks // (split_blocks or _lib.ATTN_SPLIT_BLOCKS)))
    if out is None:
        out = torch.empty(R, Hq * D, device=q.device, dtype=torch.bfloat16)
    if ws_o is None:
        ws_o = torch.empty(R * Hq * splits * D, device=q.device, dtype=torch.float32)
    if ws_ml is None:
        ws_ml = torch.empty(R * Hq * splits * 2, device=q.device, dtype=torch.float32)
    rc = _lib.load().qtts_paged_attention_prefill(q.data_ptr(), R, rows_per_stream, Hq, Hkv, D, kv_pool.data_ptr(),
                                                  layer, L, bs, nb, block_table.data_ptr(), block_table.shape[-1],
                                                  row_slot.data_ptr(), row_ctx.data_ptr(), max_ctx, split_blocks,
                                                  ws_o.data_ptr(), ws_ml.data_ptr(), out.data_ptr(), _lib.ptr(out_lo),
                                                  _lib.stream_ptr())
    _lib.check(rc, "paged_attention_prefill")
    return out


# --------------------------------------------------------------------------- 4-bit KV cache, windowed attention
# These wrappers sit on a decode step's launch path: each check is one cheap attribute read.
_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}
_Strides = C.c_int64 * 3


def _same_device(*ts) -> int:
    """Index of the CUDA device that holds every tensor (None skipped)."""
    dev = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    if dev < 0:
        raise ValueError("libqtts_b200 kernels take CUDA tensors only")
    return dev


def _launch(dev: int, what: str, fn, *args):
    """Calls an entry point with ``dev`` current and its current stream."""
    if dev == torch.cuda.current_device():
        rc = fn(*args, _lib.raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, what)


def _need_i32(name: str, t: torch.Tensor, ndim: int):
    if t.dtype is not torch.int32 or t.dim() != ndim or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor of {ndim} dimension(s)")


def _q4_dims(cache: torch.Tensor):
    """(blocks, layers, kv heads, head_dim) of a 4-bit pool."""
    if cache.dtype is not torch.uint8 or cache.dim() != 5 or not cache.is_contiguous():
        raise ValueError("q4 cache: a contiguous uint8 tensor [blocks, layers, 2, kv_heads, 9 * head_dim]")
    nb, L, two, H, chunk = cache.shape
    if two != 2 or chunk not in (9 * 64, 9 * 128):
        raise ValueError(f"q4 cache: [.., 2, kv_heads, 9 * head_dim] with head_dim 64 or 128, got {tuple(cache.shape)}")
    return nb, L, H, chunk // 9


def _q4_rows(name: str, t: torch.Tensor, n: int, layers: Optional[int], H: int, D: int):
    """Layers, type and (token, layer, head) strides of K or V rows ``[n, (layers,) H, D]``."""
    shape, st = t.shape, t.stride()
    if len(shape) == 3:
        shape, st = (shape[0], 1, shape[1], shape[2]), (st[0], 0, st[1], st[2])
    if len(shape) != 4 or shape[0] != n or shape[2] != H or shape[3] != D or (layers or shape[1]) != shape[1]:
        raise ValueError(f"{name}: rows [{n}, {'layers' if layers is None else layers}, {H}, {D}], got {tuple(t.shape)}")
    dt = _DT.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name}: float16, bfloat16 or float32, got {t.dtype}")
    if st[3] != 1:
        raise ValueError(f"{name}: channels must be contiguous")
    # a dimension of one has no stride that matters
    return shape[1], dt, _Strides(st[0] if n > 1 else 0, st[1] if shape[1] > 1 else 0, st[2] if H > 1 else 0)


def kv_write_q4(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
                layer: int = 0) -> None:
    """Quantise K/V rows ``[n, Hkv, D]`` (one layer) or ``[n, layers, Hkv, D]`` (from ``layer`` on), fp16,
    bf16 or fp32 with any token, layer and head strides, into the positions ``slot_mapping [n]`` (block
    * 16 + offset, int32, distinct; negative ones are skipped) of a 4-bit pool."""
    dev = _same_device(cache, k, v, slot_mapping)
    nb, L, H, D = _q4_dims(cache)
    _need_i32("slot_mapping", slot_mapping, 1)
    n = slot_mapping.shape[0]
    layers, dt, ks = _q4_rows("k", k, n, None, H, D)
    if layer < 0 or not 1 <= layers <= L - layer:
        raise ValueError(f"kv_write_q4: layers [{layer}, +{layers}) of {L}")
    _, vdt, vs = _q4_rows("v", v, n, layers, H, D)
    if dt != vdt:
        raise ValueError(f"k is {k.dtype}, v is {v.dtype}")
    _launch(dev, "kv_write_q4", _lib.load().qtts_kv_write_q4, cache.data_ptr(), nb, L, H, D, k.data_ptr(), v.data_ptr(),
            dt, ks, vs, layer, layers, slot_mapping.data_ptr(), n)


def kv_read_q4(cache: torch.Tensor, slot_mapping: torch.Tensor, layer: int = 0, n_layers: int = 1,
               dtype: torch.dtype = torch.float16, k: Optional[torch.Tensor] = None,
               v: Optional[torch.Tensor] = None):
    """What the positions ``slot_mapping [n]`` of a 4-bit pool hold: ``(k, v)``, each ``[n, n_layers, Hkv,
    D]`` in ``dtype`` (or written to the given ``k``, ``v``); positions outside the pool read as zeros."""
    dev = _same_device(cache, slot_mapping, k, v)
    nb, L, H, D = _q4_dims(cache)
    _need_i32("slot_mapping", slot_mapping, 1)
    n = slot_mapping.shape[0]
    if dtype not in _DT:
        raise ValueError(f"kv_read_q4: float16, bfloat16 or float32, got {dtype}")
    if n_layers < 1 or layer < 0 or layer + n_layers > L:
        raise ValueError(f"kv_read_q4: layers [{layer}, +{n_layers}) of {L}")
    if k is None:
        k = torch.empty((n, n_layers, H, D), device=cache.device, dtype=dtype)
    if v is None:
        v = torch.empty((n, n_layers, H, D), device=cache.device, dtype=k.dtype)
    _, dt, ks = _q4_rows("k", k, n, n_layers, H, D)
    _, vdt, vs = _q4_rows("v", v, n, n_layers, H, D)
    if dt != vdt:
        raise ValueError(f"k is {k.dtype}, v is {v.dtype}")
    for st in (ks, vs):
        if (n > 1 and not st[0]) or (n_layers > 1 and k.dim() == 4 and not st[1]) or (H > 1 and not st[2]):
            raise ValueError("kv_read_q4: k and v must not be broadcast tensors")
    if n and k.data_ptr() == v.data_ptr():
        raise ValueError("kv_read_q4: k and v must not be the same memory")
    _launch(dev, "kv_read_q4", _lib.load().qtts_kv_read_q4, cache.data_ptr(), nb, L, H, D, k.data_ptr(), v.data_ptr(), dt,
            ks, vs, layer, n_layers, slot_mapping.data_ptr(), n)
    return k, v


def kv_gather_q4(cache: torch.Tensor, blocks: torch.Tensor, n_tokens: int,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The first ``n_tokens`` tokens of a block list (a block-table row, a prefix entry's ids) of a 4-bit
    pool, all layers: fp16 ``[2 L, Hkv, n_tokens, D]``, as :meth:`Sched.gather` of the fp16 pool."""
    dev = _same_device(cache, blocks, out)
    nb, L, H, D = _q4_dims(cache)
    _need_i32("blocks", blocks, 1)
    if n_tokens < 0 or n_tokens > 16 * blocks.shape[0]:
        raise ValueError(f"kv_gather_q4: {n_tokens} tokens of {blocks.shape[0]} blocks")
    if out is None:
        out = torch.empty((2 * L, H, n_tokens, D), device=cache.device, dtype=torch.float16)
    elif out.dtype is not torch.float16 or out.shape != (2 * L, H, n_tokens, D) or not out.is_contiguous():
        raise ValueError(f"kv_gather_q4: out must be contiguous fp16 [{2 * L}, {H}, {n_tokens}, {D}]")
    _launch(dev, "kv_gather_q4", _lib.load().qtts_kv_gather_q4, cache.data_ptr(), nb, L, H, D, blocks.data_ptr(), n_tokens,
            out.data_ptr())
    return out


def _window_attention(what, fn, q, kv, dims, layer, block_table, row_slot, row_ctx, max_ctx, window, sinks,
                      rows_per_stream, out, out_lo):
    dev = _same_device(q, kv, block_table, row_slot, row_ctx, out, out_lo)
    nb, L, H, D = dims
    if q.dtype is not torch.float32 or q.dim() != 3 or not q.is_contiguous():
        raise ValueError(f"{what}: q must be contiguous float32 [rows, heads, {D}]")
    R, Hq, qd = q.shape
    if qd != D:
        raise ValueError(f"{what}: head_dim {qd} over a pool of {D}")
    _need_i32("block_table", block_table, 2)
    _need_i32("row_slot", row_slot, 1)
    _need_i32("row_ctx", row_ctx, 1)
    slots, mbps = block_table.shape
    if not (0 <= layer < L and 0 < max_ctx <= 16 * mbps and 0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):
        raise ValueError(f"{what}: layer {layer} of {L}, max_ctx {max_ctx} of {16 * mbps}, window {window}, sinks {sinks}")
    if rows_per_stream < 1 or R % rows_per_stream:
        raise ValueError(f"{what}: {R} rows are not streams of {rows_per_stream} tokens")
    if row_slot.shape[0] != R or row_ctx.shape[0] != R:
        raise ValueError(f"{what}: {R} query rows, {row_slot.shape[0]} slots and {row_ctx.shape[0]} contexts")
    if out is None:
        out = torch.empty((R, Hq * D), device=q.device, dtype=torch.bfloat16)
    elif out.dtype is not torch.bfloat16 or out.numel() != R * Hq * D or not out.is_contiguous():
        raise ValueError(f"{what}: out must be contiguous bfloat16 [{R}, {Hq * D}]")
    if out_lo is not None and (out_lo.dtype is not torch.bfloat16 or out_lo.numel() != R * Hq * D
                               or not out_lo.is_contiguous()):
        raise ValueError(f"{what}: out_lo must be contiguous bfloat16 [{R}, {Hq * D}]")
    if out_lo is not None and R and out_lo.data_ptr() == out.data_ptr():
        raise ValueError(f"{what}: out and out_lo must not be the same memory")
    _launch(dev, what, fn, q.data_ptr(), R, rows_per_stream, Hq, H, D, kv.data_ptr(), layer, L, 16, nb,
            block_table.data_ptr(), slots, mbps, row_slot.data_ptr(), row_ctx.data_ptr(), max_ctx, window, sinks,
            out.data_ptr(), None if out_lo is None else out_lo.data_ptr())
    return out


def paged_attention_window(q: torch.Tensor, kv_pool: torch.Tensor, layer: int, block_table: torch.Tensor,
                           row_slot: torch.Tensor, row_ctx: torch.Tensor, max_ctx: int, window: int, sinks: int = 0,
                           rows_per_stream: int = 1, out: Optional[torch.Tensor] = None,
                           out_lo: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`paged_attention` under a sliding window: a row of context ``c`` sees key ``j < c`` when ``j >=
    c - window`` or ``j < sinks`` (``window`` 0: every key).  ``q [R, Hq, D]`` fp32 over ``kv_pool [blocks,
    L, 2, Hkv, 16, D]`` fp16, ``D`` 64 or 128, any whole ``Hq / Hkv``; rows without a visible key get
    zeros.  ``rows_per_stream`` > 1: the rows are streams of that many consecutive query tokens (a
    prompt chunk), which share the blocks they read.  Returns bf16 ``[R, Hq * D]`` (``out_lo``: its bf16
    residual; together they hold 16 bits, in whichever of its forms the call's sizes choose).  For plain causal
    attention with two query heads a KV head and ``D`` 128, :func:`paged_attention` and
    :func:`paged_attention_prefill` are as fast or faster."""
    if kv_pool.dtype is not torch.float16 or kv_pool.dim() != 6 or not kv_pool.is_contiguous():
        raise ValueError("paged_attention_window: a contiguous float16 pool [blocks, layers, 2, kv_heads, 16, head_dim]")
    nb, L, two, H, bs, D = kv_pool.shape
    if two != 2 or bs != 16:
        raise ValueError(f"paged_attention_window: pool [.., 2, kv_heads, 16, head_dim], got {tuple(kv_pool.shape)}")
    return _window_attention("paged_attention_window", _lib.load().qtts_paged_attention_window, q, kv_pool, (nb, L, H, D),
                             layer, block_table, row_slot, row_ctx, max_ctx, window, sinks, rows_per_stream, out, out_lo)


def paged_attention_q4(q: torch.Tensor, cache: torch.Tensor, layer: int, block_table: torch.Tensor,
                       row_slot: torch.Tensor, row_ctx: torch.Tensor, max_ctx: int, window: int = 0, sinks: int = 0,
                       rows_per_stream: int = 1, out: Optional[torch.Tensor] = None,
                       out_lo: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`paged_attention_window` over a 4-bit pool ``cache [blocks, L, 2, Hkv, 9 D]`` (uint8, written by
    :func:`kv_write_q4`); every key is visible by default.  Values enter as ``code * scale + zero``, unrounded or
    (128-row tiles of prompt chunks) to 2^-18 of their group's largest."""
    return _window_attention("paged_attention_q4", _lib.load().qtts_paged_attention_q4, q, cache, _q4_dims(cache), layer,
                             block_table, row_slot, row_ctx, max_ctx, window, sinks, rows_per_stream, out, out_lo)


def sample(logits: torch.Tensor, topk: int, gumbel: Optional[torch.Tensor] = None, temperature=None, penalty=None,
           counts: Optional[torch.Tensor] = None, eos_id: int = -1, seed: int = 0,
           noise_key: Optional[torch.Tensor] = None, step: int = 0, tok_out: Optional[torch.Tensor] = None,
           tok_ld: int = 1) -> torch.Tensor:
    """Talker head when ``counts`` is given (suppress + penalty + counts update), else CP select."""
    _need_cuda(logits, gumbel, temperature, penalty, counts, noise_key)
    R, V = logits.shape
    if tok_out is None:
        tok_out = torch.empty(R, device=logits.device, dtype=torch.int64)
        tok_ld = 1
    rc = _lib.load().qtts_sample(logits.data_ptr(), R, V, logits.stride(0), topk, _lib.ptr(gumbel),
                                 gumbel.stride(0) if gumbel is not None else 0, seed, _lib.ptr(noise_key), step,
                                 _lib.ptr(temperature), _lib.ptr(penalty), _lib.ptr(counts), eos_id,
                                 tok_out.data_ptr(), tok_ld, _lib.stream_ptr())
    _lib.check(rc, "sample")
    return tok_out


def philox_gumbel(seed: int, keys: torch.Tensor, frames: torch.Tensor, stage: int, cols: int = 50) -> torch.Tensor:
    """The Gumbel rows the samplers draw in-kernel for per-row ``keys`` (int64) and frame
    counters ``frames`` (int32) at ``stage`` (0: talker head, 1 + s: code-predictor stage s)."""
    _need_cuda(keys, frames)
    R = keys.numel()
    out = torch.empty(R, cols, device=keys.device, dtype=torch.float32)
    _lib.check(_lib.load().qtts_philox_gumbel(int(seed) & ((1 << 64) - 1), keys.data_ptr(), frames.data_ptr(), stage,
                                              R, cols, out.data_ptr(), _lib.stream_ptr()), "philox_gumbel")
    return out


def codec_sum(codes: torch.Tensor, talker_table: torch.Tensor, cp_tables: torch.Tensor,
              text_add: Optional[torch.Tensor] = None):
    """Returns ``(codec_sum fp32 [R,H], next_x fp32 [R,H])``."""
    _need_cuda(codes, talker_table, cp_tables, text_add)
    R, G = codes.shape
    V0, H = talker_table.shape
    Vc = cp_tables.shape[1]
    cs = torch.empty(R, H, device=codes.device, dtype=torch.float32)
    nx = torch.empty(R, H, device=codes.device, dtype=torch.float32)
    rc = _lib.load().qtts_codec_sum(codes.data_ptr(), R, G, talker_table.data_ptr(), V0, cp_tables.data_ptr(), Vc, H,
                                    _lib.ptr(text_add), cs.data_ptr(), nx.data_ptr(), _lib.stream_ptr())
    _lib.check(rc, "codec_sum")
    return cs, nx


class Sched:
    """Paged-state operations on a ``runtime.model.PagedPoolTensors``."""

    def __init__(self, pool):
        self.pool = pool
        self.lib = _lib.load()
        dev = pool.free_stack.device
        self.status = torch.zeros(1, device=dev, dtype=torch.int32)

    def append(self, slots: torch.Tensor, n_new: int):
        n = slots.numel()
        dev = slots.device
        mapping = torch.empty(n * n_new, device=dev, dtype=torch.int32)
        ctx = torch.empty_like(mapping)
        pos = torch.empty_like(mapping)
        cs = torch.empty(n, device=dev, dtype=torch.int32)
        cd = torch.empty_like(cs)
        rc = self.lib.qtts_sched_append(C.byref(self.pool.state), slots.data_ptr(), n, n_new, mapping.data_ptr(),
                                        ctx.data_ptr(), pos.data_ptr(), cs.data_ptr(), cd.data_ptr(),
                                        self.status.data_ptr(), _lib.stream_ptr())
        _lib.check(rc, "sched_append")
        return mapping, ctx, pos, cs, cd

    def copy_blocks(self, cs: torch.Tensor, cd: torch.Tensor):
        rc = self.lib.qtts_kv_copy_blocks(self.pool.kv.data_ptr(), self.pool.block_elems, self.pool.kv.shape[0],
                                          cs.data_ptr(), cd.data_ptr(), cs.numel(), _lib.stream_ptr())
        _lib.check(rc, "kv_copy_blocks")

    def share_prefix(self, slot: int, blocks: torch.Tensor, prefix_len: int):
        rc = self.lib.qtts_sched_share_prefix(C.byref(self.pool.state), slot, blocks.data_ptr(), prefix_len,
                                              self.status.data_ptr(), _lib.stream_ptr())
        _lib.check(rc, "sched_share_prefix")

    def make_entry(self, slot: int, prefix_len: int) -> torch.Tensor:
        bs = self.pool.state.block_size
        out = torch.empty(max(1, -(-prefix_len // bs)), device=self.pool.free_stack.device, dtype=torch.int32)
        rc = self.lib.qtts_sched_make_entry(C.byref(self.pool.state), slot, prefix_len, out.data_ptr(),
                                            _lib.stream_ptr())
        _lib.check(rc, "sched_make_entry")
        return out[: -(-prefix_len // bs)]

    def drop_blocks(self, blocks: torch.Tensor):
        rc = self.lib.qtts_sched_drop_blocks(C.byref(self.pool.state), blocks.data_ptr(), blocks.numel(),
                                             _lib.stream_ptr())
        _lib.check(rc, "sched_drop_blocks")

    def release(self, slot: int):
        _lib.check(self.lib.qtts_sched_release(C.byref(self.pool.state), slot, _lib.stream_ptr()), "sched_release")

    def scatter(self, rows: torch.Tensor, mapping: torch.Tensor):
        """rows ``[n, L*2, Hkv, D]`` fp16 into the pool (quantised when it is a 4-bit one)."""
        if self.pool.kv.dtype == torch.uint8:
            return kv_write_q4(self.pool.kv, rows[:, 0::2], rows[:, 1::2], mapping)
        L2, Hkv, D = rows.shape[1:]
        rc = self.lib.qtts_kv_scatter(self.pool.kv.data_ptr(), C.byref(self.pool.state), L2 // 2, Hkv, D,
                                      rows.data_ptr(), mapping.data_ptr(), rows.shape[0], _lib.stream_ptr())
        _lib.check(rc, "kv_scatter")

    def gather(self, slot: int, n: int) -> torch.Tensor:
        kv = self.pool.kv
        if kv.dtype == torch.uint8:
            if not 0 <= slot < self.pool.block_table.shape[0]:
                raise ValueError(f"kv_gather: slot {slot}")
            return kv_gather_q4(kv, self.pool.block_table[slot], n)
        L, Hkv, D = kv.shape[1], kv.shape[3], kv.shape[5]
        out = torch.empty(2 * L, Hkv, n, D, device=kv.device, dtype=torch.float16)
        rc = self.lib.qtts_kv_gather(kv.data_ptr(), C.byref(self.pool.state), L, Hkv, D, slot, n, out.data_ptr(),
                                     _lib.stream_ptr())
        _lib.check(rc, "kv_gather")
        return out
