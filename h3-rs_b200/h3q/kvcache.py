"""h3q.kvcache -- an 8-bit paged key / value cache: quantised as tokens are written, read back, and attended to in place
(h3q_kv_*; no counterpart in the reference, whose models see their whole sequence in every call).

    cache = KVCache.empty(pages, kv_heads, page=64, head_dim=128, device=dev)        # int8 codes, or torch.float8_e4m3fn
    write(cache, k, v, page_table, past)              # k, v [tokens, kv_heads, head_dim]: bf16, f16 or f32
    out = attention(q, cache, page_table, past + new)      # q [tokens, heads, head_dim]: bf16 or f16
    k, v = read(cache, page_table, starts, total)     # dense rows again

Page p of kv head h holds `page` tokens and one scale for K and one for V; value = code * scale.  Sequence b's tokens
i * page .. are in page page_table[b, i].  The packed tokens of a call belong to its sequences by `starts` (int32
[batch + 1], ascending from 0), or evenly without it.  page_table, past, lengths, first and starts are int32 CUDA tensors, which
the host never reads.  Calls run on the current stream of the cache's device.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import ERR_ARG, KV_E4M3, KV_INT8, H3QError, KvCacheDesc, _kind, _stream, check, lib


@dataclass
class KVCache:
    """k, v codes [pages, kv_heads, page, head_dim] (int8 or float8_e4m3fn), k_scale, v_scale f32 [pages, kv_heads]."""
    k: object
    v: object
    k_scale: object
    v_scale: object

    def __post_init__(self):
        import torch
        if self.k.dim() != 4 or self.k.shape != self.v.shape or self.k.dtype != self.v.dtype:
            raise H3QError(ERR_ARG, "KVCache: k and v are codes [pages, kv_heads, page, head_dim] of one type")
        if self.k.dtype not in (torch.int8, torch.float8_e4m3fn):
            raise H3QError(ERR_ARG, "KVCache: codes are int8 or float8_e4m3fn")
        for s in (self.k_scale, self.v_scale):
            if s.dtype != torch.float32 or s.shape != self.k.shape[:2]:
                raise H3QError(ERR_ARG, "KVCache: scales are f32 [pages, kv_heads]")
        for t in (self.k, self.v, self.k_scale, self.v_scale):
            if not t.is_cuda or not t.is_contiguous() or t.device != self.k.device:
                raise ValueError("h3q: expected contiguous CUDA tensors of one device")
        pages, heads, page, dim = self.k.shape
        self.desc = KvCacheDesc(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                                pages, heads, page, dim, KV_INT8 if self.k.dtype == torch.int8 else KV_E4M3)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page: int = 64, head_dim: int = 128, dtype=None, device=None):
        """A pool without tokens.  A page's codes and scale mean nothing until its first token is written."""
        import torch
        dtype = dtype or torch.int8
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        codes = [torch.empty((pages, kv_heads, page, head_dim), dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])


def _ints(name, t, cache, shape):
    """t as the int32 tensor that a call reads, checked."""
    import torch
    if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != cache.k.device or not t.is_contiguous():
        raise H3QError(ERR_ARG, f"kvcache: {name} is a contiguous int32 tensor {list(shape)} on the cache's device")
    return t.data_ptr()


def _rows(name, x, cache, heads):
    """The strides of rows x [tokens, heads, head_dim] whose heads are contiguous."""
    if x.dim() != 3 or x.shape[1] != heads or x.shape[2] != cache.k.shape[3] or x.device != cache.k.device:
        raise H3QError(ERR_ARG, f"kvcache: {name} is [tokens, {heads}, {cache.k.shape[3]}] on the cache's device")
    ts, hs, es = x.stride()
    if es != 1:
        raise H3QError(ERR_ARG, f"kvcache: {name} needs unit stride inside a head")
    return ts, hs


def _table(page_table, cache):
    if page_table.dim() != 2:
        raise H3QError(ERR_ARG, "kvcache: the page table is int32 [batch, pages]")
    batch, width = page_table.shape
    return _ints("page_table", page_table, cache, (batch, width)), batch, width


def write(cache: KVCache, k, v, page_table, past, starts=None) -> None:
    """Appends k and v [tokens, kv_heads, head_dim] (f32, f16 or bf16; views of a fused projection are fine) behind the
    past [batch] tokens of each sequence.  A page's scale is max(old, amax * (1 / top)); where it grows, the page's older codes are
    rounded anew (h3q_kv_write has the formula)."""
    heads = cache.k.shape[1]
    if k.dtype != v.dtype or k.shape != v.shape:
        raise H3QError(ERR_ARG, "kvcache: k and v have one shape and type")
    kind = _dtype(k.dtype)
    kt, kh = _rows("k", k, cache, heads)
    vt, vh = _rows("v", v, cache, heads)
    table, batch, width = _table(page_table, cache)
    pp = _ints("past", past, cache, (batch,))
    sp = None if starts is None else _ints("starts", starts, cache, (batch + 1,))
    check(lib().h3q_kv_write(ctypes.byref(cache.desc), k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, kind, k.shape[0], table,
                             width, pp, sp, batch, _stream(cache.k.device)))


def read(cache: KVCache, page_table, starts, total: int, dtype=None, first=None):
    """Tokens first[b] (0 without it) and on of each sequence, starts[b + 1] - starts[b] of them, as dense (k, v)
    [total, kv_heads, head_dim] of `dtype` (bf16 without it)."""
    import torch
    dtype = dtype or torch.bfloat16
    kind = _dtype(dtype)
    table, batch, width = _table(page_table, cache)
    sp = None if starts is None else _ints("starts", starts, cache, (batch + 1,))
    fp = None if first is None else _ints("first", first, cache, (batch,))
    shape = (total, cache.k.shape[1], cache.k.shape[3])
    k = torch.empty(shape, dtype=dtype, device=cache.k.device)
    v = torch.empty(shape, dtype=dtype, device=cache.k.device)
    check(lib().h3q_kv_read(ctypes.byref(cache.desc), table, width, fp, sp, batch, total, k.data_ptr(), v.data_ptr(), kind,
                            _stream(cache.k.device)))
    return k, v


def attention(q, cache: KVCache, page_table, lengths, starts=None, scale: float | None = None, causal: bool = True,
              window: int = 0, return_lse: bool = False, max_new: int = 0, workspace=None):
    """softmax(scale * q . K) V of each sequence's newest tokens q [tokens, heads, head_dim] (f16 or bf16) over the first
    lengths [batch] tokens of its cache, the new ones included.  scale: head_dim ** -0.5 without it.  window > 0: the
    last `window` keys of each row.  max_new: an upper bound of the new tokens of one sequence, where starts is given and the
    host knows one.  Returns [tokens, heads, head_dim], and with return_lse the f32 [tokens, heads] logarithms of the
    sums of exponentials."""
    import torch
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise H3QError(ERR_ARG, "kvcache: q is f16 or bf16")
    qt, qh = _rows("q", q, cache, q.shape[1] if q.dim() == 3 else 0)
    tokens, heads, dim = q.shape
    table, batch, width = _table(page_table, cache)
    lp = _ints("lengths", lengths, cache, (batch,))
    sp = None if starts is None else _ints("starts", starts, cache, (batch + 1,))
    out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if starts is None and batch:
        max_new = tokens // batch
    need = lib().h3q_kv_attention_workspace_size(tokens, batch, heads, cache.desc.kv_heads, dim, max_new)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    check(lib().h3q_kv_attention(ctypes.byref(cache.desc), q.data_ptr(), _kind(q.dtype), qt, qh, tokens, heads, table, width,
                                 lp, sp, batch, max_new, dim ** -0.5 if scale is None else scale, int(causal), window,
                                 out.data_ptr(), None if lse is None else lse.data_ptr(), workspace.data_ptr(),
                                 workspace.numel(), _stream(q.device)))
    return (out, lse) if return_lse else out


def _dtype(dtype) -> int:
    import torch
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise H3QError(ERR_ARG, "kvcache: rows are f32, f16 or bf16")
    return _kind(dtype)


__all__ = ["KVCache", "write", "read", "attention"]
