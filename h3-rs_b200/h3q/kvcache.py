"""h3q.kvcache -- an 8-bit paged key / value cache: quantised as tokens are written, read back, and attended to in place
(h3q_kv_*; no counterpart in the reference, whose models see their whole sequence in every call).

    cache = KVCache.empty(pages, kv_heads, page=64, head_dim=128, device=dev)        # int8 codes, or torch.float8_e4m3fn
    write(cache, k, v, page_table, past)              # k, v [tokens, kv_heads, head_dim]: bf16, f16 or f32
    out = attention(q, cache, page_table, past + new)      # q [tokens, heads, head_dim]: bf16 or f16
    k, v = read(cache, page_table, starts, total)     # dense rows again

Page p of kv head h holds `page` tokens and one scale for K and one for V; value = code * scale.  Sequence b's tokens
i * page .. are in page page_table[b, i].  The packed tokens of a call belong to its sequences by `starts` (int32
[batch + 1], ascending; rows before starts[0] or from starts[-1] on are not written, and zeros in an output), or evenly
without it.  page_table, past, lengths, first and starts are int32 CUDA tensors, which the host never reads.  Calls run on the
current stream of the cache's device.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import ERR_ARG, KV_E4M3, KV_INT8, H3QError, KvCacheDesc, check, lib

_KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CODES = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3}


class KVCache:
    """k, v codes [pages, kv_heads, page, head_dim] (int8 or float8_e4m3fn), k_scale, v_scale f32 [pages, kv_heads].  The
    tensors are checked once, here, and stay: others need another KVCache."""

    def __init__(self, k, v, k_scale, v_scale):
        shape, code = k.shape, _CODES.get(k.dtype)
        if len(shape) != 4 or v.shape != shape or v.dtype != k.dtype:
            raise H3QError(ERR_ARG, "KVCache: k and v are codes [pages, kv_heads, page, head_dim] of one type")
        if code is None:
            raise H3QError(ERR_ARG, "KVCache: codes are int8 or float8_e4m3fn")
        pages, heads, page, dim = shape
        f32, scales = torch.float32, (pages, heads)
        if k_scale.dtype != f32 or v_scale.dtype != f32 or k_scale.shape != scales or v_scale.shape != scales:
            raise H3QError(ERR_ARG, "KVCache: scales are f32 [pages, kv_heads]")
        device = k.get_device()  # -1: not a CUDA tensor
        if device < 0 or not (v.get_device() == k_scale.get_device() == v_scale.get_device() == device) or not (
                k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("h3q: expected contiguous CUDA tensors of one device")
        desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, page, dim, code)
        self.__dict__.update(k=k, v=v, k_scale=k_scale, v_scale=v_scale, device=device, heads=heads, dim=dim, desc=desc,
                             ref=ctypes.byref(desc))

    def __setattr__(self, name, value):
        raise AttributeError(f"KVCache: {name} stays as it was given")

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page: int = 64, head_dim: int = 128, dtype=torch.int8, device=None):
        """A pool without tokens.  A page's codes and scale mean nothing until its first token is written."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        codes = [torch.empty((pages, kv_heads, page, head_dim), dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])


def _call(cache, name, *args) -> None:
    """One call of the library on the current stream of the cache's device."""
    stream = torch._C._cuda_getCurrentRawStream(cache.device)
    if torch._C._cuda_getDevice() == cache.device:
        status = getattr(lib(), name)(cache.ref, *args, stream)
    else:
        with torch.cuda.device(cache.device):
            status = getattr(lib(), name)(cache.ref, *args, stream)
    if status:
        check(status)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(tokens, batch, heads, kv_heads, dim, max_new) -> int:
    return lib().h3q_kv_attention_workspace_size(tokens, batch, heads, kv_heads, dim, max_new)


def _ints(name, t, cache, n):
    """The address of t, checked to be the int32 [n] that a call reads; None for None."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or t.get_device() != cache.device or not t.is_contiguous():
        raise H3QError(ERR_ARG, f"kvcache: {name} is a contiguous int32 tensor [{n}] on the cache's device")
    return t.data_ptr()


def _table(t, cache):
    if t.dtype != torch.int32 or t.dim() != 2 or t.get_device() != cache.device or not t.is_contiguous():
        raise H3QError(ERR_ARG, "kvcache: the page table is a contiguous int32 tensor [batch, pages] on the cache's device")
    batch, width = t.shape
    return t.data_ptr(), batch, width


def _rows(name, x, cache, heads):
    """The token and head strides of rows x [tokens, heads, head_dim]."""
    shape = x.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != cache.dim or x.get_device() != cache.device:
        raise H3QError(ERR_ARG, f"kvcache: {name} is [tokens, {heads}, {cache.dim}] on the cache's device")
    ts, hs, es = x.stride()
    if es != 1:
        raise H3QError(ERR_ARG, f"kvcache: {name} needs unit stride inside a head")
    return ts, hs


def _kind(dtype) -> int:
    kind = _KIND.get(dtype)
    if kind is None:
        raise H3QError(ERR_ARG, "kvcache: rows are f32, f16 or bf16")
    return kind


def write(cache: KVCache, k, v, page_table, past, starts=None) -> None:
    """Appends k and v [tokens, kv_heads, head_dim] (f32, f16 or bf16; views of a fused projection are fine) behind the
    past [batch] tokens of each sequence.  A page's scale is max(old, amax * (1 / top)); where it grows, the page's older
    codes are rounded anew (h3q_kv_write has the formula)."""
    if k.dtype != v.dtype or k.shape != v.shape:
        raise H3QError(ERR_ARG, "kvcache: k and v have one shape and type")
    kind = _kind(k.dtype)
    kt, kh = _rows("k", k, cache, cache.heads)
    vt, vh = _rows("v", v, cache, cache.heads)
    table, batch, width = _table(page_table, cache)
    pp = _ints("past", past, cache, batch)
    sp = _ints("starts", starts, cache, batch + 1)
    _call(cache, "h3q_kv_write", k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, kind, k.shape[0], table, width, pp, sp, batch)


def read(cache: KVCache, page_table, starts, total: int, dtype=torch.bfloat16, first=None):
    """Tokens first[b] (0 without it) and on of each sequence, starts[b + 1] - starts[b] of them, as dense (k, v)
    [total, kv_heads, head_dim] of `dtype`."""
    kind = _kind(dtype)
    table, batch, width = _table(page_table, cache)
    sp = _ints("starts", starts, cache, batch + 1)
    fp = _ints("first", first, cache, batch)
    shape = (total, cache.heads, cache.dim)
    k = cache.k.new_empty(shape, dtype=dtype)
    v = torch.empty_like(k)
    _call(cache, "h3q_kv_read", table, width, fp, sp, batch, total, k.data_ptr(), v.data_ptr(), kind)
    return k, v


def attention(q, cache: KVCache, page_table, lengths, starts=None, scale: float | None = None, causal: bool = True,
              window: int = 0, return_lse: bool = False, max_new: int = 0, workspace=None):
    """softmax(scale * q . K) V of each sequence's newest tokens q [tokens, heads, head_dim] (f16 or bf16) over the first
    lengths [batch] tokens of its cache, the new ones included.  scale: head_dim ** -0.5 without it.  window > 0: the
    last `window` keys of each row.  max_new: an upper bound of the new tokens of one sequence, to be given with
    starts (without it one token each of ragged sequences takes about half as long again).  workspace: a contiguous tensor
    of the cache's device that no other call uses meanwhile (a new one where it is None or too small).  Returns [tokens,
    heads, head_dim], and with return_lse the f32 [tokens, heads] logarithms of the sums of exponentials."""
    if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
        raise H3QError(ERR_ARG, "kvcache: q is f16 or bf16")
    qt, qh = _rows("q", q, cache, q.shape[1] if q.dim() == 3 else 0)
    tokens, heads, dim = q.shape
    table, batch, width = _table(page_table, cache)
    lp = _ints("lengths", lengths, cache, batch)
    sp = _ints("starts", starts, cache, batch + 1)
    out = q.new_empty(q.shape)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    if starts is None and batch:
        max_new = tokens // batch
    need = _workspace_bytes(tokens, batch, heads, cache.heads, dim, max_new)
    if workspace is not None and (workspace.get_device() != cache.device or not workspace.is_contiguous()):
        raise H3QError(ERR_ARG, "kvcache: the workspace is a contiguous tensor on the cache's device")
    size = 0 if workspace is None else workspace.numel() * workspace.element_size()
    if workspace is None or size < need:
        workspace, size = q.new_empty(need, dtype=torch.uint8), need
    _call(cache, "h3q_kv_attention", q.data_ptr(), _KIND[q.dtype], qt, qh, tokens, heads, table, width, lp, sp, batch, max_new,
          dim ** -0.5 if scale is None else scale, causal, window, out.data_ptr(), lse.data_ptr() if return_lse else None,
          workspace.data_ptr(), size)
    return (out, lse) if return_lse else out


__all__ = ["KVCache", "write", "read", "attention"]
