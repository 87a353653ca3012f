"""h3q.cached -- one attention layer of a text model that runs token by token or chunk by chunk: the library's linears and
q / k RMSNorm + RoPE around the 8-bit key / value cache (h3q.kvcache).  The reference's text encoder sees its whole prompt at
once (text.rs:377-395); this is an attention layer of that kind, causal with shared kv heads, with what came before kept in
pages.  Its linears are int8 ConvRot layers and its head dim is 128; the encoder's own NVFP4 + AWQ linears
(h3q.nvfp4_linear) are not taken: a caller who has those makes the same calls around them.

    qkv = gemm_s8(x, qkv, rotate)                       [T, (heads + 2 kv_heads) * 128]
    q, k = qk_norm_rope(qkv columns, rope rows of the tokens' positions)
    write(cache, k, v)                                  behind the sequences' past tokens
    att = attention(q, cache)                           each new token against all before it and itself
    y = gemm_s8(att, out, rotate)

A prompt goes in with its tokens at once, or a chunk a call; a generated token with one row a sequence; drafted tokens with
a few.  Nothing here reads device memory on the host, so a step can be captured in a graph and replayed as past grows.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ERR_ARG, H3QError, gemm_s8, kvcache, qk_norm_rope
from .dit import Linear


@dataclass
class Layer:
    """qkv [(heads + 2 kv_heads) * 128, C] and out [C, heads * 128] are int8 ConvRot layers; q_norm, k_norm bf16 [128]."""
    qkv: Linear
    out: Linear
    q_norm: object
    k_norm: object
    heads: int
    kv_heads: int
    rot: int = 128
    eps: float = 1e-6


def positions(past, tokens: int, starts=None):
    """The position of each packed token: past[b] + its place among its sequence's new ones.  A token of no sequence (before
    starts[0] or from starts[-1] on) gets one that means nothing."""
    batch = past.numel()
    if batch == 0 and tokens > 0:
        raise H3QError(ERR_ARG, "cached: tokens without a sequence")
    at = torch.arange(tokens, device=past.device, dtype=torch.int32)
    if starts is None:
        each = tokens // max(1, batch)
        return past.repeat_interleave(each, output_size=tokens) + at % max(1, each)
    seq = torch.searchsorted(starts[1:], at, right=True).clamp_(max=max(0, batch - 1))
    return past[seq] + at - starts[seq]


def _rope_rows(rope, past, tokens: int, starts):
    """The tokens' rows of rope.  Positions are values on the device, which nothing checks before they index: one outside of the
    table takes its first or last row."""
    if rope.dim() != 3 or rope.shape[0] != 2 or rope.shape[1] < 1:
        raise H3QError(ERR_ARG, "cached: rope is [2, positions, rot / 2]")
    return rope[:, positions(past, tokens, starts).clamp_(0, rope.shape[1] - 1).long()].contiguous()


def attend(x, layer: Layer, cache: kvcache.KVCache, page_table, past, rope, starts=None, max_new: int = 0):
    """The layer on x bf16 [T, C], the new tokens of the sequences behind their past [batch] (int32) cached ones; rope f32
    [2, positions, rot / 2].  Writes the tokens' keys and values into the cache; returns bf16 [T, C].  The caller moves
    past on after the last layer.  rope reaches as far as the sequences do: a token behind its end is rotated as its last
    position, and one of no sequence (a captured step's padding) costs its row alone."""
    t, d, h, hk = x.shape[0], 128, layer.heads, layer.kv_heads
    qkv = gemm_s8(x, layer.qkv.w, layer.qkv.ws, layer.qkv.bias, rotate=True)
    cs = _rope_rows(rope, past, t, starts)
    q = qk_norm_rope(qkv, 0, h, d, (layer.q_norm, layer.eps), cs, layer.rot)
    k = qk_norm_rope(qkv, h * d, hk, d, (layer.k_norm, layer.eps), cs, layer.rot)
    v = qkv[:, (h + hk) * d:].unflatten(1, (hk, d))
    kvcache.write(cache, k, v, page_table, past, starts)
    new = t // max(1, past.numel()) if starts is None else starts[1:] - starts[:-1]
    att = kvcache.attention(q, cache, page_table, past + new, starts, max_new=max_new)
    return gemm_s8(att.reshape(t, h * d), layer.out.w, layer.out.ws, layer.out.bias, rotate=True)


__all__ = ["Layer", "positions", "attend"]
