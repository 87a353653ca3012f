"""GPU test of a text layer on the 8-bit cache (h3q.cached): a prompt in ragged chunks, then tokens one at a time, then a few
drafted ones, each step checked against dense attention in f32 on what the cache holds, through the same linears.

The layer's attention is within 2^-8 (its bf16 rounding) + 2^-10 (f16 weights) of the dense one relative to sum p |v|; the
int8 output linear then quantises both rows: its own rounding, half a step of a row's largest rotated element over 127, on every
element of K = 512 random signs, gives a relative error under 2 / 127 of the row's rms.  Held: 3e-2 of the output's rms in the 2-norm.
"""
import pytest
import torch

import h3q
from h3q import cached, kvcache
from h3q.dit import Linear

pytestmark = pytest.mark.gpu


def make_layer(dev, c, heads, kv_heads, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def linear(n, k):
        w = torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int32).to(torch.int8)
        return Linear(w, torch.full((n,), 1.0 / (73 * k ** 0.5), device=dev))

    norm = [(1 + 0.1 * torch.randn(128, generator=g, device=dev)).bfloat16() for _ in range(2)]
    return cached.Layer(linear((heads + 2 * kv_heads) * 128, c), linear(c, heads * 128), norm[0], norm[1], heads, kv_heads)


def dense_step(x, layer, cache, table, past, rope, starts, totals, news):
    """The layer with the cache's contents read back and attended to in f32."""
    h, hk = layer.heads, layer.kv_heads
    pos = cached.positions(past, x.shape[0], starts).long()
    qkv = h3q.gemm_s8(x, layer.qkv.w, layer.qkv.ws, rotate=True)
    q = h3q.qk_norm_rope(qkv, 0, h, 128, (layer.q_norm, layer.eps), rope[:, pos].contiguous(), layer.rot).float()
    edges = [0]
    for t in totals:
        edges.append(edges[-1] + t)
    k, v = kvcache.read(cache, table, torch.tensor(edges, dtype=torch.int32, device=x.device), edges[-1], torch.float32)
    rows, at = [], 0
    for b, (t, n) in enumerate(zip(totals, news)):
        kb, vb = [z[edges[b]:edges[b + 1]].repeat_interleave(h // hk, 1) for z in (k, v)]
        s = torch.einsum("nhd,thd->hnt", q[at:at + n], kb) * 128 ** -0.5
        hide = torch.arange(t, device=x.device) > torch.arange(t - n, t, device=x.device)[:, None]
        rows.append(torch.einsum("hnt,thd->nhd", s.masked_fill(hide, float("-inf")).softmax(-1), vb))
        at += n
    att = torch.cat(rows).bfloat16().reshape(x.shape[0], h * 128)
    return h3q.gemm_s8(att, layer.out.w, layer.out.ws, rotate=True)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_layer_prompt_then_tokens_then_drafts(cuda, codes):
    c, heads, hk, page, batch = 1024, 4, 2, 32, 3
    layer = make_layer(cuda, c, heads, hk, 1)
    cache = kvcache.KVCache.empty(40, hk, page, 128, codes, cuda)
    table = torch.randperm(39, device=cuda, dtype=torch.int32).view(batch, 13)
    ang = torch.arange(400, device=cuda)[:, None] * 10000.0 ** (-torch.arange(64, device=cuda) / 64)
    rope = torch.stack([ang.cos(), ang.sin()]).float()
    g = torch.Generator(device=cuda)
    g.manual_seed(2)
    past = [0, 0, 0]
    steps = [[150, 33, 300], [40, 0, 1], [1, 1, 1], [1, 1, 1], [4, 4, 4], [1, 1, 1]]
    for news in steps:
        even = len(set(news)) == 1
        edges = [0, news[0], news[0] + news[1], sum(news)]
        starts = None if even else torch.tensor(edges, dtype=torch.int32, device=cuda)
        before = torch.tensor(past, dtype=torch.int32, device=cuda)
        x = torch.randn((sum(news), c), generator=g, device=cuda).bfloat16()
        y = cached.attend(x, layer, cache, table, before, rope, starts, max(news))
        past = [p + n for p, n in zip(past, news)]
        want = dense_step(x, layer, cache, table, before, rope, starts, past, news).float()
        assert torch.isfinite(y.float()).all()
        assert ((y.float() - want).norm() <= 3e-2 * want.norm()).item(), news
    assert h3q.device_status() == 0


def test_positions(cuda):
    past = torch.tensor([5, 0, 9], dtype=torch.int32, device=cuda)
    assert cached.positions(past, 6).tolist() == [5, 6, 0, 1, 9, 10]
    starts = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=cuda)
    assert cached.positions(past, 5, starts).tolist() == [5, 6, 9, 10, 11]
