"""GPU test of a text layer on the 8-bit cache (h3q.cached) against a history of its own: keys and values are taken from the
fused projection by their columns, normalised and rotated here in 64 bits at positions counted on the host, and kept per
sequence.  Nothing of what is compared with goes through attend or the cache.

What the cache holds of a key or value x, after its page has been written to w times since: it is rounded once when it comes and
once more each time the page's scale grows, to steps of at most the last scale s.  int8: w s / 2.  e4m3 (four significant
bits): w (2^-4 |x| 1.07^w + 2^-10 s), the factor for values that earlier roundings have moved.  x itself is a bf16 rounding
of the 64-bit value for keys (2^-8 |x|, and 2^-10 of the row's rms for the order of the sums under the root and in the
rotation), the projection's own bits for values.

Output, in the 2-norm against attention over the history in 64 bits: rounding K and V moves a score by about its step over sqrt(12)
and each weight with it, V by as much, independently over the keys, so the relative error is about sqrt(2 w) steps / sqrt(12) of
unit values: page maxima near 4 give 0.009 (int8) and 0.036 (e4m3) a rounding, 0.026 and 0.1 for the four at most that
a token sees here; the output linear quantises both sides' rows (3e-2, test_gpu_cached).  Held: 6e-2 and 1.5e-1; the other's norm moves it by
0.12 to 0.15, a rotation one place on by 0.19, a column of the next head by 1.4, and each what the cache holds far beyond its bound.
"""
import pytest
import torch

import h3q
from h3q import cached, kvcache
from test_gpu_cached import make_layer

pytestmark = pytest.mark.gpu


def norm_rope(x, w, eps, rope, pos):
    """x [n, heads, 128] (64 bits): RMSNorm times w, then rotated in halves by the rope rows `pos`."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    c, s = rope[0, pos].double()[:, None], rope[1, pos].double()[:, None]
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def make_rope(dev, n):
    ang = torch.arange(n, device=dev)[:, None] * 10000.0 ** (-torch.arange(64, device=dev) / 64)
    return torch.stack([ang.cos(), ang.sin()]).float()


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_layer_against_a_history_of_its_own(cuda, codes):
    c, h, hk, page, batch = 1024, 4, 2, 32, 3
    layer = make_layer(cuda, c, h, hk, 11)
    cache = kvcache.KVCache.empty(40, hk, page, 128, codes, cuda)
    table = torch.randperm(39, device=cuda, dtype=torch.int32).view(batch, 13)
    rope = make_rope(cuda, 400)
    g = torch.Generator(device=cuda)
    g.manual_seed(12)
    keys = [torch.zeros((0, hk, 128), dtype=torch.float64, device=cuda) for _ in range(batch)]
    vals = [k.clone() for k in keys]
    size = [torch.zeros((0, hk), dtype=torch.float64, device=cuda) for _ in range(batch)]  # rms of the keys' rows before the norm's weight
    writes = [torch.zeros(13, dtype=torch.int64) for _ in range(batch)]  # to each page of a sequence
    born = [[] for _ in range(batch)]  # writes to a token's page before its own
    for news in ([150, 33, 300], [40, 0, 1], [1, 1, 1], [4, 4, 4], [0, 90, 2]):
        past = [k.shape[0] for k in keys]
        edges = [0, news[0], news[0] + news[1], sum(news)]
        starts = None if len(set(news)) == 1 else torch.tensor(edges, dtype=torch.int32, device=cuda)
        x = torch.randn((sum(news), c), generator=g, device=cuda).bfloat16()
        y = cached.attend(x, layer, cache, table, torch.tensor(past, dtype=torch.int32, device=cuda), rope, starts, max(news))
        qkv = h3q.gemm_s8(x, layer.qkv.w, layer.qkv.ws, rotate=True).view(-1, h + 2 * hk, 128).double()
        rows = []
        for b, n in enumerate(news):
            if n == 0:
                continue
            pos = torch.arange(past[b], past[b] + n, device=cuda)
            mine = qkv[edges[b]:edges[b + 1]]
            q = norm_rope(mine[:, :h], layer.q_norm, layer.eps, rope, pos)
            keys[b] = torch.cat([keys[b], norm_rope(mine[:, h:h + hk], layer.k_norm, layer.eps, rope, pos)])
            vals[b] = torch.cat([vals[b], mine[:, h + hk:]])
            size[b] = keys[b].square().mean(-1).sqrt()
            for p in range(past[b] // page, (past[b] + n - 1) // page + 1):
                writes[b][p] += 1
            born[b] += [int(writes[b][t // page]) - 1 for t in range(past[b], past[b] + n)]
            s = torch.einsum("nhd,thd->hnt", q, keys[b].repeat_interleave(h // hk, 1)) * 128 ** -0.5
            s = s.masked_fill(torch.arange(past[b] + n, device=cuda) > pos[:, None], float("-inf"))
            rows.append(torch.einsum("hnt,thd->nhd", s.softmax(-1), vals[b].repeat_interleave(h // hk, 1)))
        att = torch.cat(rows).bfloat16().reshape(x.shape[0], h * 128)
        want = h3q.gemm_s8(att, layer.out.w, layer.out.ws, rotate=True).float()
        err = ((y.float() - want).norm() / want.norm()).item()
        assert err <= (6e-2 if codes == torch.int8 else 1.5e-1), (news, err)
    # what the cache holds in the end
    total = [k.shape[0] for k in keys]
    edges = torch.tensor([0, total[0], total[0] + total[1], sum(total)], dtype=torch.int32, device=cuda)
    got = kvcache.read(cache, table, edges, sum(total), torch.float32)
    for b in range(batch):
        at = int(edges[b])
        where = torch.arange(total[b], device=cuda) // page
        w = (writes[b].to(cuda)[where] - torch.tensor(born[b], device=cuda)).double()[:, None, None]
        for back, want, scale, key in ((got[0], keys[b], cache.k_scale, True), (got[1], vals[b], cache.v_scale, False)):
            step = scale[table[b].long()].double()[where][..., None]
            tol = w * (step / 2 if codes == torch.int8 else 2.0 ** -4 * want.abs() * 1.07 ** w + 2.0 ** -10 * step)
            tol = tol * (1 + 2.0 ** -12)
            if key:
                tol = tol + 2.0 ** -8 * want.abs() + 2.0 ** -10 * size[b][..., None]
            worst = ((back[at:at + total[b]].double() - want).abs() / tol).max().item()
            assert worst <= 1.0, (b, key, worst)
    assert h3q.device_status() == 0


def test_a_step_captured_and_replayed(cuda):
    """A padded decode step captured once and replayed as its sequences grow and end, against eager steps of the rows that count."""
    c, h, hk, page, batch, bucket = 512, 4, 2, 16, 3, 8
    layer = make_layer(cuda, c, h, hk, 13)
    rope = make_rope(cuda, 100)
    table = torch.arange(18, device=cuda, dtype=torch.int32).view(batch, 6)
    caches = [kvcache.KVCache.empty(18, hk, page, 128, device=cuda) for _ in range(2)]
    g = torch.Generator(device=cuda)
    g.manual_seed(14)
    prompt = torch.randn((60, c), generator=g, device=cuda).bfloat16()
    past = torch.tensor([20, 7, 33], dtype=torch.int32, device=cuda)
    zero = torch.zeros(3, dtype=torch.int32, device=cuda)
    for cache in caches:
        cached.attend(prompt, layer, cache, table, zero, rope, torch.tensor([0, 20, 27, 60], dtype=torch.int32, device=cuda))
    x = torch.zeros((bucket, c), dtype=torch.bfloat16, device=cuda)
    starts = torch.zeros(batch + 1, dtype=torch.int32, device=cuda)  # no tokens: nothing is written while it is captured
    now = past.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cached.attend(x, layer, caches[0], table, now, rope, starts, 2)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = cached.attend(x, layer, caches[0], table, now, rope, starts, 2)
    torch.cuda.synchronize()
    for news in ([1, 1, 1], [2, 1, 2], [1, 0, 2], [0, 0, 1], [2, 2, 2]):
        n = sum(news)
        rows = torch.randn((n, c), generator=g, device=cuda).bfloat16()
        edges = torch.tensor([0, news[0], news[0] + news[1], n], dtype=torch.int32, device=cuda)
        x.normal_()
        x[:n] = rows
        starts.copy_(edges)
        now.copy_(past)
        graph.replay()
        want = cached.attend(rows, layer, caches[1], table, past, rope, edges, 2)
        torch.cuda.synchronize()
        assert torch.equal(y[:n], want), news
        past = past + (edges[1:] - edges[:-1])
    for a, b in zip((caches[0].k_scale, caches[0].v_scale), (caches[1].k_scale, caches[1].v_scale)):
        assert torch.equal(a, b)
    assert h3q.device_status() == 0
