"""Measured cases of the 8-bit paged key / value cache: writing it, reading it back and attending to it.

A cache is a pool of pages.  Page p of kv head h holds `page` tokens of `dim` 8-bit codes (int8 or e4m3) for K and for
V, and one f32 scale each: k = code * k_scale[p, h].  A sequence names its pages in its row of the page table.

  write      new keys and values are quantised into the pages behind a sequence's `past` tokens.  A page's scale is
             max(old scale, largest |x| / top) (top 127 or 448, at least 1e-30; no old scale where the page is
             begun); where it grows the page's older codes are rounded anew.  The written pages are then read back.
  read       a span of each sequence's tokens as dense rows of 16 or 32 bits.
  attention  each query row against the tokens of its sequence: softmax(scale * q . k) v, causal or not, windowed or
             not; the queries are a sequence's newest tokens.

`own` selects the library's kernels; otherwise the plain form runs: elementary torch operations in 32 bits on padded
tensors."""
import math
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_FLOOR = 1e-30


def listed():
    return [
        # one generated token for each of 64 conversations of unlike lengths: latency, and pages that grow their scale
        dict(name="write decode b64", op="write", batch=64, new=1, past=4096, ragged=True, kv_heads=8, dim=128, page=64,
             codes="int8", dtype="bf16"),
        # a batch of prompts goes into an empty cache
        dict(name="write prompts 4x8192", op="write", batch=4, new=8192, past=0, ragged=True, kv_heads=8, dim=128,
             page=64, codes="e4m3", dtype="bf16"),
        # a chunk behind odd lengths, every head its own kv head, small pages, read back in 32 bits
        dict(name="write chunk mha odd", op="write", batch=3, new=1019, past=333, ragged=True, kv_heads=40, dim=128,
             page=16, codes="int8", dtype="f32"),
        # one conversation's cache handed to a path that wants 16 bits
        dict(name="read 777", op="read", batch=1, length=777, ragged=False, kv_heads=8, dim=128, page=64, codes="int8",
             dtype="bf16"),
        # a batch of long sequences read back
        dict(name="read 16x8192", op="read", batch=16, length=8192, ragged=True, kv_heads=8, dim=128, page=32,
             codes="e4m3", dtype="bf16"),
        # the first tokens of one short conversation: the smallest call
        dict(name="decode 1x500", op="attention", batch=1, new=1, length=500, ragged=False, heads=64, kv_heads=8,
             dim=128, page=64, codes="int8", dtype="bf16", causal=True, window=0),
        # one very long conversation, one token at a time: a long axis and few rows
        dict(name="decode 1x131000", op="attention", batch=1, new=1, length=131000, ragged=False, heads=64, kv_heads=8,
             dim=128, page=64, codes="int8", dtype="bf16", causal=True, window=0),
        # serving: 64 conversations of unlike lengths, one token each
        dict(name="decode 64x16384", op="attention", batch=64, new=1, length=16384, ragged=True, heads=40, kv_heads=8,
             dim=128, page=64, codes="int8", dtype="bf16", causal=True, window=0),
        # five drafted tokens of each of 16 conversations checked in one pass
        dict(name="draft 16x5", op="attention", batch=16, new=5, length=4099, ragged=True, heads=40, kv_heads=8,
             dim=128, page=32, codes="e4m3", dtype="bf16", causal=True, window=0),
        # a prompt chunk behind a long prefix
        dict(name="chunk 2048 of 10240", op="attention", batch=2, new=2048, length=10240, ragged=False, heads=32,
             kv_heads=8, dim=128, page=64, codes="e4m3", dtype="bf16", causal=True, window=0),
        # ragged prompts with a sliding window, head dim 64, every head its own kv head
        dict(name="window 6x4000 d64", op="attention", batch=6, new=1500, length=4000, ragged=True, heads=16,
             kv_heads=16, dim=64, page=16, codes="int8", dtype="f16", causal=True, window=1024),
        # cross attention of a chunk of the packed stream to all tokens of a long one
        dict(name="cross 1000 of 32760", op="attention", batch=1, new=1000, length=32760, ragged=False, heads=40,
             kv_heads=40, dim=128, page=128, codes="int8", dtype="bf16", causal=False, window=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: batch 1..96, lengths 1..131072, 1 to 8 query heads for each kv head."""
    while True:
        op = rng.choice(["write", "write", "read", "attention", "attention", "attention", "attention"])
        c = dict(op=op, batch=_log(rng, 1, 96), ragged=rng.random() < 0.6, kv_heads=rng.choice([1, 2, 4, 8, 16, 40]),
                 dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128]), codes=rng.choice(["int8", "e4m3"]))
        if op == "write":
            c.update(new=_log(rng, 1, 8192), past=rng.choice([0, _log(rng, 1, 8192)]),
                     dtype=rng.choice(["bf16", "f16", "f32"]))
            if c["batch"] * c["new"] * c["kv_heads"] * c["dim"] * (4 if c["dtype"] == "f32" else 2) > 5 * 8192 * 8 * 128:
                continue
        elif op == "read":
            c.update(length=_log(rng, 1, 16384), dtype=rng.choice(["bf16", "f16", "f32"]))
            if c["batch"] * c["length"] * c["kv_heads"] * c["dim"] * (4 if c["dtype"] == "f32" else 2) > 18 * 8192 * 8 * 128:
                continue
        else:
            c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
            c.update(new=rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 2048)]), length=_log(rng, 1, 131072),
                     dtype=rng.choice(["bf16", "f16"]), causal=rng.random() < 0.8,
                     window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
            if c["heads"] > 64 or c["new"] > c["length"] or not c["causal"] and c["window"]:
                continue
            if c["batch"] * c["length"] * c["kv_heads"] * c["dim"] > 34 * 16384 * 8 * 128:
                continue
            if c["batch"] * c["new"] * c["heads"] * c["length"] * c["dim"] > 2 * 2048 * 32 * 9216 * 128:
                continue
        return c


def _spread(n, top, ragged, least):
    """The lengths of n sequences: all `top`, or spread from about an eighth of it to all of it, the first the longest."""
    if not ragged:
        return [top] * n
    return [max(least, min(top, int(round(top * (1.0 - 0.875 * ((i * 0.6180339887498949) % 1.0)))))) for i in range(n)]


def _lengths(case):
    """(tokens before, new tokens) of each sequence; a ragged batch of four or more has one without new tokens."""
    n = case["batch"]
    if case["op"] == "write":
        new = _spread(n, case["new"], case["ragged"], 1)
        past = _spread(n, case["past"], case["ragged"], 0)
    elif case["op"] == "read":
        return [0] * n, _spread(n, case["length"], case["ragged"], 1)
    else:
        total = _spread(n, case["length"], case["ragged"], 1)
        new = [min(a, b) for a, b in zip(_spread(n, case["new"], case["ragged"], 1), total)]
        past = [a - b for a, b in zip(total, new)]
    if case["ragged"] and n >= 4:
        past[n - 1], new[n - 1] = past[n - 1] + new[n - 1], 0
    return past, new


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    got = [0]
    for c in counts:
        got.append(got[-1] + c)
    return got


def _fill(g, pages, heads, page, dim, codes):
    """Codes and scales as quantised activations leave them: the largest of a page near the top of the range."""
    kind, top = _CODES[codes]
    x = torch.randn((pages, heads, page, dim), generator=g, device="cuda", dtype=torch.float32 if codes == "e4m3" else torch.float16)
    q = x.mul_(top / 4.0).clamp_(-top, top)
    q = (q.round_() if codes == "int8" else q).to(kind)
    # a head's own size, and a page's around it
    size = torch.rand((1, heads), generator=g, device="cuda") + 0.5
    scale = size * (4.0 / top) * (0.75 + 0.5 * torch.rand((pages, heads), generator=g, device="cuda"))
    return q, scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    past, new = _lengths(case)
    page, dim, hk = case["page"], case["dim"], case["kv_heads"]
    total = [a + b for a, b in zip(past, new)]
    width = max(1, max(-(-t // page) for t in total))
    used = sum(-(-t // page) for t in total)
    pool = used + 2  # the last page belongs to nobody
    kq, ks = _fill(g, pool, hk, page, dim, case["codes"])
    vq, vs = _fill(g, pool, hk, page, dim, case["codes"])
    ks[-1], vs[-1] = 1.0, 1.0
    table = torch.zeros((case["batch"], width), dtype=torch.int32, device="cuda")
    order = torch.randperm(used, generator=g, device="cuda", dtype=torch.int32)
    at = 0
    for b, t in enumerate(total):
        k = -(-t // page)
        table[b, :k] = order[at:at + k]
        at += k
    s = dict(case=case, k=kq, v=vq, k_scale=ks, v_scale=vs, table=table)
    if case["op"] == "write":
        kind = _TYPES[case["dtype"]]
        t = sum(new)
        # k and v as the fused projection leaves them: columns of one row
        qkv = torch.randn((t, 2 * hk * dim), generator=g, device="cuda")
        qkv = (qkv * (0.5 + torch.rand((t, 1), generator=g, device="cuda"))).to(kind)
        first = [a // page * page for a in past]
        back = [a + b - f if b else 0 for a, b, f in zip(past, new, first)]
        s.update(new_k=qkv[:, :hk * dim].unflatten(1, (hk, dim)), new_v=qkv[:, hk * dim:].unflatten(1, (hk, dim)),
                 past=_i32(past), starts=_i32(_starts(new)), first=_i32(first), back=_i32(_starts(back)),
                 n_back=sum(back), most=max(-(-b // page) for b in back))
    elif case["op"] == "read":
        s.update(starts=_i32(_starts(new)), n=sum(new))
    else:
        q = torch.randn((sum(new), case["heads"], dim), generator=g, device="cuda").to(_TYPES[case["dtype"]])
        s.update(q=q, lengths=_i32(total), starts=_i32(_starts(new)) if case["ragged"] else None, most=max(new))
    if "h3-rs_b200" not in sys.path:
        sys.path.insert(0, "h3-rs_b200")
    return s


# ------------------------------------------------------------------------------------------------ the library's calls
def _run_own(s):
    from h3q import kvcache
    case = s["case"]
    cache = kvcache.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["op"] == "write":
        kvcache.write(cache, s["new_k"], s["new_v"], s["table"], s["past"], s["starts"])
        k, v = kvcache.read(cache, s["table"], s["back"], s["n_back"], s["new_k"].dtype, s["first"])
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if case["op"] == "read":
        k, v = kvcache.read(cache, s["table"], s["starts"], s["n"], _TYPES[case["dtype"]])
        return {"k": k, "v": v}
    out, lse = kvcache.attention(s["q"], cache, s["table"], s["lengths"], s["starts"], causal=case["causal"],
                                 window=case["window"], return_lse=True, max_new=s["most"])
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------------------ the plain form
def _plain_put(codes, scale, x, s, page, top):
    """x [t, heads, dim] goes into the pages it belongs to, in place."""
    past, starts, table, most = s["past"].long(), s["starts"].long(), s["table"].long(), s["most"]
    batch, t = past.shape[0], x.shape[0]
    dev = x.device
    at = torch.arange(t, device=dev)
    seq = torch.searchsorted(starts[1:], at, right=True)
    off = past % page
    slot = off[seq] + at - starts[seq]  # place in the span of pages that the sequence's new tokens touch
    heads, dim = x.shape[1:]
    span = torch.zeros((batch, most * page, heads, dim), device=dev)
    span[seq, slot] = x.float()
    span = span.unflatten(1, (most, page)).transpose(2, 3)  # [batch, most, heads, page, dim]
    place = torch.arange(most * page, device=dev)
    new = starts[1:] - starts[:-1]
    fresh = ((place >= off[:, None]) & (place < (off + new)[:, None])).unflatten(1, (most, page))
    nth = (past // page)[:, None] + torch.arange(most, device=dev)
    hit = fresh.any(-1)
    nobody = codes.shape[0] - 1
    ids = torch.where(hit, torch.gather(table, 1, nth.clamp(max=table.shape[1] - 1)), nobody)
    held = (nth * page < past[:, None])[..., None]  # the page holds older tokens
    old = torch.where(held, scale[ids], 0.0)  # [batch, most, heads]
    size = (span.abs() * fresh[:, :, None, :, None]).amax((-1, -2))
    now = torch.maximum(old, (size / top).clamp_min(_FLOOR))
    q = span * (1.0 / now)[..., None, None]
    kept = codes[ids].float()
    again = kept * (old / now)[..., None, None]
    y = torch.where(fresh[:, :, None, :, None], q, torch.where((now > old)[..., None, None], again, kept)).clamp(-top, top)
    y = torch.where(torch.isnan(y), 0.0, y)
    codes[ids] = (y.round() if codes.dtype == torch.int8 else y).to(codes.dtype)
    scale[ids] = now


def _plain_take(codes, scale, table, starts, n, first, kind):
    page = codes.shape[2]
    starts = starts.long()
    at = torch.arange(n, device=codes.device)
    seq = torch.searchsorted(starts[1:], at, right=True)
    pos = at - starts[seq]
    if first is not None:
        pos = pos + first.long()[seq]
    ids = table.long()[seq, pos // page]
    return (codes[ids, :, pos % page].float() * scale[ids][..., None]).to(kind)


def _plain_attention(s):
    case, page, dim = s["case"], s["case"]["page"], s["case"]["dim"]
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].long()
    batch, hk, heads = table.shape[0], case["kv_heads"], case["heads"]
    per, dev = heads // hk, q.device
    t = q.shape[0]
    starts = torch.arange(batch + 1, device=dev) * (t // batch) if s["starts"] is None else s["starts"].long()
    at = torch.arange(t, device=dev)
    seq = torch.searchsorted(starts[1:], at, right=True)
    nth = at - starts[seq]
    most = s["most"]
    new = starts[1:] - starts[:-1]

    def dense(codes, scale):
        x = codes[table].float() * scale[table][..., None, None]  # [batch, pages, hk, page, dim]
        return x.transpose(1, 2).reshape(batch, hk, -1, dim)

    k, v = dense(s["k"], s["k_scale"]), dense(s["v"], s["v_scale"])
    rows = torch.zeros((batch, most, heads, dim), device=dev)
    rows[seq, nth] = q.float()
    rows = rows.reshape(batch, most, hk, per, dim).permute(0, 2, 3, 1, 4).reshape(batch, hk, per * most, dim)
    score = torch.matmul(rows, k.transpose(-1, -2)).mul_(dim ** -0.5)
    del k
    pos = (lengths - new)[:, None] + torch.arange(most, device=dev)
    key = torch.arange(score.shape[-1], device=dev)
    seen = (key < lengths[:, None])[:, None, :].expand(batch, most, -1)
    if case["causal"]:
        seen = seen & (key <= pos[..., None])
    if case["window"]:
        seen = seen & (key > pos[..., None] - case["window"])
    score = score.unflatten(2, (per, most)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    some = top > -math.inf
    top = torch.where(some, top, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (per, most)) / torch.where(some, total, 1.0)
    lse = (top + total.log())[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[seq, nth].to(q.dtype)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).reshape(batch, most, heads)[seq, nth].contiguous()}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "write":
        top = _CODES[case["codes"]][1]
        _plain_put(s["k"], s["k_scale"], s["new_k"], s, case["page"], top)
        _plain_put(s["v"], s["v_scale"], s["new_v"], s, case["page"], top)
        kind = _TYPES[case["dtype"]]
        take = [_plain_take(s[x], s[x + "_scale"], s["table"], s["back"], s["n_back"], s["first"], kind) for x in "kv"]
        nobody = s["k"].shape[0] - 1
        s["k_scale"][nobody] = 1.0
        s["v_scale"][nobody] = 1.0
        return {"k": take[0], "v": take[1], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if case["op"] == "read":
        kind = _TYPES[case["dtype"]]
        return {x: _plain_take(s[x], s[x + "_scale"], s["table"], s["starts"], s["n"], None, kind) for x in "kv"}
    return _plain_attention(s)


# ------------------------------------------------------------------------------------------------ work and 64 bits
def work(case):
    past, new = _lengths(case)
    page, dim, hk = case["page"], case["dim"], case["kv_heads"]
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]

    def pages(a, b):  # pages that tokens a..b-1 touch
        return -(-b // page) - a // page if b > a else 0

    if case["op"] == "write":
        t = sum(new)
        back = sum(a + b - a // page * page for a, b in zip(past, new) if b)
        scales = sum(pages(a, a + b) for a, b in zip(past, new)) * hk * 4
        return {"bytes": 2 * (t * hk * dim * (size + 1) + back * hk * dim * size + (back - t) * hk * dim + 2 * scales),
                "flops": 4 * t * hk * dim}
    if case["op"] == "read":
        t = sum(new)
        return {"bytes": 2 * (t * hk * dim * (size + 1) + sum(pages(0, b) for b in new) * hk * 4), "flops": 2 * t * hk * dim}
    pairs = keys = scales = 0
    for a, b in zip(past, new):
        total, w = a + b, case["window"]
        low = max(0, a + 1 - w) if w else 0
        if not b:
            continue
        keys += total - low
        scales += pages(low, total)
        if not case["causal"]:
            pairs += b * total
        elif not w:
            pairs += b * a + b * (b + 1) // 2
        else:
            pairs += sum(min(w, a + 1 + i) for i in range(b))
    rows = sum(new) * case["heads"]
    return {"bytes": 2 * (keys * hk * dim + scales * hk * 4) + rows * (2 * dim * size + 4), "flops": 4 * pairs * case["heads"] * dim}


def exact(case, seed):
    past, new = _lengths(case)
    s = prepare(case, seed)
    page, dim, hk = case["page"], case["dim"], case["kv_heads"]
    table = s["table"].tolist()
    if case["op"] == "attention":
        pairs = sum(b * (a + b) for a, b in zip(past, new)) * case["heads"] * dim
        if pairs > 3e12:
            return None
        outs, lses, at = [], [], 0
        per = case["heads"] // hk
        for b, (a, n) in enumerate(zip(past, new)):
            if not n:
                continue
            ids = torch.tensor(table[b][:-(-(a + n) // page)], device="cuda", dtype=torch.long)
            low = max(0, a + 1 - case["window"]) if case["window"] else 0
            o = torch.empty((n, case["heads"], dim), dtype=torch.float64, device="cuda")
            z = torch.empty((n, case["heads"]), dtype=torch.float64, device="cuda")
            j = torch.arange(low, a + n, device="cuda")
            for h in range(hk):
                k = (s["k"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[low:a + n]
                v = (s["v"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[low:a + n]
                for i in range(0, n, 256):
                    m = min(256, n - i)
                    x = s["q"][at + i:at + i + m, h * per:(h + 1) * per].double()
                    w = torch.einsum("mpd,kd->mpk", x, k) / math.sqrt(dim)
                    where = a + i + torch.arange(m, device="cuda")[:, None]
                    hide = torch.zeros((m, j.numel()), dtype=torch.bool, device="cuda")
                    if case["causal"]:
                        hide |= j > where
                    if case["window"]:
                        hide |= j <= where - case["window"]
                    w = w.masked_fill(hide[:, None], -math.inf)
                    z[i:i + m, h * per:(h + 1) * per] = torch.logsumexp(w, -1)
                    o[i:i + m, h * per:(h + 1) * per] = torch.softmax(w, -1) @ v
            outs.append(o)
            lses.append(z)
            at += n
        return {"out": torch.cat(outs), "lse": torch.cat(lses)}
    found = {}
    for x in "kv":
        codes, scale = s[x].double(), s[x + "_scale"].double()
        top = _CODES[case["codes"]][1]
        rows, at = [], 0
        for b, (a, n) in enumerate(zip(past, new)):
            if not n:
                continue
            begin = a // page if case["op"] == "write" else 0
            for i in range(begin, -(-(a + n) // page)):
                p, lo, hi = table[b][i], max(a - i * page, 0), min(a + n - i * page, page)
                if case["op"] == "write":
                    y = s["new_" + x][at + i * page + lo - a:at + i * page + hi - a].double().transpose(0, 1)
                    old = scale[p] if lo else torch.zeros_like(scale[p])
                    now = torch.maximum(old, (y.abs().amax((1, 2)) / top).clamp_min(_FLOOR))
                    kept = codes[p, :, :lo] * (old / now)[:, None, None]
                    both = torch.cat([kept, y / now[:, None, None]], 1)
                    both = both.round() if case["codes"] == "int8" else both.float().to(torch.float8_e4m3fn).double()
                    scale[p] = now
                    rows.append((both * now[:, None, None]).transpose(0, 1))
                else:
                    rows.append((codes[p, :, :hi] * scale[p][:, None, None]).transpose(0, 1))
            at += n
        found[x] = torch.cat(rows)
        if case["op"] == "write":
            found[x + "_scale"] = scale
    return found
