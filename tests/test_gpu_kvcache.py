"""GPU tests of the 8-bit paged key / value cache (h3q.kvcache) against its definition in 64 bits.

Written codes: s = max(old, amax / top, 1e-30) and code = round(x / s) in 64 bits.  The kernels form s and x * (1 / s) in
f32 (relative errors of a few 2^-24), so a scale is within 4 * 2^-24 of the 64-bit one, and a stored value within half
a step of x, widened by the f32 error of the quotient (at most top * 2^-21 steps); a requantised older value moves by
half a step more.

Attention: with A = sum_j p_j |v_j|, the f16 weights cost at most 2^-11 A, their subnormals 2^-25 max_j(p_j vs_j)
sum_j |vcode_j|, scores and sums in f32 2^-16 A (a score error e moves a weight by e; 2^-17 covers D = 128 products of
the sizes used here), the output's rounding 2^-8 (bf16, 8 significant bits) or 2^-11 (f16) of the value.  lse is held to 2^-17 (1 + max |score|).
"""
import math

import pytest
import torch

import h3q
from h3q import kvcache

pytestmark = pytest.mark.gpu

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _starts(n):
    s = [0]
    for c in n:
        s.append(s[-1] + c)
    return s


def make_cache(dev, codes, hk, page, dim, totals, seed, spare=3):
    """A filled cache whose unused tokens and pages hold the worst bits, its page table and the dense 64-bit k, v, vcode, vs."""
    g = _gen(seed, dev)
    need = [-(-t // page) for t in totals]
    pages = sum(need) + spare
    width = max(need + [1]) + 1
    top = TOP[codes]
    raw = [(torch.randn((pages, hk, page, dim), generator=g, device=dev) * top / 4).clamp(-top, top) for _ in range(2)]
    k, v = [(x.round() if codes == torch.int8 else x).to(codes) for x in raw]
    ks, vs = [0.05 * (0.2 + torch.rand((pages, hk), generator=g, device=dev)) * 127 / top for _ in range(2)]
    perm = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.full((len(totals), width), -7, dtype=torch.int32)
    bad = 0x7f if codes == torch.float8_e4m3fn else 0x80
    at = 0
    used = set()
    for b, t in enumerate(totals):
        for i in range(need[b]):
            p = perm[at]
            at += 1
            used.add(p)
            table[b, i] = p
            if (i + 1) * page > t:
                for c in (k, v):
                    c.view(torch.uint8)[p, :, t - i * page:] = bad
    for p in range(pages):
        if p not in used:
            for c in (k, v):
                c.view(torch.uint8)[p] = bad
            ks[p] = float("nan")
            vs[p] = float("nan")
    return kvcache.KVCache(k, v, ks.contiguous(), vs.contiguous()), table.to(dev)


def dense(cache, table, b, t):
    """(k, v, vcode, vs) of the first t tokens of sequence b, [hk, t, dim] (vs [hk, t]) in 64 bits; a missing page: None rows."""
    page = cache.k.shape[2]
    ids = table[b, :-(-t // page)].long()
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = c[ids].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :t]
        f = s[ids].double().t().repeat_interleave(page, 1)[:, :t]
        out += [x, f]
    return out[0] * out[1][..., None], out[2] * out[3][..., None], out[2], out[3]


def check_attention(q, cache, table, totals, news, got, lse, scale, causal, window, gone=None):
    hk, dim = cache.k.shape[1], cache.k.shape[3]
    heads = q.shape[1]
    per = heads // hk
    at = 0
    u = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    for b, (t, n) in enumerate(zip(totals, news)):
        if n == 0:
            continue
        pos = t - n + torch.arange(n, device=q.device)[:, None]
        j = torch.arange(t, device=q.device)
        seen = torch.ones((n, t), dtype=torch.bool, device=q.device)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        if gone is not None:
            for lo, hi in gone.get(b, []):
                seen[:, lo:hi] = False
        if t:
            k, v, vc, vs = dense(cache, table, b, t)
            if gone is not None:
                for lo, hi in gone.get(b, []):
                    for x in (k, v, vc, vs):
                        x[:, lo:hi] = 0
        for h in range(heads):
            x = q[at:at + n, h].double()
            o, z = got[at:at + n, h].double(), lse[at:at + n, h].double()
            none = ~seen.any(1)
            assert (o[none] == 0).all() and (z[none] == -math.inf).all()
            if t == 0 or none.all():
                continue
            s = (x @ k[h // per].t()) * scale
            s = s.masked_fill(~seen, -math.inf)
            want_z = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1).nan_to_num(0.0)
            want = p @ v[h // per]
            a = p @ v[h // per].abs()
            sub = (p * vs[h // per]).amax(1, keepdim=True) * (seen.double() @ vc[h // per].abs())
            tol = (2.0 ** -11 + 2.0 ** -16) * a + 2.0 ** -25 * sub + u * want.abs() + 1e-37
            some = ~none
            assert torch.isfinite(o).all()
            worst = ((o - want).abs() / tol)[some].max().item()
            assert worst <= 1.0, (b, h, worst)
            size = (s.masked_fill(~seen, 0).abs().amax(1) + 1)[some]
            assert ((z - want_z)[some].abs() <= 2.0 ** -17 * size).all(), (b, h)
        at += n


def run_attention(dev, codes, kind, hk, per, dim, page, totals, news, causal=True, window=0, seed=0, starts=True, strided=False,
                  max_new=0, scale=None):
    cache, table = make_cache(dev, codes, hk, page, dim, totals, seed)
    g = _gen(seed + 1, dev)
    heads = hk * per
    rows = torch.randn((sum(news), 3 * heads, dim), generator=g, device=dev).to(kind)
    q = rows[:, heads:2 * heads] if strided else rows[:, :heads].contiguous()
    got, lse = kvcache.attention(q, cache, table, _i32(totals, dev), _i32(_starts(news), dev) if starts else None,
                                 scale=scale, causal=causal, window=window, return_lse=True, max_new=max_new)
    check_attention(q, cache, table, totals, news, got, lse, dim ** -0.5 if scale is None else scale, causal, window)
    again = kvcache.attention(q, cache, table, _i32(totals, dev), _i32(_starts(news), dev) if starts else None, scale=scale,
                              causal=causal, window=window, max_new=max_new)
    assert torch.equal(got, again)
    assert h3q.device_status() == 0


I8, E4 = torch.int8, torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16

# (codes, kind, kv heads, query heads to a kv head, dim, page, totals, news, causal, window)
ATTENTION = [
    (I8, BF, 8, 8, 128, 64, [1], [1], True, 0),
    (I8, BF, 2, 1, 128, 16, [17], [1], True, 0),
    (E4, HF, 3, 4, 64, 32, [0, 5, 128, 129, 700], [0, 1, 1, 1, 1], True, 0),
    (E4, BF, 1, 5, 128, 128, [127, 128, 1000], [5, 2, 3], True, 0),          # 25 rows
    (I8, HF, 2, 16, 64, 16, [333, 1, 16], [1, 1, 1], True, 0),
    (I8, BF, 2, 2, 128, 64, [4097, 2, 700], [1, 1, 1], True, 300),           # a window
    (E4, HF, 1, 8, 64, 64, [900, 64], [4, 4], True, 17),
    (I8, BF, 2, 4, 128, 32, [515, 3], [3, 3], False, 0),                     # not causal
    (E4, BF, 2, 3, 128, 64, [2, 0, 40], [7, 5, 40], True, 0),                # rows before the first key: empty
    (I8, BF, 1, 8, 128, 64, [300], [300], True, 0),                          # a prompt
    (E4, HF, 2, 2, 64, 16, [1000, 257, 130], [513, 257, 1], True, 0),
    (I8, HF, 1, 3, 128, 128, [777, 50, 1300], [129, 50, 301], False, 0),
    (E4, BF, 2, 5, 128, 32, [1500, 800], [400, 77], True, 130),
    (I8, BF, 1, 1, 64, 64, [2048, 0, 600], [1025, 0, 600], True, 0),
    (I8, BF, 3, 1, 128, 64, [5, 261], [5, 133], True, 1),                    # every row sees itself alone
]


@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(cuda, case):
    codes, kind, hk, per, dim, page, totals, news, causal, window = ATTENTION[case]
    run_attention(cuda, codes, kind, hk, per, dim, page, totals, news, causal, window, seed=100 + case,
                  max_new=max(news) if case % 2 else 0, strided=case % 3 == 1)


@pytest.mark.parametrize("new", [1, 9, 200])
def test_attention_of_rows_that_are_not_aligned(cuda, new):
    """q begins 2 bytes behind a 16-byte boundary and its rows lie an odd number of elements apart."""
    totals = [new + 77]
    cache, table = make_cache(cuda, I8, 2, 32, 128, totals, 12)
    flat = torch.randn(1 + new * (4 * 128 + 3), generator=_gen(1, cuda), device=cuda).to(BF)
    q = flat[1:].view(new, 4 * 128 + 3)[:, :512].unflatten(1, (4, 128))
    n = _i32(totals, cuda)
    assert q.data_ptr() % 16 == 2 and (new == 1 or q.stride(0) == 515)
    assert torch.equal(kvcache.attention(q, cache, table, n), kvcache.attention(q.contiguous(), cache, table, n))


@pytest.mark.parametrize("new", [1, 3, 40])
def test_attention_without_starts(cuda, new):
    run_attention(cuda, I8, BF, 2, 4, 128, 64, [100, 70, 333], [new] * 3, seed=new, starts=False)


@pytest.mark.parametrize("new", [1, 300])
def test_attention_many_sequences(cuda, new):
    """More sequences than a CTA has threads, most of them short, some without tokens."""
    totals = [(7 * i) % 90 + (400 if i % 50 == 0 else 0) for i in range(700)]
    news = [(0 if t == 0 or i % 11 == 0 else min(t, new if i % 50 == 0 else 1)) for i, t in enumerate(totals)]
    run_attention(cuda, I8, HF, 1, 2, 64, 16, totals, news, seed=3, max_new=max(news))


@pytest.mark.parametrize("new", [1, 5, 70])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_one_head_split_over_every_worker(cuda, new, dim):
    run_attention(cuda, E4, BF, 1, 5, dim, 128, [50001], [new], seed=29)


@pytest.mark.parametrize("new", [1, 4])
def test_attention_of_short_sequences_beside_long_ones(cuda, new):
    totals = [new + 37 * i % 211 for i in range(60)] + [9001] + [new] * 5
    run_attention(cuda, I8, HF, 2, 8, 128, 16, totals, [new] * len(totals), seed=31)


def test_attention_scores_of_any_size(cuda):
    """Scores up to several hundred: one key takes all the weight, and the running maximum moves often."""
    run_attention(cuda, I8, BF, 1, 4, 128, 64, [1500], [3], seed=5, scale=4.0)
    run_attention(cuda, E4, HF, 1, 4, 64, 32, [600], [200], seed=6, scale=-3.0)
    run_attention(cuda, I8, BF, 1, 4, 128, 64, [700], [2], seed=7, scale=0.0)


@pytest.mark.parametrize("new", [2, 150])
def test_attention_scales_of_pages_far_apart(cuda, new):
    """A page of zeros at the smallest scale takes weight; a page of large values takes next to none."""
    totals, news = [400], [new]
    cache, table = make_cache(cuda, I8, 1, 32, 128, totals, 9)
    ids = table[0].tolist()
    cache.v_scale[ids[0]] = 1e-30
    cache.v.view(torch.uint8)[ids[0]] = 0
    cache.v_scale[ids[2]] = 1e4
    cache.k_scale[ids[2]] = 1e-30
    cache.v_scale[ids[4]] = 1e-6
    q = torch.randn((new, 4, 128), generator=_gen(1, cuda), device=cuda).to(BF)
    got, lse = kvcache.attention(q, cache, table, _i32(totals, cuda), return_lse=True)
    check_attention(q, cache, table, totals, news, got, lse, 128 ** -0.5, True, 0)


@pytest.mark.parametrize("kind,size", [(BF, 1e30), (BF, 1e-30), (HF, 1e-5), (HF, 3e4)])
def test_attention_queries_of_any_size(cuda, kind, size):
    """Rows far from 1 (bf16 beyond the range of f16) with a scale that brings the scores back."""
    totals, news = [300, 20], [1, 20]
    cache, table = make_cache(cuda, I8, 2, 64, 128, totals, 4)
    q = (torch.randn((21, 4, 128), generator=_gen(2, cuda), device=cuda).clamp(-2, 2) * size).to(kind)
    got, lse = kvcache.attention(q, cache, table, _i32(totals, cuda), _i32(_starts(news), cuda), scale=0.1 / size,
                                 return_lse=True)
    check_attention(q, cache, table, totals, news, got, lse, float(torch.tensor(0.1 / size, dtype=torch.float32)), True, 0)


@pytest.mark.parametrize("news", [[1, 2], [90, 200]])
def test_attention_without_some_pages(cuda, news):
    """A table entry that names no page hides its tokens; a row whose every key is hidden gives zeros."""
    totals = [200, 400]
    cache, table = make_cache(cuda, E4, 2, 64, 64, totals, 8)
    table[0, 1] = -1
    table[1, 0] = 1 << 30
    table[1, 3] = -5
    q = torch.randn((sum(news), 4, 64), generator=_gen(3, cuda), device=cuda).to(HF)
    got, lse = kvcache.attention(q, cache, table, _i32(totals, cuda), _i32(_starts(news), cuda), return_lse=True)
    fixed = table.clone()
    fixed[fixed < 0] = 0
    fixed[fixed >= cache.k.shape[0]] = 0
    check_attention(q, cache, fixed, totals, news, got, lse, 0.125, True, 0, gone={0: [(64, 128)], 1: [(0, 64), (192, 256)]})
    table.fill_(-1)
    got, lse = kvcache.attention(q, cache, table, _i32(totals, cuda), _i32(_starts(news), cuda), return_lse=True)
    assert (got == 0).all() and (lse == -math.inf).all()


def test_attention_of_more_tokens_than_allowed_for(cuda):
    """A sequence that breaks the caller's max_new gets NaN, the others their results; a bound that is not tight changes nothing."""
    totals, news = [50, 80, 30], [1, 40, 2]
    cache, table = make_cache(cuda, I8, 2, 16, 64, totals, 6)
    q = torch.randn((43, 4, 64), generator=_gen(5, cuda), device=cuda).to(BF)
    args = (q, cache, table, _i32(totals, cuda), _i32(_starts(news), cuda))
    good, lse = kvcache.attention(*args, max_new=40, return_lse=True)
    check_attention(q, cache, table, totals, news, good, lse, 0.125, True, 0)
    assert torch.equal(good, kvcache.attention(*args)) and torch.equal(good, kvcache.attention(*args, max_new=43))
    got, lse = kvcache.attention(*args, max_new=2, return_lse=True)
    assert torch.isnan(got[1:41]).all() and torch.isnan(lse[1:41]).all()
    check_attention(q[:1], cache, table, [50], [1], got[:1], lse[:1], 0.125, True, 0)
    check_attention(q[41:], cache, table[2:], [30], [2], got[41:], lse[41:], 0.125, True, 0)


def test_attention_beyond_32_bit_offsets(cuda):
    """Pages whose codes lie more than 2^32 bytes into the pool."""
    page, hk, dim = 64, 8, 128
    pages = (1 << 32) // (page * hk * dim) + 64
    cache = kvcache.KVCache.empty(pages, hk, page, dim, device=cuda)
    small, st = make_cache(cuda, I8, hk, page, dim, [500], 11)
    table = torch.full((1, 9), -1, dtype=torch.int32, device=cuda)
    for i in range(8):
        src, dst = int(st[0, i]), pages - 1 - 3 * i
        table[0, i] = dst
        for a, b in ((cache.k, small.k), (cache.v, small.v), (cache.k_scale, small.k_scale), (cache.v_scale, small.v_scale)):
            a[dst] = b[src]
    for new in (1, 60):
        q = torch.randn((new, 16, dim), generator=_gen(new, cuda), device=cuda).to(BF)
        n = _i32([500], cuda)
        assert torch.equal(kvcache.attention(q, cache, table, n), kvcache.attention(q, small, st, n))
    starts = _i32([0, 500], cuda)
    for a, b in zip(kvcache.read(cache, table, starts, 500), kvcache.read(small, st, starts, 500)):
        assert torch.equal(a, b)
    x = torch.randn((500, hk, dim), generator=_gen(7, cuda), device=cuda).to(BF)
    zero = _i32([0], cuda)
    kvcache.write(cache, x, x, table, zero)
    kvcache.write(small, x, x, st, zero)
    for a, b in zip(kvcache.read(cache, table, starts, 500), kvcache.read(small, st, starts, 500)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------- write and read

def _steps(codes, code):
    """The spacing of the code type around `code` (at least that of its smallest numbers)."""
    if codes == I8:
        return torch.ones_like(code)
    return 2.0 ** (torch.floor(torch.log2(code.abs().clamp_min(2.0 ** -6))) - 3)


# (codes, kind, kv heads, dim, page, pasts, news)
WRITE = [
    (I8, BF, 8, 128, 64, [0], [1]),
    (I8, BF, 2, 128, 64, [63, 64, 65, 0, 7], [1, 1, 1, 1, 0]),
    (E4, HF, 3, 64, 16, [0, 5, 15, 31], [1, 0, 2, 1]),
    (E4, BF, 1, 128, 128, [100, 0, 256], [300, 129, 1]),
    (I8, torch.float32, 2, 64, 32, [1, 0, 33], [31, 100, 64]),
    (I8, HF, 40, 128, 16, [3], [77]),
    (E4, torch.float32, 1, 64, 64, [0, 0, 10], [64, 1, 500]),
    (I8, BF, 1, 128, 128, [1, 300], [1000, 3]),
]


@pytest.mark.parametrize("case", range(len(WRITE)))
@pytest.mark.parametrize("loud", [0.01, 30.0])
def test_write_and_read(cuda, case, loud):
    """Old pages quieter and louder than the new rows: scales that stay and scales that grow."""
    codes, kind, hk, dim, page, pasts, news = WRITE[case]
    totals = [a + n for a, n in zip(pasts, news)]
    cache, table = make_cache(cuda, codes, hk, page, dim, totals, 20 + case)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    t = sum(news)
    g = _gen(case, cuda)
    wide = (torch.randn((t, 3 * hk, dim), generator=g, device=cuda) * loud).to(kind)
    if case % 2:  # a view whose rows are not aligned to 16 bytes
        flat = torch.zeros(wide.numel() + 1, dtype=kind, device=cuda)
        flat[1:] = wide.flatten()
        wide = flat[1:].view_as(wide)
    k, v = wide[:, hk:2 * hk], wide[:, 2 * hk:]
    kvcache.write(cache, k, v, table, _i32(pasts, cuda), _i32(_starts(news), cuda))
    starts = _starts(totals)
    dense_k, dense_v = kvcache.read(cache, table, _i32(starts, cuda), starts[-1], torch.float32)
    top = TOP[codes]
    touched = set()
    for which, (x, back, c0, s0, s1) in enumerate(((k, dense_k, before[0], before[2], cache.k_scale),
                                                  (v, dense_v, before[1], before[3], cache.v_scale))):
        for b, (past, n) in enumerate(zip(pasts, news)):
            for i in range(past // page, -(-(past + n) // page) if n else 0):
                p = int(table[b, i])
                touched.add(p)
                lo, hi = max(past - i * page, 0), min(past + n - i * page, page)
                at = _starts(news)[b] + i * page + lo - past
                new = x[at:at + hi - lo].double().transpose(0, 1)
                old = s0[p].double() if lo else torch.zeros(hk, dtype=torch.float64, device=cuda)
                want = torch.maximum(old, (new.abs().amax((1, 2)) / top).clamp_min(1e-30))
                s = s1[p].double()
                assert ((s - want).abs() <= 4 * 2.0 ** -24 * want).all()
                rows = back[starts[b] + i * page:starts[b] + i * page + hi].double().transpose(0, 1)
                code = rows / s[:, None, None]
                step = _steps(codes, new / s[:, None, None]) * s[:, None, None]
                assert ((rows[:, lo:] - new).abs() <= step * (0.5 + top * 2.0 ** -21)).all()
                assert (code.abs() <= top * (1 + 1e-6)).all()
                if lo:
                    kept = c0[p, :, :lo].double() * s0[p].double()[:, None, None]
                    step = _steps(codes, kept / s[:, None, None]) * s[:, None, None]
                    grew = (s > old)[:, None, None]
                    bound = torch.where(grew, step * (0.5 + top * 2.0 ** -21), 2.0 ** -23 * kept.abs())
                    assert ((rows[:, :lo] - kept).abs() <= bound).all()
    # nothing else changed
    rest = [p for p in range(cache.k.shape[0]) if p not in touched]
    for now, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        now, was = now[rest].view(torch.uint8 if now.dtype != torch.float32 else torch.int32), was[rest]
        assert torch.equal(now, was.view(torch.uint8 if was.dtype != torch.float32 else torch.int32))


@pytest.mark.parametrize("codes", [I8, E4])
def test_tokens_one_by_one_fill_pages_as_a_chunk_does(cuda, codes):
    """The last scale of a page is the same whichever way its tokens came, and codes are within a rounding for each growth."""
    hk, dim, page, n = 2, 64, 16, 37
    x = torch.randn((n, hk, dim), generator=_gen(1, cuda), device=cuda).to(BF)
    table = _i32([[2, 0, 3]], cuda)
    one, many = [kvcache.KVCache.empty(4, hk, page, dim, codes, cuda) for _ in range(2)]
    kvcache.write(many, x, x, table, _i32([0], cuda))
    for i in range(n):
        kvcache.write(one, x[i:i + 1], x[i:i + 1], table, _i32([i], cuda))
    assert torch.equal(one.k_scale, many.k_scale) and torch.equal(one.v_scale, many.v_scale)
    starts = _i32([0, n], cuda)
    a, b = [kvcache.read(c, table, starts, n, torch.float32)[0] for c in (one, many)]
    top = TOP[codes]
    scale = many.k_scale[table[0].long()].repeat_interleave(page, 0)[:n][..., None]
    step = _steps(codes, (b / scale).double()).float() * scale
    assert ((a - b).abs() <= 6 * step).all()  # amax of a page grows a few times in 16 draws, each half a step, in two directions


@pytest.mark.parametrize("codes", [I8, E4])
@pytest.mark.parametrize("n", [1, 40])
def test_write_of_rows_that_are_not_finite(cuda, codes, n):
    """NaN is stored as 0 and an infinity as the largest code; neither sets the scale.  Rows of zeros leave the smallest scale."""
    hk, dim, page = 2, 64, 16
    x = torch.randn((n, hk, dim), generator=_gen(n, cuda), device=cuda)
    x[0, 0, 3] = float("nan")
    x[0, 0, 5] = float("inf")
    x[0, 0, 7] = -float("inf")
    x[:, 1] = 0
    cache = kvcache.KVCache.empty(3, hk, page, dim, codes, cuda)
    table = _i32([[1, 0, 2]], cuda)
    kvcache.write(cache, x, x, table, _i32([0], cuda))
    k, v = kvcache.read(cache, table, _i32([0, n], cuda), n, torch.float32)
    assert torch.equal(k, v)
    s = cache.k_scale[1, 0]
    clean = torch.where(torch.isfinite(x[:page, 0]), x[:page, 0], 0.0)
    assert abs(float(s) - float(clean.abs().max()) / TOP[codes]) <= 4 * 2.0 ** -24 * float(s)
    assert k[0, 0, 3] == 0 and k[0, 0, 5] == TOP[codes] * s and k[0, 0, 7] == -TOP[codes] * s
    assert (k[:, 1] == 0).all() and float(cache.k_scale[1, 1]) == pytest.approx(1e-30, rel=1e-6)


def test_places_outside_the_table(cuda):
    """Tokens before place 0 or behind the table's last page read as zeros and are dropped when written."""
    cache, table = make_cache(cuda, I8, 1, 16, 64, [32], 3, spare=0)  # one page more in the table, which names none
    starts = _i32([0, 60], cuda)
    k, _ = kvcache.read(cache, table, starts, 60, torch.float32, _i32([-10], cuda))
    all32, _ = kvcache.read(cache, table, _i32([0, 32], cuda), 32, torch.float32)
    assert (k[:10] == 0).all() and torch.equal(k[10:42], all32) and (k[42:] == 0).all()
    x = torch.ones((60, 1, 64), device=cuda)
    kvcache.write(cache, x, x, table, _i32([-10], cuda), starts)
    k, _ = kvcache.read(cache, table, _i32([0, 32], cuda), 32, torch.float32)
    assert ((k - 1).abs() <= 2.0 ** -22).all()


def test_read_spans(cuda):
    """Spans that begin inside a page, empty ones, and tokens of a page that is not there (zeros), in each type."""
    totals = [100, 0, 65, 300]
    cache, table = make_cache(cuda, I8, 3, 32, 64, totals, 2)
    table[3, 2] = -1
    first, n = [33, 0, 64, 1], [60, 0, 1, 299]
    starts = _starts(n)
    want = []
    for b in range(4):
        ids = table[b, :-(-totals[b] // 32)].long()
        x = cache.k[ids.clamp_min(0)].float() * cache.k_scale[ids.clamp_min(0)][..., None, None]
        x = torch.where((ids < 0)[:, None, None, None], 0.0, x).permute(0, 2, 1, 3).flatten(0, 1)
        want.append(x[first[b]:first[b] + n[b]])
    want = torch.cat(want)
    for kind in (torch.float32, HF, BF):
        k, v = kvcache.read(cache, table, _i32(starts, cuda), starts[-1], kind, _i32(first, cuda))
        assert torch.equal(k, want.to(kind))


def test_calls_follow_the_current_stream_and_replay_in_a_graph(cuda):
    """A decode step (write, then attend) captured once and replayed as the sequences grow."""
    hk, heads, dim, page, batch = 2, 8, 128, 16, 3
    eager, graph = [kvcache.KVCache.empty(20, hk, page, dim, device=cuda) for _ in range(2)]
    for c in (eager, graph):
        c.k.zero_()
        c.v.zero_()
    table = torch.arange(18, dtype=torch.int32, device=cuda).view(batch, 6)
    past = _i32([0, 14, 40], cuda)
    x = torch.randn((60, 2 * hk, dim), generator=_gen(1, cuda), device=cuda).to(BF)
    q = torch.randn((20, batch, heads, dim), generator=_gen(2, cuda), device=cuda).to(BF)
    for c in (eager, graph):
        kvcache.write(c, x[:54, :hk], x[:54, hk:], table, _i32([0, 0, 0], cuda), _i32([0, 0, 14, 54], cuda))
    step_x, step_q, step_past = x[:batch].clone(), q[0].clone(), past.clone()
    side = torch.cuda.Stream()

    def step(c):
        kvcache.write(c, step_x[:, :hk], step_x[:, hk:], table, step_past)
        return kvcache.attention(step_q, c, table, step_past + 1)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graph)  # writes the tokens that the first replay writes again
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(graph)
    torch.cuda.synchronize()
    for i in range(5):
        step_x.copy_(x[3 * i:3 * i + 3])
        step_q.copy_(q[i])
        step_past.copy_(past + i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(eager))


def test_empty_calls(cuda):
    cache, table = make_cache(cuda, I8, 2, 16, 64, [5, 3], 1)
    none = torch.empty((0, 2, 64), dtype=BF, device=cuda)
    zero = _i32([0, 0], cuda)
    starts = _i32([0, 0, 0], cuda)
    kvcache.write(cache, none, none, table, zero, starts)
    assert kvcache.read(cache, table, starts, 0)[0].shape == (0, 2, 64)
    assert kvcache.attention(none, cache, table, zero, starts).shape == (0, 2, 64)


def test_refusals(cuda):
    cache, table = make_cache(cuda, I8, 2, 16, 64, [5, 3], 1)
    q = torch.zeros((2, 4, 64), dtype=BF, device=cuda)
    n = _i32([5, 3], cuda)
    kv = q[:, :2]
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.transpose(1, 2)), dict(table=table.long()), dict(table=table[0]),
                dict(lengths=n.long()), dict(lengths=n[:1]), dict(starts=n), dict(window=-1), dict(window=4, causal=False),
                dict(scale=float("nan")), dict(q=torch.zeros((3, 4, 64), dtype=BF, device=cuda)), dict(table=table.cpu())):
        a = dict(q=q, table=table, lengths=n, starts=None, window=0, causal=True, scale=None) | bad
        with pytest.raises(h3q.H3QError):
            kvcache.attention(a["q"], cache, a["table"], a["lengths"], a["starts"], scale=a["scale"], causal=a["causal"],
                              window=a["window"])
    with pytest.raises(h3q.H3QError):
        kvcache.write(cache, kv, kv.float(), table, n)
    with pytest.raises(h3q.H3QError):
        kvcache.write(cache, kv.to(torch.int32), kv.to(torch.int32), table, n)
    with pytest.raises(h3q.H3QError):
        kvcache.write(cache, q, q, table, n)
    with pytest.raises(h3q.H3QError):
        kvcache.read(cache, table, n, 2)
    with pytest.raises(h3q.H3QError):
        kvcache.read(cache, table, _i32([0, 1, 2], cuda), 2, torch.int8)
    with pytest.raises(AttributeError):  # the checks were of the tensors that it holds
        cache.k = cache.k.clone()
    with pytest.raises(h3q.H3QError):
        kvcache.KVCache(cache.k, cache.v, cache.k_scale.double(), cache.v_scale)
    with pytest.raises(h3q.H3QError):
        kvcache.KVCache(cache.k, cache.v.view(torch.float8_e4m3fn), cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        kvcache.KVCache(cache.k.cpu(), cache.v, cache.k_scale, cache.v_scale)
    odd = kvcache.KVCache.empty(2, 2, 24, 64, device=cuda)
    with pytest.raises(h3q.H3QError) as e:
        kvcache.read(odd, table, _i32([0, 1, 2], cuda), 2)
    assert e.value.status == h3q.ERR_UNSUPPORTED
