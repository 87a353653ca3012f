"""GPU tests of the 8-bit paged key / value cache where attention and reads are easily wrong: values of pages far apart, a
key that takes nearly all the weight, scales that are no scales, queries that are not numbers, tables shorter than a
sequence, and rows that belong to no sequence.  Definition and tolerances are test_gpu_kvcache's unless stated.
"""
import math

import pytest
import torch

import h3q
from h3q import kvcache
from test_gpu_kvcache import BF, E4, HF, I8, _gen, _i32, _starts, check_attention, make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,per,total", [(1, 4, 400), (8, 4, 400), (200, 1, 400), (1, 5, 30000), (70, 5, 30000)])
@pytest.mark.parametrize("large", [1e12, 1e35])
@pytest.mark.parametrize("score", [0.0, 1.0])
def test_values_of_pages_far_apart(cuda, new, per, total, large, score):
    """Pages of zeros at the smallest scale beside pages of values up to 1e37: each key counts in the denominator as its score
    says, however small its values are beside others', and whichever worker or warp sees them."""
    cache, table = make_cache(cuda, I8, 1, 16, 64, [total], 41)
    ids = table[0, :-(-total // 16)].long()
    cache.v_scale[ids[0::2]] = 1e-30
    cache.v.view(torch.uint8)[ids[0::2]] = 0
    cache.v_scale[ids[1::4]] = large
    cache.v_scale[ids[: len(ids) // 3]] = 1e-30  # the first workers see nothing else
    q = torch.randn((new, per, 64), generator=_gen(1, cuda), device=cuda).to(BF) * score
    got, lse = kvcache.attention(q, cache, table, _i32([total], cuda), return_lse=True)
    check_attention(q, cache, table, [total], [new], got, lse, 0.125, True, 0)
    assert h3q.device_status() == 0


@pytest.mark.parametrize("new", [5, 150])
@pytest.mark.parametrize("window", [0, 300])
def test_values_of_pages_far_apart_behind_masks(cuda, new, window):
    """The same with windows that leave only quiet or only loud pages to a row, and stretches of pages that are not there."""
    total, page = 3000, 32
    cache, table = make_cache(cuda, E4, 2, page, 128, [total], 42)
    ids = table[0, :-(-total // page)].long()
    cache.v_scale[ids[0::3]] = 1e-30
    cache.v_scale[ids[1::7]] = 1e25
    cache.v_scale[ids[-4:]] = 1e-28  # what the newest rows see beside themselves is 2^170 louder
    gone = [(320, 704), (2304, 2560), (2720, 2784)]
    holes = table.clone()
    for lo, hi in gone:
        holes[0, lo // page:hi // page] = -1
    q = torch.randn((new, 4, 128), generator=_gen(2, cuda), device=cuda).to(BF)
    got, lse = kvcache.attention(q, cache, holes, _i32([total], cuda), window=window, return_lse=True)
    check_attention(q, cache, table, [total], [new], got, lse, 128 ** -0.5, True, window, gone={0: gone})
    assert h3q.device_status() == 0


@pytest.mark.parametrize("codes", [I8, E4])
@pytest.mark.parametrize("new,per", [(1, 1), (5, 4), (40, 4)])
def test_a_key_of_nearly_all_weight_and_no_value(cuda, codes, new, per):
    """The first key has 0.99 of a row's weight and zeros for a value, so the row's output is the sum over the others, whose
    weights are 2^-20 of the first's.  Weights are f16 times a power of two that brings the row's largest w to 2^7 or more, so
    the smallest step is 2^-24 and a weight's rounding costs 2^-11 of it or 2^-25 of that power: 2^-32 max(p vs) sum |vcode|
    in all; the other terms are those of check_attention."""
    hk, dim, page, n, batch = 16, 64, 128, 12800, 24  # 384 rows of work share a pool: few of them are cut
    g = _gen(7, cuda)
    raw = [torch.zeros((n // page, hk, page, dim), device=cuda) for _ in range(2)]
    raw[0][0, :, 0] = 100.0
    raw[1].uniform_(60, 120, generator=g)
    raw[1][0, :, 0] = 0
    k, v = [(x.round() if codes == I8 else x).to(codes) for x in raw]
    ks = torch.full((n // page, hk), 0.01, device=cuda)
    vs = torch.full((n // page, hk), 0.02, device=cuda)
    cache = kvcache.KVCache(k, v, ks, vs)
    table = torch.arange(n // page, dtype=torch.int32, device=cuda).repeat(batch, 1)
    q = torch.ones((batch * new, hk * per, dim), device=cuda).to(HF)  # q . k = 64 for the first key, 0 for the others
    kfirst = float(k[0, 0, 0, 0].float())
    scale = math.log(99.0 * n) / (64 * kfirst * float(ks[0, 0]))
    got, lse = kvcache.attention(q, cache, table, _i32([n] * batch, cuda), scale=scale, return_lse=True)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    vd = v.double().transpose(0, 1).flatten(1, 2) * float(vs[0, 0])  # [hk, n, dim]
    first = math.exp(scale * 64 * kfirst * float(ks[0, 0]))
    sums = vd.cumsum(1)
    for i in range(new):
        m = n - new + 1 + i  # keys that token i of a sequence sees
        total = first + m - 1
        want = sums[:, m - 1] / total
        o = got.view(batch, new, hk, per, dim)[:, i].double()
        sub = (first / total) * vd[:, :m].abs().sum(1)
        tol = (2.0 ** -11 + 2.0 ** -16 + 2.0 ** -11) * want + 2.0 ** -32 * sub
        worst = ((o - want[None, :, None]).abs() / tol[None, :, None]).max().item()
        assert worst <= 1.0, (i, worst)
        assert ((lse.view(batch, new, hk * per)[:, i].double() - math.log(total)).abs() <= 2.0 ** -17 * 20).all()


@pytest.mark.parametrize("new", [1, 8, 200])
def test_scales_below_the_smallest(cuda, new):
    """Scales of 0, below 1e-30, negative and NaN count as 1e-30 in attention, those of K and of V alike, in every kernel."""
    totals = [400]
    bad, table = make_cache(cuda, I8, 2, 16, 128, totals, 13)
    ids = table[0, :25].tolist()
    good = kvcache.KVCache(bad.k, bad.v, bad.k_scale.clone(), bad.v_scale.clone())
    for i, x in enumerate((0.0, 5e-31, -0.03, float("nan"), -math.inf)):
        bad.k_scale[ids[2 * i]] = x
        bad.v_scale[ids[2 * i + 11]] = x
        good.k_scale[ids[2 * i]] = 1e-30
        good.v_scale[ids[2 * i + 11]] = 1e-30
    q = torch.randn((new, 8, 128), generator=_gen(1, cuda), device=cuda).to(BF)
    n = _i32(totals, cuda)
    want, want_lse = kvcache.attention(q, good, table, n, return_lse=True)
    check_attention(q, good, table, totals, [new], want, want_lse, 128 ** -0.5, True, 0)
    got, lse = kvcache.attention(q, bad, table, n, return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("new,causal,window", [(3, True, 0), (8, True, 0), (8, True, 40), (120, True, 0), (120, True, 50), (120, False, 0)])
def test_a_table_shorter_than_the_sequence(cuda, new, causal, window):
    """Tokens behind the table's last page are not there; the queries keep their positions, so masks stay where they were."""
    totals = [170, 90]
    cache, table = make_cache(cuda, I8, 2, 32, 64, totals, 14)
    q = torch.randn((2 * new, 8, 64), generator=_gen(2, cuda), device=cuda).to(BF)
    news = [new, new]
    short = table[:, :3].contiguous()  # 96 tokens
    got, lse = kvcache.attention(q, cache, short, _i32(totals, cuda), causal=causal, window=window, return_lse=True)
    fixed = table.clamp_min(0)
    check_attention(q, cache, fixed, totals, news, got, lse, 0.125, causal, window, gone={0: [(96, 170)]})


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("new,total", [(1, 300), (1, 30000), (8, 300), (70, 300), (70, 30000)])
def test_a_query_that_is_not_a_number(cuda, kind, new, total):
    """A NaN in a query makes its row and its lse NaN, also where the row's keys are split between workers; the other rows
    are what they are without it."""
    cache, table = make_cache(cuda, I8, 1, 64, 64, [total], 15)
    q = torch.randn((new, 4, 64), generator=_gen(3, cuda), device=cuda).to(kind)
    n = _i32([total], cuda)
    want, want_lse = kvcache.attention(q, cache, table, n, return_lse=True)
    q[new // 2, 1, 5] = float("nan")
    got, lse = kvcache.attention(q, cache, table, n, return_lse=True)
    assert torch.isnan(got[new // 2, 1]).all() and torch.isnan(lse[new // 2, 1])
    rest = torch.ones((new, 4), dtype=torch.bool, device=cuda)
    rest[new // 2, 1] = False
    assert torch.equal(got[rest], want[rest]) and torch.equal(lse[rest], want_lse[rest])


@pytest.mark.parametrize("first,news", [(16, [1, 1, 1, 1, 0]), (33, [40, 7]), (5, [200, 90]), (700, [150, 60])])
def test_a_first_sequence_that_begins_behind_row_0(cuda, first, news):
    """Rows before starts[0] are nobody's: they are not written, and the others are as in a call without them.  Pages whose
    scale is 0 would show a page of another place being rounded anew."""
    pasts = [40 + 30 * b for b in range(len(news))]
    totals = [a + n for a, n in zip(pasts, news)]
    one, table = make_cache(cuda, I8, 2, 16, 64, totals, 17)
    for b, past in enumerate(pasts):
        for i in range(past // 16):
            one.k_scale[table[b, i]] = 0
            one.v_scale[table[b, i]] = 0
    two = kvcache.KVCache(*[x.clone() for x in (one.k, one.v, one.k_scale, one.v_scale)])
    t = sum(news)
    x = torch.randn((first + t, 4, 64), generator=_gen(5, cuda), device=cuda).to(BF)
    starts, late = _i32(_starts(news), cuda), _i32([first + s for s in _starts(news)], cuda)
    past, n = _i32(pasts, cuda), _i32(totals, cuda)
    kvcache.write(one, x[first:, :2], x[first:, 2:], table, past, starts)
    kvcache.write(two, x[:, :2], x[:, 2:], table, past, late)
    for a, b in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(kvcache.read(one, table, starts, t, first=past), kvcache.read(one, table, late, first + t, first=past)):
        assert torch.equal(a, b[first:])
    q = torch.randn((8, first + t, 64), generator=_gen(6, cuda), device=cuda).to(BF).transpose(0, 1)  # heads lie far apart
    for most in (0, max(news)):
        want = kvcache.attention(q[first:], one, table, n, starts, max_new=most)
        assert torch.equal(want, kvcache.attention(q, one, table, n, late, max_new=most)[first:])
    assert h3q.device_status() == 0


def _litter(*shapes):
    """Leaves memory of these sizes full of NaN to the allocator."""
    for shape, kind in shapes:
        torch.full(shape, float("nan"), dtype=kind, device="cuda")


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("extra", [3, 700])
def test_rows_of_no_sequence(cuda, new, extra):
    """Rows behind the last sequence's (the padding of a captured step) or before the first are zeros, with an lse of -inf."""
    totals, news = [100, 60], [new, new]
    cache, table = make_cache(cuda, I8, 2, 32, 64, totals, 16)
    t = 2 * new + extra
    q = torch.randn((t, 8, 64), generator=_gen(4, cuda), device=cuda).to(BF)
    n, starts = _i32(totals, cuda), _i32(_starts(news), cuda)
    for most in (0, new):
        _litter(((t, 8, 64), BF), ((t, 8), torch.float32))
        got, lse = kvcache.attention(q, cache, table, n, starts, return_lse=True, max_new=most)
        check_attention(q, cache, table, totals, news, got, lse, 0.125, True, 0)
        assert (got[2 * new:] == 0).all() and (lse[2 * new:] == -math.inf).all()
        _litter(((t, 8, 64), BF), ((t, 8), torch.float32))
        late, late_lse = kvcache.attention(q, cache, table, n, starts + extra, return_lse=True, max_new=most)
        check_attention(q[extra:], cache, table, totals, news, late[extra:], late_lse[extra:], 0.125, True, 0)
        assert (late[:extra] == 0).all() and (late_lse[:extra] == -math.inf).all()
    starts = _i32([0, 100, 160], cuda)
    for kind in (torch.float32, HF, BF):
        shape = (160 + extra, 2, 64)
        _litter((shape, kind), (shape, kind))
        k, v = kvcache.read(cache, table, starts, 160 + extra, kind)
        want_k, want_v = kvcache.read(cache, table, starts, 160, kind)
        assert torch.equal(k[:160], want_k) and torch.equal(v[:160], want_v)
        assert (k[160:] == 0).all() and (v[160:] == 0).all()
        _litter((shape, kind), (shape, kind))
        k, v = kvcache.read(cache, table, starts + extra, 160 + extra, kind)
        assert torch.equal(k[extra:], want_k) and torch.equal(v[extra:], want_v)
        assert (k[:extra] == 0).all() and (v[:extra] == 0).all()


def test_workspaces(cuda):
    """A workspace that the kernels could not write to is refused; one of any type is taken by its bytes, and a new one where
    it is too small or has none."""
    totals = [300, 20]
    cache, table = make_cache(cuda, I8, 2, 32, 64, totals, 18)
    q = torch.randn((80, 8, 64), generator=_gen(7, cuda), device=cuda).to(BF)
    n = _i32(totals, cuda)
    want = kvcache.attention(q, cache, table, n)
    need = h3q.lib().h3q_kv_attention_workspace_size(80, 2, 8, 2, 64, 40)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device=cuda)[::2],
                torch.empty(1, dtype=torch.uint8, device=cuda).expand(need), torch.empty(need, device="meta")):
        with pytest.raises(h3q.H3QError) as e:
            kvcache.attention(q, cache, table, n, workspace=bad)
        assert e.value.status == h3q.ERR_ARG and "workspace" in str(e.value)
    with pytest.raises(h3q.H3QError):  # not on a 16-byte boundary
        kvcache.attention(q, cache, table, n, workspace=torch.empty(need + 1, dtype=torch.uint8, device=cuda)[1:])
    guard = torch.full((need // 4 + 64,), 7.0, device=cuda)
    for ws in (guard[:need // 4 + 1], torch.empty(16, dtype=torch.uint8, device=cuda),
               torch.empty(0, dtype=torch.uint8, device=cuda), torch.empty(need, dtype=torch.uint8, device=cuda)):
        assert torch.equal(kvcache.attention(q, cache, table, n, workspace=ws), want)
    assert (guard[need // 4 + 1:] == 7).all()
