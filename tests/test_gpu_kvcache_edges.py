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
