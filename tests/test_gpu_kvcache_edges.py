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
