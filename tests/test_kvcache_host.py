"""CPU tests of the 8-bit cache's C ABI: its argument checks answer before any device work."""
import ctypes

import pytest

import h3q

FAKE = 1 << 20  # an aligned address that no call here dereferences


def desc(**kw):
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pages=4, kv_heads=2, page=64, head_dim=128, codes=0) | kw
    return h3q.KvCacheDesc(**a)


def attention(d=None, q=FAKE, kind=2, tokens=4, heads=8, table=FAKE, width=3, lengths=FAKE, starts=FAKE, batch=2, max_new=0,
              scale=1.0, causal=1, window=0, out=FAKE, ws=FAKE, ws_bytes=0, ts=1024, hs=128):
    return h3q.lib().h3q_kv_attention(ctypes.byref(d or desc()), q, kind, ts, hs, tokens, heads, table, width, lengths,
                                      starts, batch, max_new, scale, causal, window, out, None, ws, ws_bytes, None)


def write(d=None, k=FAKE, kind=2, tokens=4, table=FAKE, width=3, past=FAKE, starts=FAKE, batch=2, ts=256, hs=128):
    return h3q.lib().h3q_kv_write(ctypes.byref(d or desc()), k, ts, hs, k, ts, hs, kind, tokens, table, width, past, starts,
                                  batch, None)


def read(d=None, table=FAKE, width=3, starts=FAKE, batch=2, tokens=4, out=FAKE, kind=2):
    return h3q.lib().h3q_kv_read(ctypes.byref(d or desc()), table, width, None, starts, batch, tokens, out, out, kind, None)


@pytest.mark.parametrize("call", [attention, write, read])
def test_cache_checks(call):
    for bad in (dict(pages=-1), dict(kv_heads=0), dict(codes=2), dict(k=None), dict(v=FAKE + 8), dict(k_scale=FAKE + 1)):
        assert call(desc(**bad)) == h3q.ERR_ARG, bad
    for bad in (dict(head_dim=96), dict(page=24), dict(page=256), dict(kv_heads=5000)):
        assert call(desc(**bad)) == h3q.ERR_UNSUPPORTED, bad
        assert "this build handles" in h3q.last_error()


@pytest.mark.parametrize("call", [attention, write, read])
def test_sequence_checks(call):
    for bad in (dict(tokens=-1), dict(batch=-1), dict(width=-1), dict(table=None), dict(batch=0), dict(starts=None, batch=3)):
        assert call(**bad) == h3q.ERR_ARG, bad
    for bad in (dict(tokens=1 << 25), dict(batch=1 << 21), dict(width=1 << 27)):
        assert call(**bad) == h3q.ERR_UNSUPPORTED, bad


def test_attention_checks():
    for bad in (dict(kind=0), dict(kind=3), dict(heads=7), dict(heads=0), dict(q=None), dict(out=None), dict(lengths=None),
                dict(out=FAKE + 8), dict(q=FAKE + 1), dict(scale=float("inf")), dict(window=-1), dict(max_new=-1),
                dict(causal=0, window=5), dict(ts=-1), dict(hs=-1)):
        assert attention(**bad) == h3q.ERR_ARG, bad
    assert attention(ws_bytes=16) == h3q.ERR_WORKSPACE
    assert attention(ws=None, ws_bytes=1 << 40) == h3q.ERR_WORKSPACE
    assert attention(ws=FAKE + 8, ws_bytes=1 << 40) == h3q.ERR_ARG


def test_write_and_read_checks():
    for bad in (dict(kind=3), dict(k=None), dict(past=None), dict(k=FAKE + 1), dict(ts=-1), dict(hs=-2)):
        assert write(**bad) == h3q.ERR_ARG, bad
    for bad in (dict(kind=-1), dict(out=None), dict(out=FAKE + 4)):
        assert read(**bad) == h3q.ERR_ARG, bad


def test_empty_calls_do_nothing():
    assert attention(tokens=0, batch=0, starts=None) == h3q.OK
    assert write(tokens=0, batch=0, starts=None) == h3q.OK
    assert read(tokens=0, batch=0, starts=None) == h3q.OK
    assert write(desc(pages=0, k=None, v=None, k_scale=None, v_scale=None)) == h3q.OK


def test_workspace_size():
    size = h3q.lib().h3q_kv_attention_workspace_size
    assert size(0, 0, 8, 8, 128, 0) == 0
    assert size(4, 2, 8, 2, 128, 1) > 0
    assert size(4096, 2, 8, 2, 128, 4096) >= size(4096, 2, 8, 2, 128, 0)
