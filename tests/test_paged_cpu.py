"""Refusals of the paged-cache entry points: all of them come before any device work, so they are checked without one."""
import ctypes as C

import numpy as np
import pytest


def desc(lthn, **kw):
    """A description that is fine; its addresses are aligned and never used."""
    d = dict(k=1 << 20, v=1 << 21, page_table=1 << 22, page_stride=0, row_stride=0, head_stride=0, pages=8, page_size=16, table_stride=4,
             seqs=2, kv_heads=2, head_dim=64)
    d.update(kw)
    return lthn.PagedKVDesc(*[d[n] for n, _ in lthn.PagedKVDesc._fields_])


A = 1 << 24   # an aligned address


def append(lthn, d, rope=None, q=A, k=A, v=A, dtype=1, qs=0, ks=0, vs=0, seq=A, pos=A, rows=2, q_heads=4, q_out=A + 4096, q_dtype=1, qos=0):
    return lthn.lib().lthn_paged_kv_append(None, d, rope, q, k, v, dtype, qs, ks, vs, seq, pos, rows, q_heads, q_out, q_dtype, qos)


def decode(lthn, d, o=None, q=A, dtype=1, qs=0, lens=A, rows=2, q_heads=4, out=A, os=0, ws=A, n=1 << 30):
    return lthn.lib().lthn_paged_sdpa_decode(None, d, o, q, dtype, qs, lens, rows, q_heads, out, os, None, ws, n)


def prefill(lthn, d, o=None, q=A, qs=0, start=A, lens=A, seqs=2, total=9, q_heads=4, ctx=0, out=A, os=0, ws=A, n=1 << 40):
    return lthn.lib().lthn_paged_prefill_attention(None, d, o, q, qs, start, lens, seqs, total, q_heads, ctx, out, os, None, ws, n)


BAD_CACHE = [dict(k=None), dict(v=None), dict(page_table=None), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(page_size=0), dict(page_size=-1),
             dict(pages=-1), dict(table_stride=-1), dict(seqs=-1), dict(kv_heads=0), dict(kv_heads=-2), dict(head_dim=80), dict(head_dim=0),
             dict(head_dim=512), dict(row_stride=129), dict(head_stride=68), dict(page_stride=2052), dict(row_stride=-128), dict(page_stride=-4096)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache_descriptions_are_refused(lthn, bad):
    for call in (append, decode, prefill):
        assert call(lthn, desc(lthn, **bad)) == 1, call.__name__
        assert lthn.lib().lthn_last_error()


def test_null_descriptions_are_refused(lthn):
    for call in (append, decode, prefill):
        assert call(lthn, None) == 1


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(dtype=2), dict(q_dtype=-1), dict(q_heads=-1), dict(k=None), dict(v=None), dict(seq=None),
                                 dict(pos=None), dict(q_out=None), dict(k=A + 4), dict(v=A + 8), dict(q=A + 2), dict(q_out=A + 8), dict(ks=132),
                                 dict(vs=-3), dict(qs=260), dict(qos=20), dict(qos=128), dict(q_out=A, q_dtype=0), dict(q_out=A, qs=512)], ids=str)
def test_append_refuses(lthn, bad):
    assert append(lthn, desc(lthn), **bad) == 1


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=-2), dict(interleaved=2), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(q_norm=A + 4), dict(k_norm=A + 8)], ids=str)
def test_append_refuses_rope(lthn, bad):
    r = dict(inv_freq=A, rotary_dim=64, interleaved=0, q_norm=None, k_norm=None, eps=1e-6)
    r.update(bad)
    assert append(lthn, desc(lthn), lthn.RopeParams(*[r[n] for n, _ in lthn.RopeParams._fields_])) == 1


BAD_OPTIONS = [dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1)]


@pytest.mark.parametrize("bad", BAD_OPTIONS, ids=str)
def test_attention_refuses_options(lthn, bad):
    for call in (decode, prefill):
        assert call(lthn, desc(lthn), lthn.attn_options(**bad)) == 1


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=3), dict(dtype=5), dict(q_heads=0), dict(q_heads=3), dict(q_heads=-2), dict(q=None), dict(out=None),
                                 dict(lens=None), dict(ws=None), dict(n=16), dict(q=A + 8), dict(out=A + 4), dict(ws=A + 8), dict(qs=257), dict(os=12),
                                 dict(os=128)], ids=str)
def test_decode_refuses(lthn, bad):
    assert decode(lthn, desc(lthn), **bad) == 1


@pytest.mark.parametrize("bad", [dict(seqs=-1), dict(seqs=3), dict(total=-1), dict(ctx=-1), dict(q_heads=0), dict(q_heads=5), dict(q=None), dict(out=None),
                                 dict(start=None), dict(lens=None), dict(ws=None), dict(n=8), dict(q=A + 2), dict(out=A + 8), dict(ws=A + 4), dict(qs=257),
                                 dict(os=12), dict(os=128), dict(qs=128), dict(total=(1 << 30) + 1), dict(q_heads=258)], ids=str)
def test_prefill_refuses(lthn, bad):
    assert prefill(lthn, desc(lthn), **bad) == 1


def test_empty_calls_are_clean(lthn):
    d = desc(lthn)
    assert append(lthn, d, rows=0, k=None, v=None, seq=None, pos=None) == 0
    assert decode(lthn, d, rows=0, q=None, out=None, lens=None, ws=None) == 0
    assert prefill(lthn, d, seqs=0, q=None, out=None, start=None, lens=None, ws=None) == 0
    assert prefill(lthn, d, total=0, q=None, out=None, start=None, lens=None, ws=None) == 0


def test_workspace_queries(lthn):
    d, n = desc(lthn, seqs=64), C.c_size_t()
    L = lthn.lib()
    for rows in (1, 64):
        assert L.lthn_paged_sdpa_decode_workspace(d, rows, 4, 1, C.byref(n)) == 0 and n.value > 0
    assert L.lthn_paged_prefill_attention_workspace(d, 1, 100, 4, 0, C.byref(n)) == 0 and n.value >= 16
    assert L.lthn_paged_sdpa_decode_workspace(d, 1, 4, 1, None) == 1
    assert L.lthn_paged_prefill_attention_workspace(d, 1, 1, 4, 0, None) == 1
    assert L.lthn_paged_sdpa_decode_workspace(d, 65, 4, 1, C.byref(n)) == 1


def test_rope_inv_freq(lthn):
    f = lthn.rope_inv_freq(10000.0, 128, 64)
    assert f.dtype == np.float64 and f.shape == (32,)
    assert np.allclose(f, [10000.0 ** (-2 * i / 128) for i in range(32)], rtol=1e-15)
