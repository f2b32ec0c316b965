"""Prompt chunks of a few sequences among very many without new tokens. Tolerances: those of test_gpu_paged.py."""
import numpy as np
import pytest

from paged_util import HostCache, attention, from_bf16, to_bf16
from test_gpu_paged import W, close, same_lse, upload
from test_paged_cpu import desc, prefill


def test_more_sequences_than_the_call_takes_are_refused(lthn):
    d = desc(lthn, seqs=1 << 21)
    assert prefill(lthn, d, seqs=(1 << 20) + 1) == 1 and b"sequences" in lthn.lib().lthn_last_error()
    d = desc(lthn, seqs=1 << 20, kv_heads=16)
    assert prefill(lthn, d, seqs=1 << 20, total=1 << 20, q_heads=16) == 1 and b"sequences" in lthn.lib().lthn_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [100, 5000, 1 << 15, (1 << 15) + 1, 1 << 20])
@pytest.mark.parametrize("kv", [1, 3])
def test_prefill_few_of_many_sequences(lthn, seqs, kv):
    """Under a table wide enough that most chunks of the plan are not there, and with rows that nobody owns: many look-ups find nothing."""
    rng = np.random.default_rng(51)
    D, G, page = 64, 2, 1 << 16
    lens, new = [300, 120, 77, 1], [3, 1, 70, 1]
    where = np.array([0, seqs // 3, seqs - 2, seqs - 1])
    c = HostCache(rng, lens, page, kv, D, spare=0)
    table = np.full((seqs, 2), -7, dtype=np.int32)
    table[where, :c.table_stride] = c.table
    every = rng.integers(0, 1 << 16, seqs).astype(np.int32)          # lengths of sequences without new tokens: nobody needs their pages
    every[where] = lens
    count = np.zeros(seqs, dtype=np.int64)
    count[where] = new
    start = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    total = int(start[-1]) + 200                                     # rows that nobody owns behind them
    Hq = kv * G
    q, qb = upload(lthn, rng.standard_normal((total, Hq, D)), False)
    out = lthn.Buf.from_array(to_bf16(np.full((total, Hq, D), 5.0)))
    lse = lthn.Buf.from_array(np.full((total, Hq), 5.0, dtype=np.float32))
    dev = lthn.PagedKV(lthn.Buf.from_array(c.k), lthn.Buf.from_array(c.v), lthn.Buf.from_array(table), pages=c.pages, page_size=page, kv_heads=kv,
                       head_dim=D, seqs=seqs, table_stride=2)
    ws = lthn.Buf(lthn.paged_prefill_attention_workspace(dev, seqs, total, Hq))
    lthn.paged_prefill_attention(dev, qb, lthn.Buf.from_array(start), lthn.Buf.from_array(every), seqs, total, Hq, out, ws, lse=lse)
    lthn.sync()
    assert lthn.device_status() == 0
    got, sums = from_bf16(out.download(np.uint16, (total, Hq, D))), lse.download(np.float32, (total, Hq))
    for s, n in enumerate(lens):
        rows = slice(start[where[s]], start[where[s] + 1])
        want, wl, mag = attention(c, s, q[rows], n - new[s], n)
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag)
        same_lse(sums[rows], wl)
    assert np.all(got[start[-1]:] == 5.0) and np.all(sums[start[-1]:] == 5.0)
