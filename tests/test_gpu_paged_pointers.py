"""Pointers that a kernel could not use are errors of the call: host memory in the place of every argument, before anything is launched.
(Misaligned ones: test_paged_pointers_cpu.py.)"""
import ctypes as C

import numpy as np
import pytest

from paged_util import HostCache, attention, from_bf16, to_bf16
from test_gpu_paged import W, close

pytestmark = pytest.mark.gpu

HOST = np.zeros(1 << 16, dtype=np.uint8)
ADDRESS = (HOST.ctypes.data + 255) & ~255


@pytest.fixture()
def calls(lthn):
    """The three calls as functions of their arguments by name, and arguments that are fine."""
    c = HostCache(np.random.default_rng(71), [10, 4], 8, 1, 64)
    dev = c.device(lthn)
    b = lthn.Buf(1 << 20)
    b.zero()
    work = lthn.Buf(8 << 20)
    one = lthn.Buf.from_array(np.array([0, 1, 2, 0], dtype=np.int32))
    lens = lthn.Buf.from_array(np.array(c.lens, dtype=np.int32))
    f64 = lthn.Buf.from_array(lthn.rope_inv_freq(1e4, 64))
    f32 = lthn.Buf.from_array(np.ones(64, dtype=np.float32))
    L = lthn.lib()
    cache = {n: getattr(dev.desc, n) for n, _ in lthn.PagedKVDesc._fields_}
    a = dict(cache, q=b.ptr, kk=b.ptr + 4096, vv=b.ptr + 8192, q_out=b.ptr + 16384, out=b.ptr + 32768, lse=b.ptr + 65536, row_seq=one.ptr, row_pos=lens.ptr,
             kv_lens=lens.ptr, q_start=one.ptr, inv_freq=f64.ptr, q_norm=f32.ptr, k_norm=f32.ptr, slopes=f32.ptr, prefix=one.ptr, work=work.ptr)

    def desc(x):
        return lthn.PagedKVDesc(*[x[n] for n, _ in lthn.PagedKVDesc._fields_])

    def append(x):
        r = lthn.RopeParams(x["inv_freq"], 64, 0, x["q_norm"], x["k_norm"], 1e-6)
        return L.lthn_paged_kv_append(None, desc(x), r, x["q"], x["kk"], x["vv"], 1, 0, 0, 0, x["row_seq"], x["row_pos"], 2, 2, x["q_out"], 1, 0)

    def decode(x):
        o = lthn.AttnOptions(0.0, 0.0, x["slopes"], 0, x["prefix"])
        return L.lthn_paged_sdpa_decode(None, desc(x), o, x["q"], 1, 0, x["kv_lens"], 2, 2, x["out"], 0, x["lse"], x["work"], 8 << 20)

    def prefill(x):
        o = lthn.AttnOptions(0.0, 0.0, x["slopes"], 0, x["prefix"])
        return L.lthn_paged_prefill_attention(None, desc(x), o, x["q"], 0, x["q_start"], x["kv_lens"], 2, 2, 2, 0, x["out"], 0, x["lse"], x["work"], 8 << 20)
    keep = (c, dev, b, work, one, lens, f64, f32)
    return dict(append=append, decode=decode, prefill=prefill), a, keep


COMMON = ["k", "v", "page_table", "q"]
ARGS = ([("append", n) for n in COMMON + ["kk", "vv", "q_out", "row_seq", "row_pos", "inv_freq", "q_norm", "k_norm"]] +
        [(call, n) for call in ("decode", "prefill") for n in COMMON + ["kv_lens", "out", "lse", "work", "slopes", "prefix"]] + [("prefill", "q_start")])


@pytest.mark.parametrize("call,name", ARGS)
def test_host_memory_is_refused_wherever_it_stands(lthn, calls, call, name):
    run, good, _ = calls
    assert run[call](dict(good, **{name: ADDRESS})) == 1
    assert b"memory of the current device" in lthn.lib().lthn_last_error()
    assert run[call](good) == 0
    assert lthn.device_status() == 0


def test_memory_of_one_allocation_and_of_many(lthn, calls):
    """Arguments that lie in more allocations than the check remembers, optional ones left out, and pinned host memory for lengths."""
    run, good, _ = calls
    for call in run.values():
        assert call(good) == 0
        assert call(dict(good, slopes=None, prefix=None, lse=None, inv_freq=None, q_norm=None, k_norm=None)) == 0
    lthn.sync()
    assert lthn.device_status() == 0


def test_lengths_in_pinned_host_memory(lthn):
    """Page-locked host memory that the device can reach holds the lengths, as a server writes them."""
    rng = np.random.default_rng(72)
    c = HostCache(rng, [33, 70], 16, 1, 64)
    dev = c.device(lthn)
    h = C.c_void_p()
    lthn.check(lthn.lib().lthn_host_alloc(C.byref(h), 4096))
    try:
        lens = np.ctypeslib.as_array(C.cast(h, C.POINTER(C.c_int32)), (2,))
        lens[:] = c.lens
        q = to_bf16(rng.standard_normal((2, 2, 64)))
        out = lthn.Buf(2 * 2 * 64 * 2)
        ws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, 2, 2, lthn.BF16))
        at = type("P", (), {"data_ptr": lambda self: h.value})()
        lthn.paged_sdpa_decode(dev, lthn.Buf.from_array(q), lthn.BF16, at, 2, 2, out, ws)
        lthn.sync()
        got = from_bf16(out.download(np.uint16, (2, 2, 64)))
    finally:
        lthn.lib().lthn_host_free(h)
    for r, n in enumerate(c.lens):
        want, _, mag = attention(c, r, from_bf16(q[r:r + 1]), n - 1, n)
        close(got[r:r + 1], want, 2.0 ** -8 * np.abs(want) + W * mag)
