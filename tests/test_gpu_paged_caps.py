"""The tanh cap of the paged attention calls over its whole range, against the formula in 64 bits.

Tolerances. Those of test_gpu_paged.py: a weight is off, relatively, by W = 2e-5 at scores of |q| |k| scale up to about 30. The cap itself adds
an error of at most 2^-20 of the score (f32 arithmetic of tanh), 6e-6 at the scores of up to 6 of standard normal q and k and so within
W; with q made t times larger, scores and their errors are t times larger before the cap, whose slope is at most 1."""
import numpy as np
import pytest

from paged_util import HostCache, attention
from test_gpu_paged import W, close, options, run_decode, run_prefill, widen

pytestmark = pytest.mark.gpu

# (cap, factor of q): caps far above the scores ("no cap", as some callers write it), near them, far below
CAPS = [(200.0, 1), (1e3, 1), (1e4, 1), (1e6, 1), (1e30, 1), (1e38, 1), (3.4e38, 1), (30.0, 4), (5.0, 4), (2.0, 1), (0.5, 1), (1e-3, 1), (1e-30, 1), (1e-42, 1)]


def same_lse(got, want, factor):
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    f = np.isfinite(want)
    assert np.all(np.abs(got[f] - want[f]) <= factor * W + 2.0 ** -22 * np.abs(want[f]))


@pytest.mark.parametrize("cap,factor", CAPS)
@pytest.mark.parametrize("D,kv,G", [(64, 1, 3), (128, 2, 2), (256, 1, 2)])
@pytest.mark.parametrize("slopes", [False, True])
def test_prefill_caps(lthn, cap, factor, D, kv, G, slopes):
    rng = np.random.default_rng(41)
    new, past = [150, 3, 64], [0, 200, 130]
    lens = [a + b for a, b in zip(new, past)]
    c = HostCache(rng, lens, 16, kv, D)
    o, kws = options(lthn, rng, kv * G, lens, softcap=cap, slopes=slopes)
    q = rng.standard_normal((sum(new), kv * G, D)) * factor
    q[::7] = 0.0                                     # scores of exactly zero
    x, got, lse, start = run_prefill(lthn, c, q, new, o)
    for s, n in enumerate(lens):
        rows = slice(start[s], start[s + 1])
        want, wl, mag = attention(c, s, x[rows], n - new[s], n, **kws[s])
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + factor * W) * mag)
        same_lse(lse[rows], wl, factor)


@pytest.mark.parametrize("cap,factor", CAPS)
@pytest.mark.parametrize("D,kv,G,f32", [(64, 1, 9, False), (128, 2, 2, True), (256, 1, 4, False)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_caps(lthn, cap, factor, D, kv, G, f32, wide):
    rng = np.random.default_rng(42)
    lens = [400, 1, 0, 99, 163]
    c = HostCache(rng, lens, 24, kv, D)
    if wide:
        c = widen(c, 1 << 17)
    o, kws = options(lthn, rng, kv * G, lens, softcap=cap)
    q = rng.standard_normal((len(lens), kv * G, D)) * factor
    q[3] = 0.0
    x, got, lse = run_decode(lthn, c, q, f32, o)
    rounded = 0.0 if f32 else 2.0 ** -8
    for r, n in enumerate(lens):
        want, wl, mag = attention(c, r, x[r:r + 1], n - 1, n, **kws[r])
        close(got[r:r + 1], want, (rounded + 2.0 ** -23) * np.abs(want) + (factor * W + (rounded if G > 8 else 0.0)) * mag)
        same_lse(lse[r:r + 1], wl, factor)


@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30])
def test_a_prompt_and_the_token_behind_it_agree(lthn, cap):
    """The last row of a prompt chunk and the one-token call give the same sums under the same options."""
    rng = np.random.default_rng(43)
    c = HostCache(rng, [300], 16, 2, 128)
    o, kws = options(lthn, rng, 4, [300], softcap=cap)
    q = rng.standard_normal((40, 4, 128))
    _, got, lse, _ = run_prefill(lthn, c, q, [40], o)
    x, one, one_lse = run_decode(lthn, c, q[-1:], False, o)
    _, _, mag = attention(c, 0, x, 299, 300, **kws[0])
    close(got[-1:], one, 2.0 ** -8 * np.abs(one) + 2.0 ** -8 * np.abs(got[-1:]) + (2.0 ** -8 + 2 * W) * mag)
    assert np.all(np.abs(lse[-1] - one_lse[0]) <= 2 * W + 2.0 ** -22 * np.abs(one_lse[0]))


def test_prefill_caps_far_from_and_near_the_scores_in_one_tile(lthn):
    """Rows of small scores beside rows whose scores are several caps: both forms of the cap in one tile of keys, and a key whose
    score is several caps beside keys whose scores are a small part of it."""
    rng = np.random.default_rng(44)
    c = HostCache(rng, [260], 16, 1, 128)
    k, v = c.get(0, 260)
    k[::9] *= 6.0
    c.put(0, np.arange(260), k, v)
    o, kws = options(lthn, rng, 2, [260], softcap=4.0)
    q = rng.standard_normal((200, 2, 128)) * 2.0 ** rng.uniform(-6, 2, (200, 1, 1))
    x, got, lse, _ = run_prefill(lthn, c, q, [200], o)
    want, wl, mag = attention(c, 0, x, 60, 260, **kws[0])
    close(got, want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 24 * W) * mag)      # |q| up to 4 and |k| up to 6 times larger
    same_lse(lse, wl, 24)


@pytest.mark.parametrize("cap", [63.0, 64.0, 65.0, 100.0, 1000.0])
@pytest.mark.parametrize("D,slopes", [(64, False), (128, True), (256, False)])
def test_prefill_scores_around_a_large_cap(lthn, cap, D, slopes):
    """The same around the caps where the form changes: scores from hundredths to several times of 30."""
    rng = np.random.default_rng(45)
    c = HostCache(rng, [260, 70], 16, 1, D)
    for s, n in enumerate(c.lens):
        k, v = c.get(s, n)
        k[::9] *= 6.0
        c.put(s, np.arange(n), k, v)
    o, kws = options(lthn, rng, 2, c.lens, softcap=cap, slopes=slopes)
    new = [200, 70]
    q = rng.standard_normal((270, 2, D)) * 2.0 ** rng.uniform(-6, 3, (270, 1, 1))
    x, got, lse, start = run_prefill(lthn, c, q, new, o)
    for s, n in enumerate(c.lens):
        rows = slice(start[s], start[s + 1])
        want, wl, mag = attention(c, s, x[rows], n - new[s], n, **kws[s])
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 48 * W) * mag)      # |q| up to 8 and |k| up to 6 times larger
        same_lse(lse[rows], wl, 48)
