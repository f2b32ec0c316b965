"""The paged-cache operators against the same formulas in 64 bits.

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, to f32 by 2^-24.
Append: the rotation of (a, b) is two f32 products and a sum, each off by 2^-24, with a sine and cosine off by a few
2^-24 and, under a norm, a sum of up to 256 squares and four more roundings: 2^-20 (|a| + |b|) covers them; a bf16 result adds 2^-8.
Attention: a weight e^(s-m) is off, relatively, by the error of s: D products summed in f32, |q| |k| scale <= about 30
in these tests times 2^-23 for each of a few partial sums, below 2e-5. That error is multiplied with sum w |v| (`mag`), as is the rounding of
the weights to bf16 (2^-8) where the header says that they are rounded; a bf16 output adds 2^-8 |out|. The log-sum-exp is off by the
error of s plus that of a logarithm."""
import numpy as np
import pytest

from paged_util import HostCache, attention, from_bf16, to_bf16, turn

pytestmark = pytest.mark.gpu

W = 2e-5


def close(got, want, tol):
    got = np.asarray(got, dtype=np.float64)
    assert np.all(np.isfinite(got)), "not finite"
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} values off, worst {np.max(np.abs(got - want) - tol)} over"


def same_lse(got, want):
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    f = np.isfinite(want)
    assert np.all(np.abs(got[f] - want[f]) <= W + 2.0 ** -22 * np.abs(want[f]))


def upload(lthn, x, f32):
    """The values as the device holds them, and the buffer."""
    if f32:
        x = np.ascontiguousarray(x, dtype=np.float32)
        return x, lthn.Buf.from_array(x)
    b = to_bf16(x)
    return from_bf16(b), lthn.Buf.from_array(b)


def fetch(buf, shape, f32):
    return buf.download(np.float32, shape) if f32 else from_bf16(buf.download(np.uint16, shape))


# ------------------------------------------------------------------------------------------------ append ----

APPEND = [
    # D, kv, G, page, f32 in, f32 q out, norms, interleaved, rotary, head-major, rows, far
    (128, 2, 2, 16, False, False, "", False, 128, False, 1, 0),
    (128, 2, 3, 16, True, True, "qk", False, 128, False, 37, 5),
    (256, 4, 2, 24, True, False, "qk", True, 256, True, 19, 131000),
    (64, 1, 5, 1, False, True, "k", False, 32, False, 33, 1000),
    (64, 3, 1, 7, True, True, "q", True, 64, True, 70, 3),
    (128, 1, 0, 64, False, False, "k", False, 128, False, 130, 200000),   # no queries
    (256, 1, 16, 100, False, False, "", True, 2, False, 5, 77),
    (128, 16, 2, 32, True, True, "qk", False, 0, False, 12, 9),           # norm alone
]


@pytest.mark.parametrize("D,kv,G,page,fin,fq,norms,inter,rotary,major,rows,far", APPEND)
def test_append(lthn, D, kv, G, page, fin, fq, norms, inter, rotary, major, rows, far):
    rng = np.random.default_rng(rows + D)
    S, Hq = 3, kv * G
    lens = [far + (rows + 2) // 3] * S if far < 5000 else [rows // 2, 1, rows]
    c = HostCache(rng, lens, page, kv, D, major, room=rows)
    seq = rng.integers(0, S, rows).astype(np.int32)
    pos = np.zeros(rows, dtype=np.int32)
    fill = list(lens)
    for r in range(rows):
        pos[r] = fill[seq[r]]
        fill[seq[r]] += 1
    if far >= 5000:                                        # far positions by way of a sparse table: the same pages, moved back
        shift = far // page
        table = np.full((S, c.table_stride + shift), -1, dtype=np.int32)
        table[:, shift:] = c.table
        c.table, c.table_stride = table, table.shape[1]
        pos = pos + np.int32(shift * page)
    seq[rows // 2] = -1 if rows > 4 else seq[rows // 2]    # a padding row
    keep = seq >= 0
    width = (Hq + 2 * kv) * D
    x, xb = upload(lthn, rng.standard_normal((rows, width + 8)) * 2, fin)      # one projection, rows 8 elements apart
    size = 4 if fin else 2
    part = lambda o: type("P", (), {"data_ptr": lambda self: xb.ptr + o * D * size})()  # noqa: E731
    q, k, v = (x[:, a * D:b * D].reshape(rows, -1, D) for a, b in ((0, Hq), (Hq, Hq + kv), (Hq + kv, Hq + 2 * kv)))
    inv = lthn.rope_inv_freq(10000.0, D, rotary) if rotary else None
    wq, wk = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32), (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    up = lambda a: None if a is None else lthn.Buf.from_array(a)  # noqa: E731
    rope = lthn.rope_params(up(inv), rotary, inter, up(wq) if "q" in norms else None, up(wk) if "k" in norms else None, 1e-5)
    mark = to_bf16(np.full((rows, max(Hq, 1), D), 3.0)) if not fq else np.full((rows, max(Hq, 1), D), 3.0, dtype=np.float32)
    qo = lthn.Buf.from_array(mark)
    dev = c.device(lthn)
    lthn.paged_kv_append(dev, part(Hq), part(Hq + kv), up(seq), up(pos), rows, lthn.F32 if fin else lthn.BF16, rope=rope,
                         q=part(0) if Hq else None, q_heads=Hq, q_out=qo, out_dtype=lthn.F32 if fq else lthn.BF16, q_stride=width + 8,
                         k_stride=width + 8, v_stride=width + 8)
    lthn.sync()
    assert lthn.device_status() == 0
    kp, vp = (b.download(np.uint16, c.k.shape) for b in dev._keep[:2])
    page_of, off = c.table[seq[keep], pos[keep] // page], pos[keep] % page

    def reach(a):      # what the errors of a rotated pair are relative to
        return np.abs(turn(np.abs(a), pos * 0, None)) + np.abs(a).max(-1, keepdims=True)

    want_k = turn(k, pos, inv, inter, wk if "k" in norms else None, 1e-5)[keep]
    got_k, got_v = from_bf16(c.rows(kp)[page_of, off]), from_bf16(c.rows(vp)[page_of, off])
    close(got_k, want_k, 2.0 ** -8 * np.abs(want_k) + 2.0 ** -20 * reach(want_k))
    assert np.array_equal(c.rows(vp)[page_of, off], to_bf16(v[keep]))
    # everything else as it was
    untouched = np.ones(c.rows(c.k).shape[:2], dtype=bool)
    untouched[page_of, off] = False
    assert np.array_equal(c.rows(kp)[untouched], c.rows(c.k)[untouched])
    assert np.array_equal(c.rows(vp)[untouched], c.rows(c.v)[untouched])
    if Hq:
        got = fetch(qo, (rows, Hq, D), fq)
        want = turn(q, pos, inv, inter, wq if "q" in norms else None, 1e-5)
        close(got[keep], want[keep], (0 if fq else 2.0 ** -8) * np.abs(want[keep]) + 2.0 ** -20 * reach(want[keep]))
        assert np.all(got[~keep] == 3.0)


@pytest.mark.parametrize("D,kv,G,page,fin,fq,norms,inter,rotary,major,rows,far", [
    (128, 16, 2, 32, False, False, "qk", False, 128, False, 400, 50),     # more rows than are shared between blocks
    (256, 8, 8, 16, True, True, "q", True, 192, True, 150, 4000),
    (64, 12, 8, 24, False, True, "k", False, 64, False, 310, 9),
])
def test_append_blocks_of_several_passes(lthn, D, kv, G, page, fin, fq, norms, inter, rotary, major, rows, far):
    test_append(lthn, D, kv, G, page, fin, fq, norms, inter, rotary, major, rows, far)


def test_append_in_place_queries(lthn):
    rng = np.random.default_rng(1)
    rows, kv, Hq, D = 9, 2, 4, 128
    c = HostCache(rng, [rows], 16, kv, D)
    x, b = upload(lthn, rng.standard_normal((rows, (Hq + 2 * kv) * D)), False)
    at = lambda o: type("P", (), {"data_ptr": lambda self: b.ptr + o * D * 2})()  # noqa: E731
    inv = lthn.rope_inv_freq(10000.0, D)
    pos = np.arange(rows, dtype=np.int32)
    st = (Hq + 2 * kv) * D
    lthn.paged_kv_append(c.device(lthn), at(Hq), at(Hq + kv), lthn.Buf.from_array(pos * 0), lthn.Buf.from_array(pos), rows, lthn.BF16,
                         rope=lthn.rope_params(lthn.Buf.from_array(inv), D), q=at(0), q_heads=Hq, q_out=at(0), q_stride=st, k_stride=st, v_stride=st,
                         q_out_stride=st)
    got = from_bf16(b.download(np.uint16, x.shape))
    want = turn(x[:, :Hq * D].reshape(rows, Hq, D), pos, inv)
    close(got[:, :Hq * D].reshape(rows, Hq, D), want, 2.0 ** -8 * np.abs(want) + 1e-5)
    assert np.array_equal(got[:, Hq * D:], x[:, Hq * D:])


@pytest.mark.parametrize("what", ["page below", "page above", "position below", "position above", "sequence"])
def test_append_reports_indices_outside_the_table(lthn, what):
    """Such a row is not stored and the status word says so; the other rows are."""
    rng = np.random.default_rng(2)
    c = HostCache(rng, [20, 20], 8, 2, 64)
    seq, pos = np.array([0, 1, 1], dtype=np.int32), np.array([3, 9, 17], dtype=np.int32)
    if what == "page below":
        c.table[1, 1] = -1
    elif what == "page above":
        c.table[1, 1] = c.pages
    elif what == "position below":
        pos[1] = -1
    elif what == "position above":
        pos[1] = c.table_stride * c.ps
    else:
        seq[1] = 2
    x, b = upload(lthn, rng.standard_normal((3, 2, 64)), False)
    dev = c.device(lthn)
    lthn.paged_kv_append(dev, b, b, lthn.Buf.from_array(seq), lthn.Buf.from_array(pos), 3, lthn.BF16)
    with pytest.raises(lthn.LthnError) as e:
        lthn.device_status()
    assert e.value.code == 1
    assert lthn.device_status() == 0          # read and cleared
    for r in (0, 2):
        c.put(seq[r], pos[r:r + 1], x[r:r + 1], x[r:r + 1])
    assert np.array_equal(dev._keep[0].download(np.uint16, c.k.shape), c.k)
    assert np.array_equal(dev._keep[1].download(np.uint16, c.v.shape), c.v)


# ------------------------------------------------------------------------------------------------ decode ----

def options(lthn, rng, Hq, lens, softcap=0.0, slopes=False, window=0, prefix=0, scale=0.0):
    """The options and the same as keywords of the 64-bit form (per sequence)."""
    sl = (2.0 ** -rng.uniform(1, 8, Hq)).astype(np.float32) if slopes else None
    pre = np.minimum(np.asarray(lens), prefix).astype(np.int32) if prefix else None
    o = lthn.attn_options(scale, softcap, None if sl is None else lthn.Buf.from_array(sl), window, None if pre is None else lthn.Buf.from_array(pre))
    return o, [dict(scale=scale or None, softcap=softcap, slopes=sl, window=window, prefix=0 if pre is None else int(pre[s])) for s in range(len(lens))]


def run_decode(lthn, c, q, f32, opts=None, stream=None, lens=None, stride=0, ws=None):
    rows, Hq, D = q.shape
    x, qb = upload(lthn, q, f32)
    out, lse = lthn.Buf(rows * Hq * D * 4), lthn.Buf(rows * Hq * 4)
    dt = lthn.F32 if f32 else lthn.BF16
    dev = c.device(lthn)
    ws = ws or lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, rows, Hq, dt))
    lthn.paged_sdpa_decode(dev, qb, dt, lthn.Buf.from_array(np.asarray(c.lens if lens is None else lens, dtype=np.int32)), rows, Hq, out, ws,
                           options=opts, lse=lse, stream=stream)
    lthn.sync()
    assert lthn.device_status() == 0
    return x, fetch(out, (rows, Hq, D), f32), lse.download(np.float32, (rows, Hq))


def check_decode(lthn, c, q, f32, opts=None, kws=None):
    x, got, lse = run_decode(lthn, c, q, f32, opts)
    G = q.shape[1] // c.kv
    rounded = 0.0 if f32 else 2.0 ** -8
    for r, n in enumerate(c.lens):
        want, wl, mag = attention(c, r, x[r:r + 1], n - 1, n, **(kws[r] if kws else {}))
        close(got[r:r + 1], want, rounded * np.abs(want) + (W + (rounded if G > 8 else 0.0)) * mag + (2.0 ** -23) * np.abs(want))
        same_lse(lse[r:r + 1], wl)


DECODE = [
    # D, kv, G, page, f32, head-major, lens
    (128, 2, 2, 16, False, False, [1]),
    (128, 2, 2, 16, True, False, [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129]),
    (64, 1, 1, 1, True, False, [0, 1, 333, 64]),
    (64, 3, 5, 24, False, True, [200, 0, 0, 511, 7]),
    (256, 4, 2, 16, True, False, [1279]),
    (256, 1, 8, 100, False, False, [700, 64, 1]),
    (256, 2, 16, 32, False, True, [65, 300]),
    (128, 1, 16, 8, False, False, [1025]),
    (128, 2, 17, 64, False, False, [130, 5]),
    (128, 1, 12, 128, True, False, [257, 1]),
    (128, 8, 4, 7, True, True, [50, 999, 64]),
    (64, 16, 1, 256, False, False, [256, 255, 257]),
]


@pytest.mark.parametrize("D,kv,G,page,f32,major,lens", DECODE)
def test_decode(lthn, D, kv, G, page, f32, major, lens):
    rng = np.random.default_rng(len(lens) + D + G)
    c = HostCache(rng, lens, page, kv, D, major)
    check_decode(lthn, c, rng.standard_normal((len(lens), kv * G, D)), f32)


MASKS = [dict(window=1), dict(window=64), dict(window=100, prefix=10), dict(prefix=5000), dict(softcap=30.0), dict(slopes=True), dict(scale=0.3),
         dict(softcap=5.0, slopes=True, window=70, prefix=64, scale=0.5)]


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("D,kv,G,f32", [(128, 2, 3, True), (64, 2, 9, False), (256, 1, 4, False)])
def test_decode_masks(lthn, mask, D, kv, G, f32):
    rng = np.random.default_rng(7)
    lens = [400, 1, 0, 99, 64, 163]
    c = HostCache(rng, lens, 24, kv, D)
    o, kws = options(lthn, rng, kv * G, lens, **mask)
    check_decode(lthn, c, rng.standard_normal((len(lens), kv * G, D)), f32, o, kws)


def widen(c, rows):
    """The same cache under a table with room for `rows` more rows a sequence: how a call is dealt out depends on the longest row it can have."""
    more = (rows + c.ps - 1) // c.ps
    c.table = np.ascontiguousarray(np.hstack([c.table, np.full((len(c.lens), more), -7, dtype=np.int32)]))
    c.table_stride += more
    return c


@pytest.mark.parametrize("D,kv,G,page,f32,major,lens", DECODE)
def test_decode_under_a_wide_table(lthn, D, kv, G, page, f32, major, lens):
    rng = np.random.default_rng(len(lens) + D + G)
    c = widen(HostCache(rng, lens, page, kv, D, major), 1 << 17)
    check_decode(lthn, c, rng.standard_normal((len(lens), kv * G, D)), f32)


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("D,kv,G,f32,rows", [(128, 1, 3, True, 1 << 17), (64, 1, 9, False, 1 << 17), (256, 1, 4, False, 0)])
def test_decode_masks_few_rows(lthn, mask, D, kv, G, f32, rows):
    rng = np.random.default_rng(34)
    lens = [400, 1, 0, 99, 64, 163, 1023]
    c = widen(HostCache(rng, lens, 24, kv, D), rows)
    o, kws = options(lthn, rng, kv * G, lens, **mask)
    check_decode(lthn, c, rng.standard_normal((len(lens), kv * G, D)), f32, o, kws)


def test_decode_many_rows_and_one_long(lthn):
    """More rows than a block scans at once; one row far longer than the others is cut over many blocks."""
    rng = np.random.default_rng(11)
    lens = [int(n) for n in rng.integers(0, 90, 300)]
    lens[137] = 20011
    lens[299] = 1
    c = HostCache(rng, lens, 16, 1, 64)
    check_decode(lthn, c, rng.standard_normal((300, 2, 64)), True)


def test_decode_one_row_over_the_whole_gpu(lthn):
    rng = np.random.default_rng(12)
    c = HostCache(rng, [60001], 64, 1, 64)
    check_decode(lthn, c, rng.standard_normal((1, 4, 64)), False)


def test_decode_extreme_scores(lthn):
    """Scores of some hundreds: one key takes all the weight, and the maximum is what keeps the exponentials finite."""
    rng = np.random.default_rng(13)
    c = HostCache(rng, [300, 65], 16, 2, 64)
    q = rng.standard_normal((2, 4, 64)) * 300
    x, got, lse = run_decode(lthn, c, q, True)
    for r, n in enumerate(c.lens):
        want, wl, mag = attention(c, r, x[r:r + 1], n - 1, n)
        # |q| |k| scale is 300 times larger here, and so is the error of a score
        close(got[r:r + 1], want, 300 * W * mag)
        assert np.all(np.abs(lse[r] - wl[0]) <= 300 * W)


def test_decode_bad_pages_are_reported(lthn):
    rng = np.random.default_rng(14)
    c = HostCache(rng, [100, 40], 16, 2, 64)
    c.table[0, 3] = c.pages + 5
    q, qb = upload(lthn, rng.standard_normal((2, 4, 64)), False)
    dev, out = c.device(lthn), lthn.Buf(2 * 4 * 64 * 2)
    ws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, 2, 4, lthn.BF16))
    for lens in ([100, 40], [0, 10 ** 6]):      # a bad page; a length behind the table
        lthn.paged_sdpa_decode(dev, qb, lthn.BF16, lthn.Buf.from_array(np.array(lens, dtype=np.int32)), 2, 4, out, ws)
        with pytest.raises(lthn.LthnError) as e:
            lthn.device_status()
        assert e.value.code == 1
    lthn.paged_sdpa_decode(dev, qb, lthn.BF16, lthn.Buf.from_array(np.array([48, 40], dtype=np.int32)), 2, 4, out, ws)
    assert lthn.device_status() == 0            # the bad page is behind the length: nobody needs it


def test_decode_bad_pages_and_strided_rows_under_a_wide_table(lthn):
    """The refusals and the layout of the two tests beside this one where a call is dealt out over the whole GPU."""
    rng = np.random.default_rng(35)
    kv, G, D, rows = 2, 2, 64, 3
    Hq = kv * G
    c = widen(HostCache(rng, [100, 0, 470], 16, kv, D), 1 << 17)
    q = np.full((rows, Hq * D + 16), np.nan)
    q[:, :Hq * D] = rng.standard_normal((rows, Hq * D))
    x, qb = upload(lthn, q, False)
    dev = c.device(lthn)
    out = lthn.Buf.from_array(to_bf16(np.full((rows + 1, Hq * D + 24), 7.0)))
    ws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, rows, Hq, lthn.BF16))

    def run(lens):
        lthn.paged_sdpa_decode(dev, qb, lthn.BF16, lthn.Buf.from_array(np.array(lens, dtype=np.int32)), rows, Hq, out, ws, q_stride=Hq * D + 16,
                               out_stride=Hq * D + 24)
    for lens in ([116, 0, 470], [100, 10 ** 6, 470]):        # an entry that is no page; a length behind the table
        run(lens)
        with pytest.raises(lthn.LthnError) as e:
            lthn.device_status()
        assert e.value.code == 1
    run(c.lens)
    assert lthn.device_status() == 0
    got = from_bf16(out.download(np.uint16, (rows + 1, Hq * D + 24)))
    assert np.all(got[:, Hq * D:] == 7.0) and np.all(got[rows] == 7.0)
    for r, n in enumerate(c.lens):
        want, _, mag = attention(c, r, x[r:r + 1, :Hq * D].reshape(1, Hq, D), n - 1, n)
        close(got[r, :Hq * D].reshape(1, Hq, D), want, 2.0 ** -8 * np.abs(want) + W * mag)


def test_decode_strided_rows_leave_the_rest(lthn):
    rng = np.random.default_rng(15)
    rows, kv, G, D = 3, 2, 2, 64
    Hq = kv * G
    c = HostCache(rng, [30, 0, 70], 8, kv, D)
    q = np.full((rows, Hq * D + 16), np.nan)
    q[:, :Hq * D] = rng.standard_normal((rows, Hq * D))
    x, qb = upload(lthn, q, False)
    out = lthn.Buf.from_array(to_bf16(np.full((rows + 1, Hq * D + 24), 7.0)))
    dev = c.device(lthn)
    ws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, rows, Hq, lthn.BF16))
    lthn.paged_sdpa_decode(dev, qb, lthn.BF16, lthn.Buf.from_array(np.array(c.lens, dtype=np.int32)), rows, Hq, out, ws, q_stride=Hq * D + 16,
                           out_stride=Hq * D + 24)
    got = from_bf16(out.download(np.uint16, (rows + 1, Hq * D + 24)))
    assert np.all(got[:, Hq * D:] == 7.0) and np.all(got[rows] == 7.0)
    for r, n in enumerate(c.lens):
        want, _, mag = attention(c, r, x[r:r + 1, :Hq * D].reshape(1, Hq, D), n - 1, n)
        close(got[r, :Hq * D].reshape(1, Hq, D), want, 2.0 ** -8 * np.abs(want) + W * mag)


def test_host_memory_is_refused(lthn):
    """A host address where device memory belongs is an error of the call, not of the kernel."""
    c = HostCache(np.random.default_rng(16), [10], 8, 1, 64)
    dev = c.device(lthn)
    host = np.zeros(4096, dtype=np.uint16)
    b = lthn.Buf(1 << 20)
    dev.desc.k = (host.ctypes.data + 15) & ~15
    n = lthn.Buf.from_array(np.array([10], dtype=np.int32))
    for call in (lambda: lthn.paged_sdpa_decode(dev, b, lthn.BF16, n, 1, 1, b, lthn.Buf(8 << 20)),
                 lambda: lthn.paged_kv_append(dev, b, b, n, n, 1, lthn.BF16),
                 lambda: lthn.paged_prefill_attention(dev, b, n, n, 1, 1, 1, b, lthn.Buf(8 << 20))):
        with pytest.raises(lthn.LthnError) as e:
            call()
        assert e.value.code == 1


# ----------------------------------------------------------------------------------------------- prefill ----

def run_prefill(lthn, c, q, new, opts=None, ctx=0, gap=0, ws=None):
    """q [total, Hq, D]; sequence s owns the next new[s] rows, behind `gap` rows that nobody owns."""
    total, Hq, D = q.shape
    x, qb = upload(lthn, q, False)
    out = lthn.Buf.from_array(to_bf16(np.full((total, Hq, D), 5.0)))
    lse = lthn.Buf.from_array(np.full((total, Hq), 5.0, dtype=np.float32))
    start = gap + np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    dev = c.device(lthn)
    ws = ws or lthn.Buf(lthn.paged_prefill_attention_workspace(dev, len(new), total, Hq, ctx))
    lthn.paged_prefill_attention(dev, qb, lthn.Buf.from_array(start.astype(np.int32)), lthn.Buf.from_array(np.array(c.lens, dtype=np.int32)), len(new),
                                 total, Hq, out, ws, max_ctx=ctx, options=opts, lse=lse)
    lthn.sync()
    assert lthn.device_status() == 0
    return x, from_bf16(out.download(np.uint16, (total, Hq, D))), lse.download(np.float32, (total, Hq)), start


def check_prefill(lthn, c, q, new, opts=None, kws=None, ctx=0, gap=0):
    x, got, lse, start = run_prefill(lthn, c, q, new, opts, ctx, gap)
    for s, n in enumerate(c.lens):
        rows = slice(start[s], start[s + 1])
        want, wl, mag = attention(c, s, x[rows], n - new[s], n, **(kws[s] if kws else {}))
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag)
        same_lse(lse[rows], wl)
    for rest in (got[:start[0]], got[start[-1]:], lse[:start[0]], lse[start[-1]:]):
        assert np.all(rest == 5.0)


PREFILL = [
    # D, kv, G, page, head-major, new, past
    (128, 1, 1, 16, False, [1], [0]),
    (128, 2, 2, 16, False, [130], [0]),
    (128, 2, 2, 32, False, [64, 1, 0, 33], [0, 100, 5, 64]),
    (64, 3, 3, 24, True, [77, 128, 129], [0, 0, 1]),
    (64, 1, 16, 1, False, [9, 20], [300, 0]),
    (256, 2, 2, 16, False, [200], [50]),
    (256, 1, 7, 100, True, [31, 5, 64], [0, 700, 63]),
    (128, 4, 8, 64, False, [3, 4, 1], [1000, 20, 0]),
    (128, 1, 96, 8, False, [5], [40]),
    (128, 2, 1, 128, False, [513], [127]),
    (64, 2, 2, 7, False, [300, 299], [11, 500]),
    (256, 1, 1, 16, False, [1, 1, 1], [0, 63, 64]),
]


@pytest.mark.parametrize("D,kv,G,page,major,new,past", PREFILL)
def test_prefill(lthn, D, kv, G, page, major, new, past):
    rng = np.random.default_rng(sum(new) + D)
    c = HostCache(rng, [a + b for a, b in zip(new, past)], page, kv, D, major)
    check_prefill(lthn, c, rng.standard_normal((sum(new), kv * G, D)), new)


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("D,kv,G", [(128, 2, 2), (64, 1, 3), (256, 1, 2)])
def test_prefill_masks(lthn, mask, D, kv, G):
    rng = np.random.default_rng(8)
    new, past = [150, 1, 70, 64], [0, 200, 130, 400]
    lens = [a + b for a, b in zip(new, past)]
    c = HostCache(rng, lens, 16, kv, D)
    o, kws = options(lthn, rng, kv * G, lens, **mask)
    check_prefill(lthn, c, rng.standard_normal((sum(new), kv * G, D)), new, o, kws)


@pytest.mark.parametrize("D,kv,G", [(128, 1, 2), (64, 2, 1), (256, 1, 1)])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("new", [[400], [30, 90]])
def test_prefill_growing_scores(lthn, D, kv, G, page, new):
    """Keys that grow along the sequence: the running maximum moves again and again, and what was summed before is scaled down."""
    rng = np.random.default_rng(25)
    past = [500, 333][:len(new)]
    lens = [a + b for a, b in zip(new, past)]
    c = HostCache(rng, lens, page, kv, D)
    for s, n in enumerate(lens):
        k, v = c.get(s, n)
        c.put(s, np.arange(n), k * (0.2 + np.arange(n)[:, None, None] / 150.0), v)
    q = rng.standard_normal((sum(new), kv * G, D))
    x, got, lse, start = run_prefill(lthn, c, q, new)
    for s, n in enumerate(lens):
        rows = slice(start[s], start[s + 1])
        want, wl, mag = attention(c, s, x[rows], n - new[s], n)
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 8 * W) * mag)      # |k| is up to 6 times larger, and so are the errors of s
        assert np.all(np.abs(lse[rows] - wl) <= 8 * W + 2.0 ** -22 * np.abs(wl))


def test_prefill_many_sequences(lthn):
    rng = np.random.default_rng(21)
    new = [int(n) for n in rng.integers(0, 7, 300)]
    past = [int(n) for n in rng.integers(0, 40, 300)]
    c = HostCache(rng, [a + b for a, b in zip(new, past)], 8, 1, 64)
    check_prefill(lthn, c, rng.standard_normal((sum(new), 2, 64)), new)


@pytest.mark.parametrize("D,kv,G,new,past", [(128, 1, 2, [5, 3], [9000, 4000]), (64, 1, 4, [17], [20000]), (256, 1, 1, [2], [5001])])
@pytest.mark.parametrize("ctx", [0, 100, 30000])
def test_prefill_few_rows_long_axis(lthn, D, kv, G, new, past, ctx):
    """Also with a bound on the lengths that is too small: it only chooses how the work is cut."""
    rng = np.random.default_rng(22)
    c = HostCache(rng, [a + b for a, b in zip(new, past)], 64, kv, D)
    check_prefill(lthn, c, rng.standard_normal((sum(new), kv * G, D)), new, ctx=ctx)


@pytest.mark.parametrize("mask", [{}, dict(slopes=True), dict(slopes=True, window=333, prefix=40)], ids=str)
@pytest.mark.parametrize("D,kv,G,seqs", [(128, 1, 4, 2), (64, 2, 1, 5), (256, 1, 2, 3), (64, 1, 2, 32), (128, 1, 2, 33)])
@pytest.mark.parametrize("ctx", [0, 20000])
def test_prefill_chunks_of_unlike_lengths(lthn, mask, D, kv, G, seqs, ctx):
    """Sequences of one to several row tiles on contexts of none to thousands of keys: where their keys are cut depends on the lengths and on
    their number."""
    rng = np.random.default_rng(27 + seqs)
    new = [int(n) for n in rng.integers(1, 12 if seqs > 5 else 300, seqs)]
    past = [int(n) for n in 2.0 ** rng.uniform(0, 9 if seqs > 5 else 12, seqs)]
    lens = [a + b for a, b in zip(new, past)]
    c = HostCache(rng, lens, 16, kv, D)
    o, kws = options(lthn, rng, kv * G, lens, **mask)
    check_prefill(lthn, c, rng.standard_normal((sum(new), kv * G, D)), new, o, kws, ctx=ctx)


def test_prefill_rows_nobody_owns_and_rows_before_the_first_position(lthn):
    rng = np.random.default_rng(23)
    new, lens = [10, 6, 4], [4, 6, 0]          # sequence 0 has more queries than positions, sequence 2 has none at all
    c = HostCache(rng, lens, 4, 1, 64)
    q = rng.standard_normal((sum(new) + 9, 2, 64))
    check_prefill(lthn, c, q, new, gap=4)


def test_prefill_reports_a_bad_plan(lthn):
    rng = np.random.default_rng(24)
    c = HostCache(rng, [40, 40], 16, 1, 64)
    q, qb = upload(lthn, rng.standard_normal((30, 2, 64)), False)
    dev = c.device(lthn)
    out, ws = lthn.Buf(30 * 2 * 64 * 2), lthn.Buf(lthn.paged_prefill_attention_workspace(dev, 2, 30, 2))
    for start, lens, page in (([0, 20, 10], [40, 40], 0), ([0, 10, 31], [40, 40], 0), ([-1, 10, 20], [40, 40], 0), ([0, 10, 20], [40, 49], 0),
                              ([0, 10, 20], [40, 40], c.pages)):
        t = c.table.copy()
        if page:
            t[1, 2] = page
        dev._keep[2].upload(t)
        lthn.paged_prefill_attention(dev, qb, lthn.Buf.from_array(np.array(start, dtype=np.int32)), lthn.Buf.from_array(np.array(lens, dtype=np.int32)),
                                     2, 30, 2, out, ws)
        with pytest.raises(lthn.LthnError) as e:
            lthn.device_status()
        assert e.value.code == 1


# ---------------------------------------------------------------------------------------------- together ----

def test_serving_run_matches_the_dense_path(lthn):
    """Two conversations in a paged cache: prompts appended and attended, then three tokens each; the same through the dense
    cache's kernels (lthn_prefill_attention, lthn_sdpa_decode) and in 64 bits."""
    rng = np.random.default_rng(31)
    kv, G, D, page = 2, 2, 128, 16
    Hq = kv * G
    prompts, steps = [70, 45], 3
    final = [n + steps for n in prompts]
    c = HostCache(rng, [0, 0], page, kv, D, room=max(final))
    dev = c.device(lthn)
    inv = lthn.rope_inv_freq(10000.0, D)
    nq, nk = (np.float32(1) + 0.1 * rng.standard_normal(D).astype(np.float32) for _ in range(2))
    rope = lthn.rope_params(lthn.Buf.from_array(inv), D, False, lthn.Buf.from_array(nq), lthn.Buf.from_array(nk))
    out = lthn.Buf(max(prompts) * 2 * Hq * D * 4)

    def append(seq, pos, f32):
        n = len(seq)
        x, b = upload(lthn, rng.standard_normal((n, Hq + 2 * kv, D)), f32)
        st, size = (Hq + 2 * kv) * D, 4 if f32 else 2
        at = lambda o: type("P", (), {"data_ptr": lambda self: b.ptr + o * D * size})()  # noqa: E731
        qo = lthn.Buf(n * Hq * D * size)
        seq, pos = np.array(seq, dtype=np.int32), np.array(pos, dtype=np.int32)
        dt = lthn.F32 if f32 else lthn.BF16
        lthn.paged_kv_append(dev, at(Hq), at(Hq + kv), lthn.Buf.from_array(seq), lthn.Buf.from_array(pos), n, dt, rope=rope, q=at(0), q_heads=Hq,
                             q_out=qo, q_stride=st, k_stride=st, v_stride=st)
        lthn.sync()
        c.k, c.v = (p.download(np.uint16, c.k.shape) for p in dev._keep[:2])
        want = turn(x[:, Hq:Hq + kv], pos, inv, False, nk)
        got = from_bf16(c.k[c.table[seq, pos // page], pos % page])
        close(got, want, 2.0 ** -8 * np.abs(want) + 1e-5)
        return qo, fetch(qo, (n, Hq, D), f32)

    seq = [0] * prompts[0] + [1] * prompts[1]
    pos = list(range(prompts[0])) + list(range(prompts[1]))
    qb, q = append(seq, pos, False)
    start = np.array([0, prompts[0], sum(prompts)], dtype=np.int32)
    lens = lthn.Buf.from_array(np.array(prompts, dtype=np.int32))
    ws = lthn.Buf(lthn.paged_prefill_attention_workspace(dev, 2, sum(prompts), Hq))
    lthn.paged_prefill_attention(dev, qb, lthn.Buf.from_array(start), lens, 2, sum(prompts), Hq, out, ws)
    lthn.sync()
    got = from_bf16(out.download(np.uint16, (sum(prompts), Hq, D)))
    dense_out = lthn.Buf(max(prompts) * Hq * D * 2)
    for s in range(2):
        rows = slice(start[s], start[s + 1])
        want, _, mag = attention(c, s, q[rows], 0, prompts[s])
        close(got[rows], want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag)
        k, v = c.get(s, prompts[s])
        lthn.prefill_attention(lthn.Buf.from_array(q[rows].astype(np.float32)), lthn.Buf.from_array(to_bf16(k)), lthn.Buf.from_array(to_bf16(v)), dense_out,
                               prompts[s], 0, Hq, kv, D)
        lthn.sync()
        dense = from_bf16(dense_out.download(np.uint16, (prompts[s], Hq, D)))
        close(got[rows], dense, 2 * (2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag))     # each of the two may be that far off
    dws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, 2, Hq, lthn.F32))
    for t in range(steps):
        now = [n + t for n in prompts]
        qb, q = append([0, 1], now, True)
        lens = lthn.Buf.from_array(np.array(now, dtype=np.int32) + 1)
        lthn.paged_sdpa_decode(dev, qb, lthn.F32, lens, 2, Hq, out, dws)
        lthn.sync()
        got = out.download(np.float32, (2, Hq, D))
        lane = max(now) + 1
        dense = np.zeros((2, 2, lane, kv, D), dtype=np.uint16)
        for s in range(2):
            want, _, mag = attention(c, s, q[s:s + 1], now[s], now[s] + 1)
            close(got[s:s + 1], want, W * mag)
            k, v = c.get(s, now[s] + 1)
            dense[0, s, :now[s] + 1], dense[1, s, :now[s] + 1] = to_bf16(k), to_bf16(v)
        do = lthn.Buf(2 * Hq * D * 4)
        kb, vb = lthn.Buf.from_array(dense[0]), lthn.Buf.from_array(dense[1])
        rp, rl = lthn.Buf.from_array(np.array(now, dtype=np.int32)), lthn.Buf.from_array(np.arange(2, dtype=np.int32))
        lthn.check(lthn.lib().lthn_sdpa_decode(None, qb.ptr, kb.ptr, vb.ptr, rp.ptr, rl.ptr, do.ptr, 2, Hq, kv, D, lane * kv * D, 0.0, lane))
        lthn.sync()
        close(got, do.download(np.float32, (2, Hq, D)), 4e-5 * (1 + np.abs(got)))
    assert lthn.device_status() == 0


def test_captured_steps_replay_with_new_lengths(lthn):
    """A captured append and decode reads positions and lengths on the device; two graphs with a workspace each run on two streams at once."""
    rng = np.random.default_rng(32)
    kv, G, D, page, rows = 2, 4, 64, 8, 5
    Hq = kv * G
    c = HostCache(rng, [90, 10, 0, 33, 200], page, kv, D, room=8)
    dev = c.device(lthn)
    inv = lthn.rope_inv_freq(10000.0, D)
    rope = lthn.rope_params(lthn.Buf.from_array(inv), D)
    seq = lthn.Buf.from_array(np.arange(rows, dtype=np.int32))
    spare = HostCache(rng, [8] * rows, page, kv, D).device(lthn)   # first uses outside the captures, where nothing here is written
    lanes = []
    for appends in (True, False):
        st = lthn.Stream()
        w = dict(x=lthn.Buf(rows * Hq * D * 2), kv=lthn.Buf(rows * kv * D * 2), qo=lthn.Buf(rows * Hq * D * 2), out=lthn.Buf(rows * Hq * D * 2),
                 pos=lthn.Buf(rows * 4), lens=lthn.Buf(rows * 4), ws=lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, rows, Hq, lthn.BF16)))
        for b in ("x", "kv", "qo", "pos", "lens"):
            w[b].zero()
        lthn.sync()

        def step(cache):
            if appends:
                lthn.paged_kv_append(cache, w["kv"], w["kv"], seq, w["pos"], rows, lthn.BF16, rope=rope, q=w["x"], q_heads=Hq, q_out=w["qo"], stream=st)
            lthn.paged_sdpa_decode(cache, w["qo"], lthn.BF16, w["lens"], rows, Hq, w["out"], w["ws"], stream=st)
        step(spare)
        st.sync()
        w["graph"] = lthn.Graph(st)
        with w["graph"]:
            step(dev)
        lanes.append(w)
    now = np.array(c.lens, dtype=np.int32)
    for t in range(3):
        a, b = lanes
        xq = to_bf16(rng.standard_normal((rows, Hq, D)))
        a["kv"].upload(to_bf16(rng.standard_normal((rows, kv, D))))
        a["x"].upload(xq)
        a["pos"].upload(now)
        a["lens"].upload(now + 1)
        q2 = to_bf16(rng.standard_normal((rows, Hq, D)))
        b["qo"].upload(q2)
        b["lens"].upload(now)                    # only rows that were there before: independent of the append beside it
        a["graph"].launch()
        b["graph"].launch()
        lthn.sync()
        got_b = from_bf16(b["out"].download(np.uint16, (rows, Hq, D)))
        for r in range(rows):
            want, _, mag = attention(c, r, from_bf16(q2[r:r + 1]), now[r] - 1, now[r])
            close(got_b[r:r + 1], want, 2.0 ** -8 * np.abs(want) + W * mag)
        c.k, c.v = (p.download(np.uint16, c.k.shape) for p in dev._keep[:2])
        q = from_bf16(a["qo"].download(np.uint16, (rows, Hq, D)))
        want = turn(from_bf16(xq), now, inv)
        close(q, want, 2.0 ** -8 * np.abs(want) + 1e-5)
        got = from_bf16(a["out"].download(np.uint16, (rows, Hq, D)))
        for r in range(rows):
            want, _, mag = attention(c, r, q[r:r + 1], now[r], now[r] + 1)
            close(got[r:r + 1], want, 2.0 ** -8 * np.abs(want) + W * mag)
        now = now + 1
    assert lthn.device_status() == 0


@pytest.mark.parametrize("D,G,extra", [(128, 4, 0), (64, 3, 64), (256, 2, 8)])
def test_captured_prompt_chunks_in_strided_rows(lthn, D, G, extra):
    """Queries and outputs inside wider rows, two graphs on two streams at once, replayed with other chunks and lengths: from drafts behind long
    contexts, which are cut and joined, to prompts."""
    rng = np.random.default_rng(33 + D)
    kv, page, cap, total = 2, 16, [2000, 700, 40], 310
    Hq = kv * G
    qs, os = Hq * D + extra + (D if extra % D == 0 else 0), Hq * D + 24
    c = HostCache(rng, cap, page, kv, D)
    dev = c.device(lthn)
    lanes = []
    for _ in range(2):
        st = lthn.Stream()
        w = dict(q=lthn.Buf(total * qs * 2), out=lthn.Buf(total * os * 2), start=lthn.Buf(16), lens=lthn.Buf(12),
                 ws=lthn.Buf(lthn.paged_prefill_attention_workspace(dev, 3, total, Hq)))
        for b in w.values():
            b.zero()
        lthn.sync()

        def step():
            lthn.paged_prefill_attention(dev, w["q"], w["start"], w["lens"], 3, total, Hq, w["out"], w["ws"], q_stride=qs, out_stride=os, stream=st)
        step()
        st.sync()
        w["graph"] = lthn.Graph(st)
        with w["graph"]:
            step()
        lanes.append(w)
    plans = [([4, 1, 9], [2000, 650, 40]), ([0, 270, 30], [1999, 270, 31]), ([150, 0, 2], [170, 700, 2]), ([1, 1, 1], [1, 700, 0])]
    for t in range(0, len(plans), 2):
        data = []
        for w, (new, lens) in zip(lanes, plans[t:t + 2]):
            q = np.full((total, qs), 9.0)
            q[:, :Hq * D] = rng.standard_normal((total, Hq * D))
            q = to_bf16(q)
            w["q"].upload(q)
            w["out"].upload(to_bf16(np.full((total, os), 5.0)))
            start = 3 + np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
            w["start"].upload(start)
            w["lens"].upload(np.array(lens, dtype=np.int32))
            data.append((from_bf16(q)[:, :Hq * D].reshape(total, Hq, D), start, new, lens))
        lthn.sync()
        for w in lanes:
            w["graph"].launch()
        lthn.sync()
        assert lthn.device_status() == 0
        for w, (q, start, new, lens) in zip(lanes, data):
            got = from_bf16(w["out"].download(np.uint16, (total, os)))
            assert np.all(got[:, Hq * D:] == 5.0) and np.all(got[:start[0]] == 5.0) and np.all(got[start[-1]:] == 5.0)
            for s in range(3):
                rows = slice(start[s], start[s + 1])
                want, _, mag = attention(c, s, q[rows], lens[s] - new[s], lens[s])
                close(got[rows, :Hq * D].reshape(-1, Hq, D), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag)


def test_offsets_past_32_bits(lthn):
    """Pages far apart, K and V side by side in one allocation: element offsets beyond 2^32 bytes and 2^31 elements."""
    rng = np.random.default_rng(33)
    kv, D, page, n = 1, 64, 16, 40
    far = (1 << 31) + 4096                       # elements between pages
    total = 3 * far
    buf = lthn.Buf(total * 2)
    half = far // 2                              # V half a page stride behind K
    table = np.array([[2, 0, 1]], dtype=np.int32)
    c = HostCache(rng, [n], page, kv, D, spare=0)
    where = {int(c.table[0, i]): int(table[0, i]) for i in range(3)}
    for own, at in where.items():
        for pool, off in ((c.k, 0), (c.v, half)):
            a = np.ascontiguousarray(pool[own])
            lthn.check(lthn.lib().lthn_memcpy_h2d(buf.ptr + (at * far + off) * 2, a.ctypes.data, a.nbytes, None))
    lthn.sync()
    v = type("P", (), {"data_ptr": lambda self: buf.ptr + half * 2})()
    dev = lthn.PagedKV(buf, v, lthn.Buf.from_array(table), pages=3, page_size=page, kv_heads=kv, head_dim=D, seqs=1, table_stride=3, page_stride=far)
    q, qb = upload(lthn, rng.standard_normal((1, 2, D)), True)
    out = lthn.Buf(8 * 2 * D * 4)
    ws = lthn.Buf(lthn.paged_sdpa_decode_workspace(dev, 1, 2, lthn.F32))
    lens = lthn.Buf.from_array(np.array([n], dtype=np.int32))
    lthn.paged_sdpa_decode(dev, qb, lthn.F32, lens, 1, 2, out, ws)
    lthn.sync()
    want, _, mag = attention(c, 0, q, n - 1, n)
    close(out.download(np.float32, (1, 2, D)), want, W * mag)
    q, qb = upload(lthn, rng.standard_normal((5, 2, D)), False)
    ws = lthn.Buf(lthn.paged_prefill_attention_workspace(dev, 1, 5, 2))
    lthn.paged_prefill_attention(dev, qb, lthn.Buf.from_array(np.array([0, 5], dtype=np.int32)), lens, 1, 5, 2, out, ws)
    lthn.sync()
    want, _, mag = attention(c, 0, q, n - 5, n)
    close(from_bf16(out.download(np.uint16, (5, 2, D))), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + W) * mag)
    x, xb = upload(lthn, rng.standard_normal((1, kv, D)), False)
    lthn.paged_kv_append(dev, xb, xb, lthn.Buf.from_array(np.array([0], dtype=np.int32)), lthn.Buf.from_array(np.array([5], dtype=np.int32)), 1, lthn.BF16)
    lthn.sync()
    got = np.zeros(D, dtype=np.uint16)
    lthn.check(lthn.lib().lthn_memcpy_d2h(got.ctypes.data, buf.ptr + (2 * far + half + 5 * D) * 2, got.nbytes, None))
    assert np.array_equal(from_bf16(got), x[0, 0])
    assert lthn.device_status() == 0
    buf.free()
