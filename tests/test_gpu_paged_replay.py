"""The one-token attention dealt out over the whole GPU, captured and replayed on two streams at once with a workspace each: from long
rows to short and empty ones and back, so that parts which an earlier replay left must not be taken for this one's. Tolerances: those of
test_gpu_paged.py."""
import numpy as np
import pytest

from paged_util import HostCache, attention, to_bf16
from test_gpu_paged import W, close, fetch, same_lse, upload, widen

pytestmark = pytest.mark.gpu

# f32, D, kv heads, query heads of each, the most keys of each row; the last two have more rows than a block scans at once
CASES = [(False, 64, 2, 3, [900, 70, 0, 33, 2000]), (True, 128, 1, 2, [1500, 64, 700]), (False, 128, 2, 12, [3000, 1, 129]),
         (True, 64, 1, 1, [int(n) for n in np.random.default_rng(5).integers(0, 300, 150)]), (False, 256, 1, 2, [40] * 129)]


@pytest.mark.parametrize("f32,D,kv,G,most", CASES)
def test_replays_with_other_lengths(lthn, f32, D, kv, G, most):
    rng = np.random.default_rng(91)
    rows, Hq, size, dt = len(most), kv * G, 4 if f32 else 2, lthn.F32 if f32 else lthn.BF16
    c = widen(HostCache(rng, most, 16, kv, D), 1 << 17)
    dev = c.device(lthn)
    lanes = []
    for _ in range(2):
        st = lthn.Stream()
        w = dict(q=lthn.Buf(rows * Hq * D * size), out=lthn.Buf(rows * Hq * D * size), lse=lthn.Buf(rows * Hq * 4), lens=lthn.Buf(rows * 4),
                 ws=lthn.Buf.from_array(np.full(lthn.paged_sdpa_decode_workspace(dev, rows, Hq, dt), 0xFF, dtype=np.uint8)))     # NaN
        for b in ("q", "lens"):
            w[b].zero()
        lthn.sync()

        def step():
            lthn.paged_sdpa_decode(dev, w["q"], dt, w["lens"], rows, Hq, w["out"], w["ws"], lse=w["lse"], stream=st)
        step()
        st.sync()
        w["graph"] = lthn.Graph(st)
        with w["graph"]:
            step()
        lanes.append(w)
    full = np.array(most, dtype=np.int32)
    plans = [full, np.minimum(full, 1), full // 2, full * (np.arange(rows) % 2), full * 0, np.minimum(full, 65), full]
    for t in range(len(plans)):
        data = []
        for w, lens in ((lanes[0], plans[t]), (lanes[1], plans[-1 - t])):
            lens = np.ascontiguousarray(lens, dtype=np.int32)
            x, b = upload(lthn, rng.standard_normal((rows, Hq, D)), f32)
            w["q"].upload(x if f32 else to_bf16(x))
            w["lens"].upload(lens)
            w["out"].upload(np.full(rows * Hq * D * size, 0xFF, dtype=np.uint8))
            data.append((x, lens))
        lthn.sync()
        for w in lanes:
            w["graph"].launch()
        lthn.sync()
        assert lthn.device_status() == 0
        for w, (x, lens) in zip(lanes, data):
            got, lse = fetch(w["out"], (rows, Hq, D), f32), w["lse"].download(np.float32, (rows, Hq))
            rounded = 0.0 if f32 else 2.0 ** -8
            for r in range(rows):
                n = int(lens[r])
                want, wl, mag = attention(c, r, x[r:r + 1], n - 1, n)
                close(got[r:r + 1], want, (rounded + 2.0 ** -23) * np.abs(want) + (W + (rounded if G > 8 else 0.0)) * mag)
                same_lse(lse[r:r + 1], wl)
