"""What the paged prompt attention does when one of its roles never starts and the waits of the others run out: it returns by itself, the
status says so, and the next call computes as ever. Tolerances: those of test_gpu_paged.py."""
import numpy as np
import pytest

from paged_util import HostCache, from_bf16
from test_gpu_paged import check_prefill, upload

pytestmark = pytest.mark.gpu

# how the keys, values and queries come: by TMA; by TMA with a last tile that is copied row by row; the queries row by row; all row by row.
# With a context of 4000 the keys are cut and a second kernel joins the chunks.
FORMS = [(128, 16, 256, 0), (128, 16, 300, 0), (64, 16, 300, 24), (256, 16, 150, 0), (128, 5, 300, 24), (128, 16, 4000, 0)]


@pytest.mark.parametrize("D,page,n,extra", FORMS)
@pytest.mark.parametrize("role", [1, 2, 3])
def test_prefill_returns_when_a_role_gives_up(lthn, role, D, page, n, extra):
    rng = np.random.default_rng(61)
    new, Hq = 40, 2
    c = HostCache(rng, [n], page, 1, D)
    q = rng.standard_normal((new, Hq, D))
    stride = Hq * D + extra
    wide = np.zeros((new, stride))
    wide[:, :Hq * D] = q.reshape(new, -1)
    _, qb = upload(lthn, wide, False)
    dev = c.device(lthn)
    out = lthn.Buf.from_array(np.zeros((new, Hq, D), dtype=np.uint16))
    need = lthn.paged_prefill_attention_workspace(dev, 1, new, Hq)
    ws = lthn.Buf.from_array(np.full(need, 0xFF, dtype=np.uint8))
    start, lens = lthn.Buf.from_array(np.array([0, new], dtype=np.int32)), lthn.Buf.from_array(np.array([n], dtype=np.int32))

    def run():
        lthn.paged_prefill_attention(dev, qb, start, lens, 1, new, Hq, out, ws, q_stride=stride)
    run()
    assert lthn.device_status() == 0
    want = out.download(np.uint16, (new, Hq, D))
    lthn.lib().lthn_debug_paged_prefill_give_up(role)
    try:
        run()
        with pytest.raises(lthn.LthnError) as e:
            lthn.device_status()
        assert e.value.code == 5
    finally:
        lthn.lib().lthn_debug_paged_prefill_give_up(0)
    assert lthn.device_status() == 0
    out.zero()
    run()
    assert lthn.device_status() == 0
    assert np.array_equal(out.download(np.uint16, (new, Hq, D)), want) and np.all(np.isfinite(from_bf16(want)))
    check_prefill(lthn, c, q, [new])
