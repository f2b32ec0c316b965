"""rope_params and rope_inv_freq with their defaults belong together: all pairs that there are frequencies for are turned."""
import numpy as np
import pytest

from paged_util import HostCache, from_bf16, to_bf16, turn


class Held:
    def __init__(self, a):
        self.a, self.nbytes = a, a.nbytes

    def data_ptr(self):
        return self.a.ctypes.data


@pytest.mark.parametrize("D,rotary", [(128, 0), (64, 0), (256, 64), (128, 2)])
def test_rotary_dim_follows_the_frequencies(lthn, D, rotary):
    f = Held(lthn.rope_inv_freq(1e4, D, rotary))
    assert lthn.rope_params(f).rotary_dim == (rotary or D)
    assert lthn.rope_params(f, 2).rotary_dim == 2


def test_frequencies_of_unknown_number_need_it(lthn):
    at = type("P", (), {"data_ptr": lambda self: 1 << 20})()
    assert lthn.rope_params(at, 64).rotary_dim == 64
    with pytest.raises(lthn.LthnError):
        lthn.rope_params(at)


def test_more_pairs_than_frequencies_are_refused(lthn):
    f = Held(lthn.rope_inv_freq(1e4, 128, 64))
    assert lthn.rope_params(f, 64).rotary_dim == 64
    with pytest.raises(lthn.LthnError):
        lthn.rope_params(f, 66)


def test_no_frequencies_no_rotation(lthn):
    p = lthn.rope_params()
    assert p.rotary_dim == 0 and not p.inv_freq


@pytest.mark.gpu
def test_append_turns_with_the_defaults(lthn):
    rng = np.random.default_rng(81)
    rows, D = 5, 128
    c = HostCache(rng, [0], 16, 1, D, room=rows)
    dev = c.device(lthn)
    inv = lthn.rope_inv_freq(1e4, D)
    x = to_bf16(rng.standard_normal((rows, 1, D)))
    b, pos = lthn.Buf.from_array(x), np.arange(rows, dtype=np.int32)
    lthn.paged_kv_append(dev, b, b, lthn.Buf.from_array(pos * 0), lthn.Buf.from_array(pos), rows, lthn.BF16, rope=lthn.rope_params(lthn.Buf.from_array(inv)))
    lthn.sync()
    assert lthn.device_status() == 0
    got = from_bf16(dev._keep[0].download(np.uint16, c.k.shape)[c.table[0, 0], :rows])
    want = turn(from_bf16(x), pos, inv)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 1e-5)      # one rounding to bf16, and f32 products of values below 8
