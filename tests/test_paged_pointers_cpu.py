"""Arrays of the paged-cache calls whose addresses are no multiple of their elements' size are refused before any device work."""
import pytest

from test_paged_cpu import A, append, decode, desc, prefill


def last(lthn):
    return lthn.lib().lthn_last_error().decode()


@pytest.mark.parametrize("bad", [dict(seq=A + 2), dict(pos=A + 1)], ids=str)
def test_append_refuses_misaligned_arrays(lthn, bad):
    assert append(lthn, desc(lthn), **bad) == 1 and "aligned" in last(lthn)


@pytest.mark.parametrize("off", [1, 2, 4])
def test_append_refuses_misaligned_frequencies(lthn, off):
    assert append(lthn, desc(lthn), lthn.RopeParams(A + off, 64, 0, None, None, 1e-6)) == 1 and "inv_freq" in last(lthn)


def test_misaligned_page_tables_are_refused(lthn):
    for call in (append, decode, prefill):
        assert call(lthn, desc(lthn, page_table=(1 << 22) + 2)) == 1 and "page_table" in last(lthn)


@pytest.mark.parametrize("call,bad", [(decode, dict(lens=A + 2)), (prefill, dict(lens=A + 3)), (prefill, dict(start=A + 2))])
def test_attention_refuses_misaligned_lengths(lthn, call, bad):
    assert call(lthn, desc(lthn), **bad) == 1 and "aligned" in last(lthn)


@pytest.mark.parametrize("field", ["slopes", "prefix_lens"])
def test_attention_refuses_misaligned_options(lthn, field):
    for call in (decode, prefill):
        o = lthn.AttnOptions()
        setattr(o, field, A + 2)
        assert call(lthn, desc(lthn), o) == 1 and field in last(lthn)


def test_attention_refuses_misaligned_sums(lthn):
    L = lthn.lib()
    d = desc(lthn)
    assert L.lthn_paged_sdpa_decode(None, d, None, A, 1, 0, A, 2, 4, A, 0, A + 2, A, 1 << 30) == 1 and "lse" in last(lthn)
    assert L.lthn_paged_prefill_attention(None, d, None, A, 0, A, A, 2, 9, 4, 0, A, 0, A + 1, A, 1 << 40) == 1 and "lse" in last(lthn)
