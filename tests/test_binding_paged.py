"""What the Python binding makes of a paged batch's counts (CPU)."""
import pytest

import eakv_amd as E

OK = dict(page_tokens=16, n_seqs=2, max_len=100, max_new=1, n_new=2)


def make(**kw):
    a = dict(OK, **kw)
    return E.PagedBatch(None, a["page_tokens"], 64, 7, 128, a["n_seqs"], a["max_len"], a["max_new"], n_new=a["n_new"])


@pytest.mark.parametrize("kw", [
    dict(n_seqs=4096, max_new=1 << 20, n_new=None),         # 2^32 rows are not none
    dict(n_seqs=2, max_new=1 << 30, n_new=None), dict(n_new=2 ** 32 + 2), dict(max_len=2 ** 32 + 100),
    dict(max_len=2 ** 31), dict(n_seqs=2 ** 32 + 2), dict(page_tokens=2 ** 32 + 16), dict(max_new=-2 ** 32)])
def test_counts_beyond_32_bits(kw):
    with pytest.raises(ValueError):
        make(**kw)


def test_counts_within():
    b = make(n_seqs=4096, max_new=(1 << 19) - 1, n_new=None, max_len=2 ** 31 - 1)
    assert b.args.n_new == 4096 * ((1 << 19) - 1) and b.args.max_len == 2 ** 31 - 1
    assert make().args.n_new == 2
