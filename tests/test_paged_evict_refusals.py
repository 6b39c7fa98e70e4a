"""What the calls of pages, attention weights, eviction and log probabilities refuse before they
touch a device (CPU)."""
import ctypes as C

import pytest

import eakv_amd as E

INVALID = E.EAKV_ERR_INVALID


def refused(rc):
    code, msg = E.last_error()
    E.lib().eakv_clear_error()
    return rc == INVALID and code == INVALID and msg


def test_no_pool_or_batch():
    L = E.lib()
    b = C.addressof(E.PagedBatchStruct(64, 1, 64, None, 1, 16, 1, 1, 16))
    for args in ((None, b), (None, None)):
        assert refused(L.eakv_append_paged_device(*args, 0, 64, 64, 0, 128, None))
        assert refused(L.eakv_attention_paged_device(*args, 0, 64, 128, 0, 1, 1, 64, 128, None, 0, None))
        assert L.eakv_attention_paged_work_bytes(*args, 0, 1, 1) == 0
        assert refused(INVALID)


def test_binding():
    with pytest.raises(ValueError):
        E.PagedBatch(None, 16, 64, 1, 64, 1, 16, d_first=64)
    b = E.PagedBatch(None, 16, 64, 7, 128, 5, 100, max_new=3)
    got = {f: getattr(b.args, f) for f, _ in b.args._fields_}
    assert got == dict(d_tables=64, ld_table=7, d_lens=128, d_first=None, n_seqs=5, page_tokens=16,
                       n_new=15, max_new=3, max_len=100)


def test_weights_arguments():
    L = E.lib()
    one, null, empty = E.ints([1]), E.handles([]), (E._vp * 1)()
    for caches, n in ((None, 1), (null, 0), (null, -1), (null, 33), (empty, 1)):
        assert refused(L.eakv_attention_weights_batch_device(caches, n, 0, None, one, 16, 0, 8, 8, 1.0, 16,
                                                             16, None, 0, None))
        assert L.eakv_attention_weights_work_bytes(caches, n, None, one, 0, 8, 8) == 0
        assert refused(INVALID)


def test_select_arguments():
    L = E.lib()
    ok = dict(n=2, h=3, w=4096, ld=20000, tok=[100, 20000], first=4, recent=8, keep=[12, 500], idx=1 << 20,
              kept=1 << 22, ld_kept=500, work=1 << 24, size=1 << 22)

    def call(**kw):
        a = dict(ok, **kw)
        tok, keep = (E.ints(a[x]) if a[x] else None for x in ("tok", "keep"))
        return L.eakv_evict_select_device(a["n"], a["h"], a["w"], a["ld"], tok, a["first"], a["recent"],
                                          keep, a["idx"], a["kept"], a["ld_kept"], a["work"], a["size"],
                                          None)

    for kw in (dict(n=-1), dict(n=33), dict(h=0), dict(h=65537), dict(first=-1), dict(recent=-1),
               dict(tok=None), dict(keep=None), dict(tok=[100, -1]), dict(keep=[11, 500]),
               dict(keep=[101, 500]), dict(keep=[12, -1]), dict(first=1 << 30, recent=1 << 30),
               dict(tok=[100, (1 << 30) + 1], ld=1 << 31), dict(ld=19999), dict(ld_kept=499), dict(w=0), dict(idx=0), dict(work=0),
               dict(w=4097), dict(idx=(1 << 20) + 2), dict(kept=(1 << 22) + 1), dict(work=(1 << 24) + 2),
               dict(size=16)):
        assert refused(call(**kw)), kw
    assert call(n=0, tok=None, keep=None, w=0) == E.EAKV_OK
    assert call(tok=[100, 200], first=0, recent=0, keep=[0, 0], kept=0, w=0, work=0) == E.EAKV_OK
    assert L.eakv_evict_select_work_bytes(2, E.ints([8192, 100])) == 0
    assert L.eakv_evict_select_work_bytes(2, E.ints([8193, 100])) > 0
    assert L.eakv_evict_select_work_bytes(0, None) == 0
    assert L.eakv_last_error() == E.EAKV_OK
    for n, tok in ((-1, [1]), (33, [1] * 33), (1, None), (2, [5, -1]), (1, [(1 << 30) + 1])):
        assert L.eakv_evict_select_work_bytes(n, tok and E.ints(tok)) == 0
        assert refused(INVALID), (n, tok)


def test_logprobs_arguments():
    L = E.lib()
    ok = dict(n=3, v=40000, logits=1 << 20, dtype=0, ld=40001, tokens=64, top=5, lp=128, ent=192,
              tt=256, tl=512, work=4096, size=1 << 16)

    def call(**kw):
        a = dict(ok, **kw)
        return L.eakv_token_logprobs_device(a["n"], a["v"], a["logits"], a["dtype"], a["ld"], a["tokens"],
                                            a["top"], a["lp"], a["ent"], a["tt"], a["tl"], a["work"],
                                            a["size"], None)

    for kw in (dict(n=-1), dict(v=0), dict(v=(1 << 30) + 1, ld=1 << 31), dict(n=1 << 30), dict(ld=39999),
               dict(top=-1), dict(top=33), dict(dtype=2), dict(dtype=-1), dict(logits=0), dict(tokens=0),
               dict(tt=0), dict(tl=0), dict(work=0), dict(size=16), dict(work=4104), dict(tokens=66),
               dict(lp=130), dict(ent=193), dict(tt=258), dict(tl=513), dict(logits=(1 << 20) + 2),
               dict(logits=(1 << 20) + 1, dtype=1)):
        assert refused(call(**kw)), kw
    assert call(n=0, logits=0) == E.EAKV_OK
    assert call(lp=0, ent=0, top=0, logits=0) == E.EAKV_OK
    assert L.eakv_token_logprobs_work_bytes(3, 16377, 5) == 0
    assert L.eakv_token_logprobs_work_bytes(3, 16378, 5) > 0
    assert L.eakv_last_error() == E.EAKV_OK
    # a launch has fewer than 2^32 threads
    for n, v, top in ((-1, 10, 0), (1, 0, 0), (1, 10, 33), (1 << 24, 100, 0), (1 << 18, 1 << 20, 0)):
        assert L.eakv_token_logprobs_work_bytes(n, v, top) == 0
        assert refused(INVALID), (n, v, top)


def test_overlaps():
    """Results on top of inputs, of one another or of the scratch (addresses alone: nothing is
    launched)."""
    L = E.lib()

    def layout(**spans):
        at, end = {}, 1 << 24
        for name, size in spans.items():
            at[name], end = (end, size), end + (size + 15) // 16 * 16
        return at

    def every(at, outs, call):
        for out in outs:
            for other, (p, m) in at.items():
                if other == out:
                    continue
                for q in (p, p + m - 4, p - at[out][1] + 4):
                    q = (q + 15) // 16 * 16 if out == "work" else q
                    if q + at[out][1] <= p or q >= p + m:
                        continue
                    a = {x: y[0] for x, y in at.items()}
                    a[out] = q
                    assert refused(call(a)), (out, other, q - p)

    n, v, top = 5, 40000, 3
    size = L.eakv_token_logprobs_work_bytes(n, v, top)
    every(layout(logits=n * v * 4, tokens=n * 4, lp=n * 4, ent=n * 4, tt=n * top * 4, tl=n * top * 4,
                 work=size), ("lp", "ent", "tt", "tl", "work"),
          lambda a: L.eakv_token_logprobs_device(n, v, a["logits"], 0, v, a["tokens"], top, a["lp"],
                                                 a["ent"], a["tt"], a["tl"], a["work"], size, None))
    tok, keep = E.ints([9000, 100]), E.ints([4000, 50])
    size = L.eakv_evict_select_work_bytes(2, tok)
    every(layout(w=2 * 3 * 9000 * 4, idx=4050 * 4, kept=2 * 3 * 4000 * 4, work=size),
          ("idx", "kept", "work"),
          lambda a: L.eakv_evict_select_device(2, 3, a["w"], 9000, tok, 4, 4, keep, a["idx"], a["kept"],
                                               4000, a["work"], size, None))
