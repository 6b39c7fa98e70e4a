"""What the window, verification, copy and gather calls refuse before they touch a
device (CPU)."""
import eakv_amd as E


def _code(rc):
    code, _ = E.last_error()
    E.lib().eakv_clear_error()
    assert rc == code
    return rc


def test_window_arguments():
    L = E.lib()
    one = E.ints([1])
    null = E.handles([])
    for caches, n in ((None, 1), (null, 0), (null, -1), (null, 33)):
        assert _code(L.eakv_attention_window_batch_device(caches, n, 0, None, one, 16, 0, 8, 8, None, 16,
                                                          None, 0, None)) == E.EAKV_ERR_INVALID
        assert L.eakv_attention_window_work_bytes(caches, n, None, one, 0, 8, 8) == 0
        assert E.last_error()[0] == E.EAKV_ERR_INVALID
    empty = (E._vp * 1)()
    assert _code(L.eakv_attention_window_batch_device(empty, 1, 0, None, one, 16, 0, 8, 8, None, 16, None,
                                                      0, None)) == E.EAKV_ERR_INVALID


def test_verify_arguments():
    L = E.lib()
    ok = dict(n=2, k=3, v=100, counts=0, tokens=64, draft=64, ld_d=100, target=64, ld_t=100, u=64,
              kept=64, next=64, work=64, size=1 << 20)

    def call(**kw):
        a = dict(ok, **kw)
        return L.eakv_verify_drafts_device(a["n"], a["k"], a["v"], a["counts"], a["tokens"], a["draft"],
                                           a["ld_d"], a["target"], a["ld_t"], a["u"], a["kept"],
                                           a["next"], a["work"], a["size"], None)

    for kw in (dict(n=-1), dict(n=65536), dict(k=-1), dict(v=0), dict(v=(1 << 30) + 1), dict(ld_d=99),
               dict(ld_t=99), dict(tokens=0), dict(target=0), dict(u=0), dict(kept=0), dict(next=0),
               dict(work=0), dict(work=68), dict(size=8), dict(tokens=66), dict(draft=65), dict(target=67),
               dict(u=66), dict(kept=65), dict(next=66), dict(counts=2)):
        assert _code(call(**kw)) == E.EAKV_ERR_INVALID, kw
    L.eakv_clear_error()
    assert call(n=0, target=0) == E.EAKV_OK          # nothing to do
    assert L.eakv_verify_drafts_work_bytes(0, 3, 100) == 0
    assert L.eakv_verify_drafts_work_bytes(2, 3, 100) > 0
    assert L.eakv_last_error() == E.EAKV_OK
    assert L.eakv_verify_drafts_work_bytes(2, 3, 0) == 0
    assert L.eakv_last_error() == E.EAKV_ERR_INVALID
    # 257 segments would not fit the second launch: longer ones instead
    assert L.eakv_verify_drafts_work_bytes(1, 0, 1 << 30) <= 256 * 16


def test_move_arguments():
    L = E.lib()
    one = E.ints([1])
    h = (E._vp * 1)()
    assert _code(L.eakv_cache_copy_batch_device(None, 0, h, 1, 0, 1, None)) == E.EAKV_ERR_INVALID
    for a in ((None, h, 1), (h, None, 1), (h, h, 0), (h, h, 33), (h, h, 1)):
        assert _code(L.eakv_cache_gather_batch_device(*a, one, 16, one, None)) == E.EAKV_ERR_INVALID
    assert not L.eakv_cache_fork(None, 0, 1)
    assert E.last_error()[0] == E.EAKV_ERR_INVALID
    assert _code(L.eakv_cache_compact(None, 0, one, 1)) == E.EAKV_ERR_INVALID
    assert _code(L.eakv_cache_planes_device(None, 0, 0, None, None, None)) == E.EAKV_ERR_INVALID


def test_verify_overlaps():
    """Results on top of inputs, of one another or of the scratch (addresses alone: nothing
    is launched)."""
    L = E.lib()
    n, k, v = 4, 3, 100
    size = L.eakv_verify_drafts_work_bytes(n, k, v)
    at, end = {}, 4096
    for name, words in (("counts", n), ("tokens", n * k), ("draft", n * k * v), ("target", n * (k + 1) * v),
                        ("u", n * (k + 1)), ("kept", n), ("next", n), ("work", size // 4)):
        at[name], end = (end, 4 * words), end + (4 * words + 7) // 8 * 8

    def call(**kw):
        a = {x: kw.get(x, y[0]) for x, y in at.items()}
        return L.eakv_verify_drafts_device(n, k, v, a["counts"], a["tokens"], a["draft"], v, a["target"], v,
                                           a["u"], a["kept"], a["next"], a["work"], size, None)

    for out in ("kept", "next", "work"):
        for other, (p, m) in at.items():
            if other == out:
                continue
            for q in (p, p + m - 4, p - at[out][1] + 4):
                q = (q + 7) // 8 * 8 if out == "work" else q
                if q + at[out][1] <= p or q >= p + m:
                    continue
                assert _code(call(**{out: q})) == E.EAKV_ERR_INVALID, (out, other, q - p)
