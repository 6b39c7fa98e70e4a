"""What the calls of pages and of attention weights refuse given a cache: every check is made on
the host, so addresses stand for buffers and nothing is launched."""
import ctypes as C

import numpy as np
import pytest

import windows as W

pytestmark = pytest.mark.gpu

BASE = 1 << 40


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


def refused(E, rc):
    code, msg = E.last_error()
    E.lib().eakv_clear_error()
    return rc == E.EAKV_ERR_INVALID and code == E.EAKV_ERR_INVALID and bool(msg)


LAYERS, N_KV, D, ROOM = 2, 2, 128, 4096
N_Q = 8
OK = dict(tables=BASE, ld=200, lens=BASE + 65536, first=BASE + 131072, n_seqs=3, page=16, n_new=7, max_new=4,
          max_len=2000)


def batch(E, **kw):
    a = dict(OK, **kw)
    return E.PagedBatchStruct(a["tables"], a["ld"], a["lens"], a["first"], a["n_seqs"], a["page"], a["n_new"],
                              a["max_new"], a["max_len"])


BAD_BATCHES = [dict(page=p) for p in (0, -16, 1, 8, 15, 24, 100, 8192)] + [
    dict(n_seqs=-1), dict(n_seqs=4097), dict(n_new=-1), dict(max_new=-1), dict(max_len=-1), dict(tables=0),
    dict(lens=0), dict(tables=BASE + 2), dict(lens=BASE + 65537), dict(first=BASE + 131073), dict(ld=124),
    dict(ld=0), dict(ld=-1), dict(max_len=3201)]
NOTHING = [dict(n_seqs=0, tables=0, lens=0, first=0), dict(n_new=0, tables=0, lens=0, first=0),
           dict(max_new=0)]


@pytest.fixture(scope="module")
def pool(E):
    return E.Cache(LAYERS, N_KV, D, ROOM)


def test_append(E, pool):
    L = E.lib()
    ok = dict(layer=0, k=BASE + (1 << 24), v=BASE + (2 << 24), dtype=1, ld=N_KV * D)

    def call(b={}, **kw):
        a, s = dict(ok, **kw), batch(E, **b)
        return L.eakv_append_paged_device(pool.h, C.addressof(s), a["layer"], a["k"], a["v"], a["dtype"],
                                          a["ld"], None)

    for b in BAD_BATCHES:
        assert refused(E, call(b)), b
    for kw in (dict(layer=-1), dict(layer=LAYERS), dict(dtype=2), dict(ld=N_KV * D - 1), dict(k=0), dict(v=0),
               dict(k=BASE + 1), dict(v=BASE + 3), dict(dtype=0, k=BASE + 2)):
        assert refused(E, call(**kw)), kw
    for b in NOTHING:
        assert call(b, k=0, v=0) == E.EAKV_OK
    assert L.eakv_append_paged_device(pool.h, None, 0, ok["k"], ok["v"], 1, ok["ld"], None) < 0
    E.lib().eakv_clear_error()


def test_attention(E, pool):
    L = E.lib()
    ok = dict(layer=1, q=BASE + (1 << 24), ld_q=N_Q * D, dtype=1, n_q=N_Q, n_kv=N_KV, out=BASE + (2 << 24),
              ld_out=N_Q * D, work=BASE + (1 << 32), size=1 << 30)

    def call(b={}, **kw):
        a, s = dict(ok, **kw), batch(E, **b)
        return L.eakv_attention_paged_device(pool.h, C.addressof(s), a["layer"], a["q"], a["ld_q"], a["dtype"],
                                             a["n_q"], a["n_kv"], a["out"], a["ld_out"], a["work"], a["size"],
                                             None)

    for b in BAD_BATCHES:
        assert refused(E, call(b)), b
        s = batch(E, **b)
        assert L.eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, N_Q, N_KV) == 0
        assert refused(E, E.EAKV_ERR_INVALID), b
    heads = (dict(n_q=7), dict(n_q=0), dict(n_q=-8), dict(n_kv=3), dict(n_kv=0), dict(dtype=2))
    for kw in heads + (
            dict(layer=-1), dict(layer=LAYERS), dict(ld_q=N_Q * D - 1), dict(ld_out=N_Q * D - 1), dict(q=0),
            dict(out=0), dict(q=BASE + (1 << 24) + 1), dict(out=BASE + (2 << 24) + 1),
            dict(dtype=0, q=BASE + (1 << 24) + 2), dict(work=BASE + (1 << 32) + 8), dict(size=64)):
        assert refused(E, call(**kw)), kw
    for kw in heads:
        a, s = dict(ok, **kw), batch(E)
        assert L.eakv_attention_paged_work_bytes(pool.h, C.addressof(s), a["dtype"], a["n_q"], a["n_kv"]) == 0
        assert refused(E, E.EAKV_ERR_INVALID), kw
    # more work than a launch counts
    assert refused(E, call(dict(n_new=1 << 30)))
    # results and scratch on top of what is read, or of one another
    s = batch(E)
    need = L.eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, N_Q, N_KV)
    assert need > 0
    rows = (OK["n_new"] * N_Q * D) * 2
    for at, n in ((OK["tables"], (2 * 200 + 125) * 4), (OK["lens"], 3 * 4), (OK["first"], 4 * 4)):
        for x in (at, at + n - 4):
            assert refused(E, call(out=x)), hex(x)
            assert refused(E, call(work=(x + 15) & ~15 if x == at else (x - need + 15) & ~15)), hex(x)
    for at in (ok["q"] + 2, ok["q"] + rows - 2, ok["q"] - rows + 2):
        assert refused(E, call(out=at))
    assert refused(E, call(out=ok["q"], ld_out=N_Q * D + 8))       # in place: one distance
    for at in (ok["q"], ok["q"] + rows - 16, ok["out"], ok["out"] - need + 16):
        assert refused(E, call(work=at)), hex(at)
    for b in NOTHING:
        assert call(b, q=0, out=0) == E.EAKV_OK
        s = batch(E, **b)
        assert L.eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, N_Q, N_KV) == 0
    assert L.eakv_last_error() == E.EAKV_OK


def test_head_dims(E):
    L = E.lib()
    other = E.Cache(1, 1, 192, 64)
    s = batch(E, page=16, max_len=16)
    assert refused(E, L.eakv_append_paged_device(other.h, C.addressof(s), 0, BASE, BASE + 4096, 0, 192, None))
    assert refused(E, L.eakv_attention_paged_device(other.h, C.addressof(s), 0, BASE, 192, 0, 1, 1, BASE + 4096,
                                                    192, None, 0, None))


def test_weights(E):
    L = E.lib()
    rng = np.random.default_rng(1)
    caches = W.build(E, rng, [200, 2005], N_KV, D, ROOM, LAYERS)
    other, = W.build(E, rng, [2005], N_KV, 64, ROOM, LAYERS)
    ok = dict(h=E.handles(caches), n=2, layer=0, starts=[100, 2000], tok=[3, 5], q=BASE, dtype=1, n_q=N_Q,
              n_kv=N_KV, w=BASE + (1 << 24), ld=2005, work=BASE + (1 << 32), size=1 << 30)

    def call(**kw):
        a = dict(ok, **kw)
        return L.eakv_attention_weights_batch_device(
            a["h"], a["n"], a["layer"], a["starts"] and E.ints(a["starts"]), a["tok"] and E.ints(a["tok"]),
            a["q"], a["dtype"], a["n_q"], a["n_kv"], 0.0, a["w"], a["ld"], a["work"], a["size"], None)

    def need(**kw):
        a = dict(ok, **kw)
        return L.eakv_attention_weights_work_bytes(a["h"], a["n"], E.ints(a["starts"]), E.ints(a["tok"]),
                                                   a["dtype"], a["n_q"], a["n_kv"])

    both = (dict(n=0), dict(n=33), dict(h=E.handles([caches[0], other])), dict(tok=[-1, 5]),
            dict(starts=[-1, 5]), dict(starts=[100, 2005], tok=[3, 2092]), dict(dtype=2), dict(n_q=7), dict(n_kv=3),
            dict(starts=[201, 2000]))
    for kw in both + (
            dict(tok=None), dict(layer=LAYERS), dict(layer=-1), dict(ld=2004), dict(q=0), dict(w=0),
            dict(q=BASE + 1), dict(dtype=0, q=BASE + 2), dict(w=BASE + (1 << 24) + 2),
            dict(work=BASE + (1 << 32) + 8), dict(size=16)):
        assert refused(E, call(**kw)), kw
    for kw in both:
        assert need(**kw) == 0
        assert refused(E, E.EAKV_ERR_INVALID), kw
    size = need()
    assert size > 0
    q_bytes, w_bytes = 8 * N_Q * D * 2, 2 * N_KV * 2005 * 4
    for w in (BASE, BASE + q_bytes - 4, BASE - w_bytes + 4):
        assert refused(E, call(w=w)), hex(w)
    for at, n in ((BASE, q_bytes), (ok["w"], w_bytes)):
        for work in (at, (at + n - 4) & ~15, (at - size + 16) & ~15):
            assert refused(E, call(work=work)), hex(work)
    assert call(tok=[0, 0], q=0, w=0) == E.EAKV_OK
    assert E.lib().eakv_last_error() == E.EAKV_OK


def test_recorded_calls_need_a_workspace(E, pool):
    from eakv_amd.hipmem import DeviceArray, synchronize
    L = E.lib()
    buf = DeviceArray.from_host(np.zeros(1 << 16, np.uint8))
    zeros = DeviceArray.from_host(np.zeros(64, np.int32))
    s = E.PagedBatchStruct(zeros.ptr, 200, zeros.ptr, None, 1, 16, 1, 1, 3200)
    h, one, starts = E.handles([pool]), E.ints([1]), E.ints([2000])

    def record(st):
        assert refused(E, L.eakv_attention_paged_device(
            pool.h, C.addressof(s), 0, buf.ptr, N_Q * D, 0, N_Q, N_KV, buf.ptr + 32768, N_Q * D, None, 0, st))
        assert refused(E, L.eakv_attention_weights_batch_device(
            h, 1, 0, starts, one, buf.ptr, 0, N_Q, N_KV, 0.0, buf.ptr + 32768, 2001, None, 0, st))
        # the recording goes on: a sequence of no tokens
        assert L.eakv_append_paged_device(pool.h, C.addressof(s), 0, buf.ptr, buf.ptr, 0, N_KV * D, st) == 0

    synchronize()
    g = W.Graph(record)
    g.launch()
    synchronize()
    g.free()
