"""Sequences in pages of a pool: appends (bit for bit those of a cache) and attention
against the exact one of the packed planes (bounds: paging.py)."""
import numpy as np
import pytest

import paging as P
import windows as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


def planes_at(c, layer, kv):
    w, s, b = c.read_planes(layer, kv)
    gpd = c.head_dim // 64
    shape = (c.n_heads, c.max_seq_len, gpd)
    return w.reshape(shape + (32,)), s.view(np.uint32).reshape(shape), b.view(np.uint32).reshape(shape)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d,n_kv,page,lens,new,more,shift", [
    (128, 2, 16, [37, 1, 100], [5, 1, 100], 0, 0),
    (64, 3, 32, [64, 33, 5, 90], [64, 1, 0, 31], 7, 1),
    (128, 1, 256, [300], [3], 4, 0),
    (64, 4, 16, [3, 2], [7, 2], 8, 2),              # more rows than tokens: the first are dropped
])
def test_append_is_the_cache_s(E, rng, bf16, d, n_kv, page, lens, new, more, shift):
    """New tokens' planes are those that a cache of the same values has; every other byte of the pool
    stays, pages outside the pool are not written."""
    from eakv_amd.hipmem import DeviceArray
    layers = 2
    p = P.Pool(E, rng, lens, new, page, n_kv, d, layers=layers, bad=((0, 0, -1),) if len(lens) > 3 else ())
    old = rng.standard_normal((layers, 2, n_kv, p.pool.max_seq_len, d)).astype(np.float32)
    p.pool.load_raw(old, p.pool.max_seq_len)
    before = [[planes_at(p.pool, l, j) for j in (0, 1)] for l in range(layers)]
    ld = n_kv * d + more
    kv = [rng.standard_normal((p.rows, ld)).astype(np.float32) for _ in (0, 1)]
    if bf16:
        kv = [W.from_bf16(W.to_bf16(x)) for x in kv]
    dev = []
    for x in kv:
        u = W.to_bf16(x) if bf16 else x
        u = np.concatenate([np.zeros(shift, u.dtype), u.reshape(-1)])
        dev.append(DeviceArray.from_host(u))
    size = 2 if bf16 else 4
    p.batch.append(1, dev[0].ptr + shift * size, dev[1].ptr + shift * size, "bf16" if bf16 else "f32", ld)
    p.pool.sync()
    for l in range(layers):
        for j in (0, 1):
            want = [x.copy() for x in before[l][j]]
            if l == 1:
                for s, m in enumerate(new):
                    x = kv[j][p.first[s]:p.first[s + 1], :n_kv * d].reshape(m, n_kv, d)
                    x = x[max(0, m - lens[s]):]
                    at = p.place(s)[max(0, lens[s] - m):]
                    if len(x) == 0:
                        continue
                    c = E.Cache(1, n_kv, d, len(x))
                    c.load_raw(np.stack([x.transpose(1, 0, 2)] * 2)[None], len(x))
                    for to, y in zip(want, planes_at(c, 0, 0)):
                        to[:, at[at >= 0]] = y[:, at >= 0]
            for got, y in zip(planes_at(p.pool, l, j), want):
                assert np.array_equal(got, y)


HEADS = [(8, 2, 128), (32, 4, 64), (3, 1, 128), (10, 2, 64), (2, 2, 128), (40, 2, 64), (64, 1, 128)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d", HEADS)
@pytest.mark.parametrize("page,lens,new", [
    (16, [1], [1]),
    (16, [1, 2, 15, 16, 17, 31, 32, 33, 255, 256, 257, 511], [1] * 12),
    (32, [513, 1, 1025, 300, 40], [1] * 5),
    (64, [700, 3, 2000, 90], [5, 3, 2, 4]),
    (128, [600, 31, 0, 300, 7], [70, 31, 0, 1, 2]),
    (16, [40, 9], [40, 9]),
])
def test_attention(E, rng, bf16, n_q, n_kv, d, page, lens, new):
    p = P.Pool(E, rng, lens, new, page, n_kv, d)
    p.fill(P.contents(rng, p))
    c = P.Call(p, n_q, n_kv, bf16)
    q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
    c.run()
    W.check(c.get(), *P.attend(p, 0, q, n_q, n_kv), bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d,n_q,n_kv,lens,new", [
    (128, 8, 2, [9000, 20, 5000, 0, 12000], [1] * 5),
    (64, 8, 1, [20000, 100], [300, 1]),
    (128, 16, 1, [3000], [513]),
])
def test_attention_long(E, rng, bf16, d, n_q, n_kv, lens, new):
    """Units cut among blocks, more sub-tiles of a wave than one read of the table, rows and
    lengths on either side of a cut."""
    p = P.Pool(E, rng, lens, new, 16, n_kv, d)
    p.fill(P.contents(rng, p))
    c = P.Call(p, n_q, n_kv, bf16)
    q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
    c.run()
    W.check(c.get(), *P.attend(p, 0, q, n_q, n_kv), bf16)
    first = c.get()
    c.run()
    assert np.array_equal(first.view(np.uint32), c.get().view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("more,shift", [((0, 0), 1), ((24, 3), 0), ((64, 8), 2), ((5, 64), 4)])
def test_attention_strides(E, rng, bf16, more, shift):
    p = P.Pool(E, rng, [50, 600], [20, 1], 32, 2, 64, ld_more=5)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 6, 2, bf16, more, shift)
    q = c.put(rng.standard_normal((p.rows, 6, 64)).astype(np.float32))
    c.run()
    W.check(c.get(), *P.attend(p, 0, q, 6, 2), bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_attention_many_sequences(E, rng, bf16):
    lens = [int(x) for x in rng.integers(0, 60, 700)]
    new = [min(int(x), n) for x, n in zip(rng.integers(0, 3, 700), lens)]
    p = P.Pool(E, rng, lens, new, 16, 1, 64)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 4, 1, bf16)
    q = c.put(rng.standard_normal((p.rows, 4, 64)).astype(np.float32))
    c.run()
    W.check(c.get(), *P.attend(p, 0, q, 4, 1), bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_that_hold_nothing(E, rng, bf16, page):
    """Pages freed in the middle, at the start, everywhere; rows before position 0."""
    bad = ((0, 0, -1), (0, 2, 1 << 30), (1, 3, -5)) + tuple((2, k, -1) for k in range(-(-90 // page)))
    p = P.Pool(E, rng, [900, 500, 90, 3], [1, 20, 3, 9], page, 2, 128, bad=bad)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 8, 2, bf16)
    q = c.put(rng.standard_normal((p.rows, 8, 128)).astype(np.float32))
    c.run()
    got = c.get()
    want = P.attend(p, 0, q, 8, 2)
    W.check(got, *want, bf16)
    assert (got[21:24] == 0).all() and (got[24:30] == 0).all()


def test_in_place_and_uniform_rows(E, rng):
    """One buffer for q and out; rows by max_new instead of a list; another layer; a stream."""
    from eakv_amd import hipmem
    p = P.Pool(E, rng, [70, 400, 33], [2, 2, 2], 16, 2, 64, layers=2)
    x = P.contents(rng, p)
    p.fill(x, layer=1)
    c = P.Call(p, 4, 2, False)
    q = c.put(rng.standard_normal((p.rows, 4, 64)).astype(np.float32))
    c.run(layer=1)
    want = c.get()
    W.check(want, *P.attend(p, 1, q, 4, 2), False)
    st = hipmem.Stream()
    b = p.make(ragged=False)
    need = b.work_bytes(4, 2)
    work = hipmem.DeviceArray((max(need, 1),), np.uint8)
    b.attend(1, c.at(0), c.at(0), 4, 2, d_work=work.ptr, work_bytes=need, stream=st.s)
    st.synchronize()
    got = c._rows(0, c.buf[0].download()).reshape(want.shape)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_values_beyond_the_bounds_are_held(E, rng):
    """Lengths, rows and pages on the device that pass the call's bounds stay within the buffers."""
    from eakv_amd.hipmem import DeviceArray
    p = P.Pool(E, rng, [40, 40], [4, 4], 16, 1, 64)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 2, 1, False)
    c.put(rng.standard_normal((p.rows, 2, 64)).astype(np.float32))
    p.d_lens.upload(np.array([1 << 30, -7, 0], np.int32))
    for first in ([0, 1 << 30, 1 << 30], [-5, 100, 3], [7, 2, 9]):
        f = DeviceArray.from_host(np.array(first, np.int32))
        b = p.make(d_first=f.ptr)
        c.run(batch=b)
        c.get()
        dk = DeviceArray((p.rows, 64))
        b.append(0, dk.ptr, dk.ptr)
        p.pool.sync()


@pytest.mark.parametrize("bf16", [False, True])
def test_values_of_any_size(E, rng, bf16):
    """Outliers, offsets, tokens of very different size, and non-finite tokens that some rows see."""
    p = P.Pool(E, rng, [600, 300], [40, 1], 32, 2, 128)
    x = P.contents(rng, p)
    x[0][1] *= np.exp2(rng.integers(-30, 30, (1, 600, 1))).astype(np.float32)
    x[1][1] += 100.0
    x[1][1, :, :, 5] -= 1000.0
    x[1][0] += 20.0
    p.fill(x)
    c = P.Call(p, 8, 2, bf16)
    q = c.put(rng.standard_normal((p.rows, 8, 128)).astype(np.float32))
    c.run()
    got, (want, tol, half) = c.get().astype(np.float64), P.attend(p, 0, q, 8, 2)
    lim = tol + (half + W.O16 * np.abs(want) if bf16 else 0)
    assert (np.abs(got - want) <= lim).all()
    # position 580 of the first sequence: the last 20 rows see it
    x[0][1, 0, 580, 70] = np.inf
    p.fill(x)
    c.run()
    new = c.get()
    hit = np.zeros(new.shape, bool)
    hit[20:40, :4, 64:] = True
    assert np.isnan(new[hit]).all()
    assert np.array_equal(new[~hit].view(np.uint32), got.astype(np.float32)[~hit].view(np.uint32))


def test_graph_follows_the_device(E, rng):
    """A recorded append and attention, replayed with other tables, lengths and rows."""
    from eakv_amd.hipmem import DeviceArray, synchronize
    n_q, n_kv, d = 8, 2, 128
    p = P.Pool(E, rng, [300, 900, 17], [1, 1, 1], 16, n_kv, d, ld_more=80)
    x = P.contents(rng, p)
    p.fill(x)
    b = p.make(max_len=1500)
    need = b.work_bytes(n_q, n_kv)
    work = DeviceArray((need,), np.uint8)
    c = P.Call(p, n_q, n_kv, False)
    kv = [DeviceArray((p.rows, n_kv * d)) for _ in (0, 1)]

    def record(st):
        b.append(0, kv[0].ptr, kv[1].ptr, stream=st)
        c.run(batch=b, clear=False, stream=st, d_work=work.ptr, work_bytes=need)

    c.buf[1].upload(np.full(c.buf[1].nbytes, c.GUARD, np.uint8))
    synchronize()
    g = W.Graph(record)
    lens = list(p.lens)
    for step in range(4):
        rows = [rng.standard_normal((p.rows, n_kv * d)).astype(np.float32) for _ in (0, 1)]
        for to, y in zip(kv, rows):
            to.upload(y)
        q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
        p.d_lens.upload(np.asarray(lens + [0], np.int32))
        p.lens = list(lens)
        synchronize()
        g.launch()
        W.check(c.get(), *P.attend(p, 0, q, n_q, n_kv), False)
        first = c.get()
        # a sequence grows into a page that was free, another shrinks
        lens[1] -= 100 * step
        lens[2] += 1
        if step == 1:
            lens[2] = 33
            used = set(p.table[p.table < p.n_pages].tolist())
            free = [k for k in range(p.n_pages) if k not in used]
            p.table[2, 1:3] = free[:2]
            p.d_table.upload(p.table)
    g.free()
