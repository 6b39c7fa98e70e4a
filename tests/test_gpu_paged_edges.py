"""Pages, attention weights and log probabilities at the edges of how their work is divided: more kv
heads than a wave has lanes, fewer than the pool's, q heads that fill several row blocks, more
sequences than one line, units in many parts, rows in several groups, calls side by side."""
import numpy as np
import pytest

import paging as P
import test_gpu_evict as EV
import windows as W
from windows import E32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


@pytest.fixture
def rng():
    return np.random.default_rng(23)


def run(E, rng, lens, new, n_q, n_kv, d, bf16, page=16, heads=None):
    p = P.Pool(E, rng, lens, new, page, heads or n_kv, d)
    p.fill(P.contents(rng, p))
    c = P.Call(p, n_q, n_kv, bf16)
    q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
    c.run()
    got = c.get()
    W.check(got, *P.attend(p, 0, q, n_q, n_kv), bf16)
    c.run()
    assert np.array_equal(got.view(np.uint32), c.get().view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,heads,d,lens,new", [
    (70, 70, 70, 64, [700, 30, 1], [1, 3, 1]),
    (130, 65, 72, 64, [600], [2]),
    (4, 1, 3, 128, [900, 50], [1, 20]),
    (200, 1, 1, 64, [700, 40], [2, 1]),
    (99, 1, 2, 128, [520], [3]),
])
def test_heads(E, rng, bf16, n_q, n_kv, heads, d, lens, new):
    run(E, rng, lens, new, n_q, n_kv, d, bf16, heads=heads)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d,lens", [
    (2, 2, 64, [60000]), (6, 2, 128, [30000, 9]), (5, 1, 64, [45000, 0, 17000]), (16, 1, 128, [25000]),
    (1, 1, 128, [4609])])
def test_many_parts(E, rng, bf16, n_q, n_kv, d, lens):
    run(E, rng, lens, [min(n, 1) for n in lens], n_q, n_kv, d, bf16, page=64)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [64, 65, 130])
def test_sequences_of_several_row_blocks(E, rng, bf16, n):
    lens = [int(x) for x in rng.integers(0, 900, n)]
    new = [min(int(x), m) for x, m in zip(rng.integers(0, 40, n), lens)]
    run(E, rng, lens, new, 8, 1, 64, bf16)


def test_calls_side_by_side(E, rng):
    """Two batches of one pool at a time, on streams and in workspaces of their own."""
    from eakv_amd.hipmem import DeviceArray, Stream, synchronize
    p = P.Pool(E, rng, [3000, 500, 1200], [1, 1, 1], 16, 2, 128)
    p.fill(P.contents(rng, p))
    need = p.batch.work_bytes(8, 2)
    calls = []
    for _ in range(2):
        c = P.Call(p, 8, 2, False)
        q = c.put(rng.standard_normal((p.rows, 8, 128)).astype(np.float32))
        c.buf[1].upload(np.full(c.buf[1].nbytes, c.GUARD, np.uint8))
        calls.append((c, q, DeviceArray((need,), np.uint8), Stream()))
    synchronize()
    for _ in range(5):
        for c, q, work, st in calls:
            c.run(clear=False, stream=st.s, d_work=work.ptr, work_bytes=need)
    synchronize()
    for c, q, work, st in calls:
        W.check(c.get(), *P.attend(p, 0, q, 8, 2), False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d,lens,n", [
    (8, 1, 64, [700, 20], [300, 20]),           # more than 256 rows: several turns and groups
    (200, 2, 128, [300], [9]),
    (70, 70, 64, [260, 40], [1, 3]),
    (6, 2, 128, [10 * k for k in range(32)], [k % 4 for k in range(32)]),
])
def test_weights(E, rng, bf16, n_q, n_kv, d, lens, n):
    j = EV.Job(E, rng, lens, n, n_q, n_kv, d, bf16)
    j.run(0.5)
    j.check(0.5)


def test_weights_of_fewer_heads_than_the_cache_s(E, rng):
    j = EV.Job(E, rng, [400, 33], [2, 5], 4, 3, 128, False)
    j.n_q, j.n_kv = 4, 1                        # the first kv head, 4 q heads
    j.plan = E.WeightsPlan(j.caches, j.n, 4, 1, starts=j.lens, dtype="f32")
    j.w0 = j.w0.reshape(-1)[:len(j.lens) * j.ld + j.ld].reshape(-1, 1, j.ld)
    from eakv_amd.hipmem import DeviceArray
    j.dw = DeviceArray.from_host(j.w0)
    j.run(1.0)
    j.check(1.0)


def test_logprobs_of_many_short_rows(E, rng):
    from eakv_amd import hipmem
    from eakv_amd.hipmem import DeviceArray
    n, v = 70001, 3
    x = rng.standard_normal((n, v)).astype(np.float32) * 5
    t = rng.integers(0, v, n).astype(np.int32)
    dx, dt, lp, ent = DeviceArray.from_host(x), DeviceArray.from_host(t), DeviceArray((n,)), DeviceArray((n,))
    top, tl = DeviceArray((n, 4), np.int32), DeviceArray((n, 4))
    assert E.lib().eakv_token_logprobs_work_bytes(n, v, 4) == 0
    assert E.lib().eakv_token_logprobs_device(n, v, dx.ptr, 0, v, dt.ptr, 4, lp.ptr, ent.ptr, top.ptr, tl.ptr, None,
                                              0, None) == 0
    hipmem.synchronize()
    z = x.astype(np.float64)
    z -= z.max(1, keepdims=True)
    ln = z - np.log(np.exp(z).sum(1, keepdims=True))
    order = np.argsort(-x, axis=1, kind="stable")
    assert np.array_equal(top.download(), np.concatenate([order, np.full((n, 1), -1)], 1))
    want = np.take_along_axis(ln, order, 1)
    assert (np.abs(tl.download()[:, :3] - want) <= 80 * E32 + E32 * np.abs(want)).all()
    assert (tl.download()[:, 3] == -np.inf).all()
    want = ln[np.arange(n), t]
    assert (np.abs(lp.download() - want) <= 80 * E32 + E32 * np.abs(want)).all()
    h = -(np.exp(ln) * ln).sum(1)
    assert (np.abs(ent.download() - h) <= (80 + 165 * h) * E32).all()


# Large work gives each wave rows of its own; the bound on lengths decides, whatever they are.
LARGE = 1 << 27


def large(p, n_q, **kw):
    """The batch with a bound on lengths that makes its work large."""
    return p.make(max_len=LARGE // (p.rows * n_q) + 1, **kw)


def large_pool(E, rng, lens, new, page, n_q, n_kv, d, **kw):
    return P.Pool(E, rng, lens, new, page, n_kv, d, ld_more=LARGE // (sum(new) * n_q) // page + 2, **kw)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 128), (32, 4, 64), (3, 1, 128), (10, 2, 64), (2, 2, 128),
                                        (40, 2, 64), (64, 1, 128), (300, 1, 64), (70, 70, 64)])
@pytest.mark.parametrize("page,lens,new", [
    (64, [700, 3, 1300, 90], [60, 3, 2, 40]),
    (128, [600, 31, 0, 300, 7], [170, 31, 0, 1, 2]),
    (16, [40, 9, 33, 65, 64], [40, 9, 33, 17, 16]),
])
def test_rows_of_waves(E, rng, bf16, n_q, n_kv, d, page, lens, new):
    p = large_pool(E, rng, lens, new, page, n_q, n_kv, d)
    p.fill(P.contents(rng, p))
    c = P.Call(p, n_q, n_kv, bf16)
    q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
    b = large(p, n_q)
    c.run(batch=b)
    got = c.get()
    W.check(got, *P.attend(p, 0, q, n_q, n_kv), bf16)
    c.run(batch=b)
    assert np.array_equal(got.view(np.uint32), c.get().view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d,n_q,n_kv,lens,new", [
    (64, 8, 1, [20000, 100, 9000], [300, 1, 1]),    # cut units, single tokens beside them
    (128, 16, 1, [3000, 2500], [513, 20]),
    (128, 4, 4, [9000], [700]),
])
def test_rows_of_waves_long(E, rng, bf16, d, n_q, n_kv, lens, new):
    p = large_pool(E, rng, lens, new, 16, n_q, n_kv, d)
    p.fill(P.contents(rng, p))
    c = P.Call(p, n_q, n_kv, bf16, more=(8, 3), shift=1)
    q = c.put(rng.standard_normal((p.rows, n_q, d)).astype(np.float32))
    c.run(batch=large(p, n_q))
    W.check(c.get(), *P.attend(p, 0, q, n_q, n_kv), bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_waves_any_values(E, rng, bf16):
    """Pages that hold nothing, tokens of very different size, and a non-finite group that some rows
    see; rows before position 0."""
    p = large_pool(E, rng, [900, 500, 90, 30], [100, 20, 30, 40], 16, 8, 2, 128,
                   bad=((0, 0, -1), (0, 2, 1 << 30), (1, 3, -5)) + tuple((2, k, -1) for k in range(6)))
    x = P.contents(rng, p)
    x[0][1] *= np.exp2(rng.integers(-30, 30, (1, 900, 1))).astype(np.float32)
    x[1][1] += 100.0
    x[1][0] += 20.0
    p.fill(x)
    c = P.Call(p, 8, 2, bf16)
    q = c.put(rng.standard_normal((p.rows, 8, 128)).astype(np.float32))
    b = large(p, 8)
    c.run(batch=b)
    got, (want, tol, half) = c.get(), P.attend(p, 0, q, 8, 2)
    lim = tol + (half + W.O16 * np.abs(want) if bf16 else 0)
    assert (np.abs(got.astype(np.float64) - want) <= lim).all()
    assert (got[120:150] == 0).all() and (got[150:160] == 0).all()
    x[0][1, 0, 880, 70] = np.inf                # of the first sequence: its last 20 rows see it
    p.fill(x)
    c.run(batch=b)
    new = c.get()
    hit = np.zeros(new.shape, bool)
    hit[80:100, :4, 64:] = True
    assert np.isnan(new[hit]).all()
    assert np.array_equal(new[~hit].view(np.uint32), got[~hit].view(np.uint32))


def test_rows_of_waves_in_place_and_in_a_graph(E, rng):
    from eakv_amd.hipmem import DeviceArray, synchronize
    p = large_pool(E, rng, [300, 200], [50, 50], 32, 8, 2, 64)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 8, 2, False)
    q = rng.standard_normal((p.rows, 8, 64)).astype(np.float32)
    c.put(q)
    b = large(p, 8, ragged=False)
    need = b.work_bytes(8, 2)
    work = DeviceArray((need,), np.uint8)
    c.run(batch=b)
    want = c.get()
    W.check(want, *P.attend(p, 0, q, 8, 2), False)
    synchronize()
    g = W.Graph(lambda st: b.attend(0, c.at(0), c.at(0), 8, 2, d_work=work.ptr, work_bytes=need, stream=st))
    for _ in range(3):
        c.put(q)
        synchronize()
        g.launch()
        synchronize()
        got = c._rows(0, c.buf[0].download()).reshape(want.shape)
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    g.free()


def test_long_prompts_of_many_heads_are_accepted(E):
    """8 million rows of a bound of 3200 tokens; 16 times as many pass what the line counts."""
    import ctypes as C
    pool = E.Cache(1, 2, 128, 4096)
    for n, ok in ((1 << 23, True), (1 << 27, False)):
        s = E.PagedBatchStruct(1 << 40, 200, 1 << 41, 1 << 42, 3, 16, n, n, 3200)
        E.lib().eakv_clear_error()
        assert (E.lib().eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, 8, 2) > 0) == ok
        assert (E.last_error()[0] == 0) == ok
    E.lib().eakv_clear_error()


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_waves_of_many_sequences(E, rng, bf16):
    lens = [int(x) for x in rng.integers(0, 700, 90)]
    new = [min(int(x), m) for x, m in zip(rng.integers(0, 70, 90), lens)]
    p = large_pool(E, rng, lens, new, 128, 8, 2, 64)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 8, 2, bf16)
    q = c.put(rng.standard_normal((p.rows, 8, 64)).astype(np.float32))
    c.run(batch=large(p, 8))
    W.check(c.get(), *P.attend(p, 0, q, 8, 2), bf16)
