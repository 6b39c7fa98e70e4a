"""Eviction by attention weight: the weights (eakv_attention_weights_batch_device) against
64 bits, the choice (eakv_evict_select_device) against its definition, and the loop of weights,
choice and gather.

Bound of a weight: a score is off by dS <= 40 e A (windows.py: K's operands are exact here for
both types, a bf16 query is exact in f16), so a softmax weight by a factor within 2 max dS + 8 e
(exponential, its argument, the sum, the quotient), and the sum over r rows, added by 16 lanes,
row tiles and keep * w, by at most (r / 16 + 8) e of it more."""
import ctypes as C

import numpy as np
import pytest

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


def exact(cache, layer, q, start, n_q, n_kv):
    """f64 [n_kv][start + m] sums of softmax weights, and their bounds."""
    m, _, d = q.shape
    k, ks = W.values(cache, layer, 0)
    g, t = n_q // n_kv, start + m
    out, tol = np.zeros((n_kv, t)), np.zeros((n_kv, t))
    for h in range(n_q):
        kh = k[h // g, :t]
        kc = np.repeat(ks[h // g, :t], 64, 1)
        qs = q[:, h].astype(np.float64)
        s = qs @ kh.T / np.sqrt(d)
        a = np.abs(qs) @ (2 * np.abs(kh) + 2 * kc).T / np.sqrt(d)
        for i in range(m):
            n = start + i + 1
            p = np.exp(s[i, :n] - s[i, :n].max())
            p /= p.sum()
            out[h // g, :n] += p
            tol[h // g, :n] += p * (80 * E32 * a[i, :n].max() + (8 + m * g / 16 + 8) * E32)
    return out, tol


class Job:
    GUARD = -77.0

    def __init__(self, E, rng, lens, n_tokens, n_q, n_kv, d, bf16, layers=1, ld_more=3, scale=1.0):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.lens, self.n, self.n_q, self.n_kv = E, lens, n_tokens, n_q, n_kv
        total = [a + m for a, m in zip(lens, n_tokens)]
        self.room = max(total) + 2
        self.caches = W.build(E, rng, total, n_kv, d, self.room, layers, scale)
        q = rng.standard_normal((sum(n_tokens), n_q, d)).astype(np.float32)
        u = W.to_bf16(q) if bf16 else q
        self.q = W.from_bf16(u) if bf16 else q
        self.dq = DeviceArray.from_host(u if u.size else np.zeros(1, u.dtype))
        self.ld = max(total) + ld_more
        self.w0 = rng.random((len(lens) + 1, n_kv, self.ld), dtype=np.float32)
        self.dw = DeviceArray.from_host(self.w0)
        self.plan = E.WeightsPlan(self.caches, n_tokens, n_q, n_kv, starts=lens, dtype="bf16" if bf16 else "f32")

    def run(self, keep, layer=0, **kw):
        self.plan.run(layer, self.dq.ptr, self.dw.ptr, self.ld, keep, **kw)

    def check(self, keep, layer=0, w0=None):
        self.caches[0].sync()
        got, row = self.dw.download(), 0
        w0 = self.w0 if w0 is None else w0
        for i, (a, m) in enumerate(zip(self.lens, self.n)):
            t = a + m if m else 0
            assert np.array_equal(got[i, :, t:], w0[i, :, t:])      # behind the window as it was
            if m:
                want, tol = exact(self.caches[i], layer, self.q[row:row + m], a, self.n_q, self.n_kv)
                want += np.float64(np.float32(keep)) * w0[i, :, :t]
                tol += 3 * E32 * np.abs(want) + 1e-30
                err = np.abs(got[i, :, :t] - want)
                assert (err <= tol).all(), (float((err / tol).max()), i)
            row += m
        assert np.array_equal(got[-1], w0[-1])
        return got


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 128), (32, 4, 64), (3, 1, 128), (10, 2, 64), (40, 1, 128)])
@pytest.mark.parametrize("lens,n", [
    ([0], [1]), ([1, 30, 31, 32, 255, 256, 3], [1, 1, 1, 1, 1, 1, 0]), ([1000, 5, 0, 300], [4, 2, 33, 70]),
    ([4000, 700], [1, 1])])
def test_weights(E, rng, bf16, n_q, n_kv, d, lens, n):
    j = Job(E, rng, lens, n, n_q, n_kv, d, bf16)
    j.run(0.75)
    j.check(0.75)


def test_weights_overwrite_another_layer_and_repeat(E, rng):
    """keep 0 does not read what was there; a call's own workspace; the same bits again."""
    from eakv_amd import hipmem
    j = Job(E, rng, [600, 90], [2, 1], 8, 2, 128, False, layers=2)
    j.w0[:] = np.nan
    j.w0[-1] = 5.0
    j.dw.upload(j.w0)
    need = j.plan.work_bytes
    work = hipmem.DeviceArray((need,), np.uint8)
    st = hipmem.Stream()
    j.run(0.0, layer=1, d_work=work.ptr, work_bytes=need, stream=st.s)
    st.synchronize()
    got = j.dw.download()
    for i, (a, m) in enumerate(zip(j.lens, j.n)):
        want, tol = exact(j.caches[i], 1, j.q[2 * i:2 * i + m], a, 8, 2)
        assert (np.abs(got[i, :, :a + m] - want) <= tol).all()
        assert np.isnan(got[i, :, a + m:]).all()
        # rows of softmax weights: each adds up to 1
        assert np.abs(got[i, :, :a + m].sum(1, dtype=np.float64) - 4 * m).max() < 1e-4
    j.run(0.0, layer=1)
    j.caches[0].sync()
    assert np.array_equal(j.dw.download().view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
def test_weights_unseen_tokens_have_no_part(E, rng, bf16):
    """Non-finite keys behind the window's end (appended, not advanced), and one that the last
    query alone sees: its softmax is NaN, of every token, the other head's is not."""
    n_kv, d, n_q = 2, 128, 4
    j = Job(E, rng, [200], [10], n_q, n_kv, d, bf16)
    c = j.caches[0]
    c.append(np.full((n_kv, 2, d), np.inf, np.float32), 0, 0, 2)
    j.run(0.5)
    j.check(0.5)
    x = rng.standard_normal((n_kv, 1, d)).astype(np.float32)
    x[0, 0, 3] = np.inf
    c.restore(209)
    c.append(x, 0, 0, 1)
    c.advance(1)
    short = E.WeightsPlan([c], [9], n_q, n_kv, starts=[200], dtype="bf16" if bf16 else "f32")
    short.run(0, j.dq.ptr, j.dw.ptr, j.ld, 0.0)
    c.sync()
    assert np.isfinite(j.dw.download()[0, :, :209]).all()
    j.run(0.0)
    c.sync()
    got = j.dw.download()[0]
    assert np.isnan(got[0, :210]).all() and np.isfinite(got[1, :210]).all()


@pytest.mark.parametrize("scale", [30.0, 1e-3])
def test_weights_sharp_and_flat(E, rng, scale):
    j = Job(E, rng, [3000], [3], 8, 2, 64, False, scale=scale)
    j.run(1.0)
    j.check(1.0)


def choose(w, n, first, recent, keep):
    """The definition: positions of one sequence from weights [heads][..]."""
    with np.errstate(invalid="ignore", over="ignore"):
        score = w[:, :n].astype(np.float64)
        total = np.zeros(n)
        for h in range(len(score)):
            total = total + score[h]
        x = total.astype(np.float32)
    order = sorted(range(n), key=lambda t: (not (t < first or t >= n - recent), np.isnan(x[t]),
                                            -x[t] if not np.isnan(x[t]) else 0.0, t))
    return np.array(sorted(order[:keep]), np.int32)


class Choice:
    def __init__(self, E, w, n_tokens, first, recent, keep, kept=True):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.w, self.a = E, w, (n_tokens, first, recent, keep)
        self.dw = DeviceArray.from_host(w)
        self.total, self.ldk = sum(keep), max(keep) + 2
        self.index = DeviceArray((self.total + 1,), np.int32)
        self.kept = DeviceArray((w.shape[0], w.shape[1], self.ldk)) if kept else None
        self.need = E.lib().eakv_evict_select_work_bytes(len(keep), E.ints(n_tokens))
        self.work = DeviceArray((self.need + 4,), np.uint8)

    def clear(self):
        self.index.upload(np.full(self.total + 1, -9, np.int32))
        if self.kept:
            self.kept.upload(np.full(self.kept.shape, -9, np.float32))

    def run(self, stream=None):
        n, first, recent, keep = self.a
        E = self.E
        rc = E.lib().eakv_evict_select_device(
            len(keep), self.w.shape[1], self.dw.ptr, self.w.shape[2], E.ints(n), first, recent, E.ints(keep),
            self.index.ptr, self.kept.ptr if self.kept else None, self.ldk, self.work.ptr, self.need, stream)
        assert rc == 0, E.last_error()

    def check(self):
        from eakv_amd import hipmem
        hipmem.synchronize()
        n, first, recent, keep = self.a
        got = self.index.download()
        assert got[-1] == -9
        kept = self.kept.download() if self.kept else None
        at = 0
        for s, k in enumerate(keep):
            want = choose(self.w[s], n[s], first, recent, k)
            assert np.array_equal(got[at:at + k], want), (s, k)
            if kept is not None:
                assert np.array_equal(kept[s, :, :k].view(np.uint32), self.w[s][:, want].view(np.uint32))
                assert (kept[s, :, k:] == 0).all()
            at += k


def weights_of(rng, kind, n, heads, ld):
    if kind == "random":
        return np.exp(3 * rng.standard_normal((n, heads, ld))).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 4, (n, heads, ld)).astype(np.float32)
    if kind == "equal":
        return np.full((n, heads, ld), 0.25, np.float32)
    w = rng.standard_normal((n, heads, ld)).astype(np.float32)      # signs, zeros, infinities, NaN
    pick = rng.integers(0, 20, (n, heads, ld))
    for v, x in ((0, np.nan), (1, np.inf), (2, -np.inf), (3, 0.0), (4, -0.0), (5, 1e-42), (6, 3e38)):
        w[pick == v] = x
    return w


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "any"])
@pytest.mark.parametrize("n,first,recent,keep", [
    ([1], 0, 0, [1]), ([1, 5, 64], 1, 1, [0 + 1, 2, 64]), ([1000, 1025, 3, 0], 4, 100, [500, 104, 3, 0]),
    ([16384, 16000], 0, 0, [1, 8000]), ([2100] * 3, 4, 256, [2048, 2100, 260])])
def test_select(E, rng, kind, n, first, recent, keep):
    c = Choice(E, weights_of(rng, kind, len(n), 3, max(n) + 1), n, first, recent, keep)
    c.clear()
    c.run()
    c.check()


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "any"])
@pytest.mark.parametrize("n,first,recent,keep", [
    ([16385], 0, 0, [1]), ([20000, 100, 70001], 7, 500, [10000, 100, 600]), ([131072], 4, 0, [131071])])
def test_select_long(E, rng, kind, n, first, recent, keep):
    c = Choice(E, weights_of(rng, kind, len(n), 2, max(n)), n, first, recent, keep, kept=kind != "equal")
    for _ in range(2):
        c.clear()
        c.run()
        c.check()


@pytest.mark.parametrize("n", [3000, 40000])
def test_select_in_a_graph(E, rng, n):
    c = Choice(E, weights_of(rng, "random", 2, 2, n), [n, n - 7], 4, 64, [n // 2, n // 3])
    c.clear()
    from eakv_amd import hipmem
    hipmem.synchronize()
    g = W.Graph(c.run)
    for kind in ("ties", "random", "any"):
        c.w = weights_of(rng, kind, 2, 2, n)
        c.dw.upload(c.w)
        c.clear()
        hipmem.synchronize()
        g.launch()
        c.check()
        c.run()
        c.check()
    g.free()


def test_a_context_within_a_budget(E, rng):
    """Decode with weights taken at every step; past the budget the choice, the gather in place and the
    weights in their new places; the attention afterwards is that of the tokens kept."""
    from eakv_amd.hipmem import DeviceArray
    n_q, n_kv, d, budget, room = 8, 2, 64, 60, 100
    caches = W.build(E, rng, [40, 55], n_kv, d, room)
    ld = room
    w = [DeviceArray.from_host(np.zeros((2, n_kv, ld), np.float32)) for _ in (0, 1)]
    exact_w = [np.zeros((n_kv, ld)) for _ in caches]
    for step in range(25):
        x = rng.standard_normal((2, 1, 2, n_kv, 1, d)).astype(np.float32)
        dx = DeviceArray.from_host(x)
        h = E.handles(caches)
        assert E.lib().eakv_append_batch_device(h, 2, dx.ptr, 1, None) == 0
        starts = [c.seq_len for c in caches]
        q = rng.standard_normal((2, n_q, d)).astype(np.float32)
        dq = DeviceArray.from_host(q)
        E.WeightsPlan(caches, [1, 1], n_q, n_kv, starts=starts).run(0, dq.ptr, w[0].ptr, ld, 0.9)
        for i, c in enumerate(caches):
            c.advance(1)
            t = starts[i] + 1
            exact_w[i][:, :t] = np.float64(np.float32(0.9)) * exact_w[i][:, :t] + \
                exact(c, 0, q[i:i + 1], t - 1, n_q, n_kv)[0]
        n = [c.seq_len for c in caches]
        if max(n) < 64:
            continue
        keep = [min(k, budget) for k in n]
        caches[0].sync()
        index = DeviceArray((sum(keep),), np.int32)
        rc = E.lib().eakv_evict_select_device(2, n_kv, w[0].ptr, ld, E.ints(n), 4, 16, E.ints(keep), index.ptr,
                                              w[1].ptr, ld, None, 0, caches[0].stream)
        assert rc == 0, E.last_error()
        before = [[W.values(c, 0, j)[0] for j in (0, 1)] for c in caches]
        rc = E.lib().eakv_cache_gather_batch_device(h, h, 2, E.ints([0, 0]), index.ptr, E.ints(keep), None)
        assert rc == 0, E.last_error()
        caches[0].sync()
        lists = np.split(index.download(), [keep[0]])
        for i, c in enumerate(caches):
            assert np.array_equal(lists[i][:4], np.arange(4)) and lists[i][-1] == n[i] - 1
            assert np.array_equal(lists[i][-16:], np.arange(n[i] - 16, n[i]))
            c.restore(keep[i])
            for j in (0, 1):
                assert np.array_equal(W.values(c, 0, j)[0][:, :keep[i]], before[i][j][:, lists[i]])
            exact_w[i][:, :keep[i]] = exact_w[i][:, lists[i]]
            exact_w[i][:, keep[i]:] = 0.0
        w.reverse()
    got = w[0].download()
    for i, c in enumerate(caches):
        t = c.seq_len
        assert t <= 64
        # 25 steps' bounds: A is below 100 here
        assert np.abs(got[i, :, :t] - exact_w[i][:, :t]).max() < 25 * 80 * E32 * 100


def test_weights_in_a_graph(E, rng):
    from eakv_amd import hipmem
    j = Job(E, rng, [500, 40], [1, 3], 8, 2, 128, True)
    need = j.plan.work_bytes
    work = hipmem.DeviceArray((need,), np.uint8)
    hipmem.synchronize()
    g = W.Graph(lambda st: j.run(0.5, d_work=work.ptr, work_bytes=need, stream=st))
    for _ in range(3):
        w0 = rng.random(j.w0.shape, dtype=np.float32)
        j.dw.upload(w0)
        hipmem.synchronize()
        g.launch()
        j.check(0.5, w0=w0)
        j.run(0.5)
        j.caches[0].sync()
    g.free()
    with pytest.raises(E.EakvError):
        W.Graph(lambda st: j.run(0.5, stream=st))
