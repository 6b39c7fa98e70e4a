"""Drafted tokens against the target's probabilities (eakv_verify_drafts_device)
against its definition in 64 bits.  Whole numbers: they have to be equal.  (Sums in
another order move a step by 1e-15 of the row's sum, so a drawn number meets one with
a probability of about 1e-10 per case; the cases are seeded.)"""
import numpy as np
import pytest

import windows as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


def expect(counts, tokens, draft, target, uniform, vocab):
    n, k1 = uniform.shape
    k = k1 - 1
    kept, nxt = [], []
    for s in range(n):
        c = k if counts is None else max(0, min(k, int(counts[s])))
        a = 0
        while a < c:
            x = int(tokens[s, a])
            if not 0 <= x < vocab:
                break
            p = float(target[s, a, x])
            q = 1.0 if draft is None else float(draft[s, a, x])
            if not float(uniform[s, a]) * q < p:
                break
            a += 1
        p = target[s, a, :vocab].astype(np.float64)
        p = np.where(p > 0, p, 0.0)
        r = p
        if a < c:
            if draft is None:
                r = p.copy()
                if 0 <= tokens[s, a] < vocab:
                    r[tokens[s, a]] = 0.0
            else:
                with np.errstate(invalid="ignore"):
                    r = target[s, a, :vocab].astype(np.float64) - draft[s, a, :vocab]
                r = np.where(r > 0, r, 0.0)
        if not r.sum() > 0:
            r = p
        kept.append(a)
        if not r.sum() > 0:
            nxt.append(-1)
            continue
        upto = np.cumsum(r)
        over = np.nonzero((upto > float(uniform[s, k]) * upto[-1]) & (r > 0))[0]
        nxt.append(int(over[0]) if over.size else int(np.nonzero(r > 0)[0][-1]))
    return np.array(kept, np.int32), np.array(nxt, np.int32)


class Job:
    def __init__(self, E, counts, tokens, draft, target, uniform, vocab):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.vocab = E, vocab
        self.n, k1 = uniform.shape
        self.k = k1 - 1
        self.bufs = [None if a is None else DeviceArray.from_host(a)
                     for a in (counts, tokens, draft, target, uniform)]
        self.ld = [0 if a is None else a.shape[-1] for a in (draft, target)]
        self.kept, self.next = (DeviceArray((self.n + 1,), np.int32) for _ in range(2))
        self.size = E.lib().eakv_verify_drafts_work_bytes(self.n, self.k, vocab)
        assert self.size > 0
        self.work = DeviceArray((self.size,), np.uint8)

    def run(self, stream=None):
        c, t, d, p, u = (0 if b is None else b.ptr for b in self.bufs)
        rc = self.E.lib().eakv_verify_drafts_device(
            self.n, self.k, self.vocab, c, t, d, self.ld[0], p, self.ld[1], u, self.kept.ptr,
            self.next.ptr, self.work.ptr, self.size, stream)
        assert rc == 0, self.E.last_error()

    def get(self):
        from eakv_amd import hipmem
        hipmem.synchronize()
        a, b = self.kept.download(), self.next.download()
        assert a[-1] == 77 and b[-1] == 77          # behind the last sequence
        return a[:-1], b[:-1]

    def clear(self):
        for x in (self.kept, self.next):
            x.upload(np.full(self.n + 1, 77, np.int32))


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def inputs(rng, n, k, vocab, onehot=False, pad=0, sharp=2.0):
    logits = (rng.standard_normal((n, k + 1, vocab + pad)) * sharp).astype(np.float32)
    target = softmax(logits)
    draft = softmax(logits[:, :k] + 0.6 * rng.standard_normal((n, k, vocab + pad)).astype(np.float32))
    u = rng.random((n, k, 1))
    tokens = (draft[..., :vocab].cumsum(-1) < u * draft[..., :vocab].sum(-1, keepdims=True)).sum(-1)
    tokens = np.minimum(tokens, vocab - 1).astype(np.int32)
    return tokens, None if onehot else draft, target, rng.random((n, k + 1), dtype=np.float32)


@pytest.mark.parametrize("onehot", [False, True])
@pytest.mark.parametrize("n,k,vocab,pad", [
    (1, 1, 1, 0), (3, 2, 3, 1), (5, 4, 1023, 0), (2, 7, 1025, 3), (9, 3, 4097, 0), (4, 5, 32000, 0),
    (64, 4, 5000, 1), (300, 2, 777, 0), (2, 1, 270001, 0), (3, 70, 500, 0), (6, 0, 900, 0),
    (40, 3, 110001, 0), (3, 4, 16384, 0), (2, 3, 16385, 2), (7, 2, 32768, 1), (5, 2, 32769, 0),
    (130, 2, 12288, 0), (9, 2, 12289, 1), (4, 3, 4095, 1), (1, 2, 256, 0)])
def test_against_definition(E, rng, n, k, vocab, pad, onehot):
    print("verify", n, k, vocab, pad, onehot, flush=True)
    tokens, draft, target, u = inputs(rng, n, k, vocab, onehot, pad)
    if k == 0:
        tokens, draft = None, None
    for counts in (None, rng.integers(-1, k + 2, n).astype(np.int32)):
        job = Job(E, counts, tokens, draft, target, u, vocab)
        job.clear()
        job.run()
        a, b = job.get()
        wa, wb = expect(counts, tokens, draft, target, u, vocab)
        assert np.array_equal(a, wa) and np.array_equal(b, wb)


def test_edges(E, rng):
    """Equal distributions, empty rows, NaN and negative values, tokens outside the
    vocabulary, drawn numbers 0 and just below 1, weight on one token."""
    n, k, v = 12, 3, 2050
    tokens, draft, target, u = inputs(rng, n, k, v)
    draft[0] = target[0, :k]                     # all kept
    target[1] = 0.0                              # nothing anywhere
    u[2, 0] = 0.999                              # rejected, and nothing left of p - q: p itself
    draft[2, 0] = 2 * target[2, 0]
    target[3, :, ::2] = np.nan
    target[3, :, 1] = -1.0
    tokens[4] = [v, -1, 5]
    tokens[5, 1] = 2147483647
    u[6, k], u[7, k] = 0.0, np.float32(1 - 2 ** -24)
    target[8] = 0.0
    target[8, :, v - 1] = 1.0
    tokens[8] = v - 1
    u[8] = np.float32(1 - 2 ** -24)
    target[9] = 0.0
    target[9, :, 0] = 1.0
    u[9, k] = 0.0
    draft[10, :, :] = 0.0                        # q(x) = 0: kept where p > 0
    u[11] = 0.0
    for d in (draft, None):
        job = Job(E, None, tokens, d, target, u, v)
        job.clear()
        job.run()
        a, b = job.get()
        wa, wb = expect(None, tokens, d, target, u, v)
        assert np.array_equal(a, wa) and np.array_equal(b, wb), (a, wa, b, wb)
    assert wb[1] == -1 and wa[1] == 0


def test_distribution(E):
    """The token at the first position (kept draft, or the one drawn in its place) is
    distributed as the target's row, whatever the draft's: 40,000 sequences of one
    distribution, each frequency within 5 standard deviations."""
    rng = np.random.default_rng(5)
    n, v = 40000, 8
    p, q = softmax(rng.standard_normal(v)), softmax(rng.standard_normal(v))
    tokens = rng.choice(v, size=(n, 1), p=q / q.sum(dtype=np.float64)).astype(np.int32)
    target = np.broadcast_to(p, (n, 2, v)).copy()
    draft = np.broadcast_to(q, (n, 1, v)).copy()
    job = Job(E, None, tokens, draft, target, rng.random((n, 2), dtype=np.float32), v)
    job.clear()
    job.run()
    a, b = job.get()
    got = np.bincount(np.where(a == 1, tokens[:, 0], b), minlength=v) / n
    assert (np.abs(got - p) < 5 * np.sqrt(p * (1 - p) / n)).all()


def test_recorded_in_a_graph(E, rng):
    jobs = []
    for n, v in ((5, 3001), (3, 900)):
        tokens, draft, target, u = inputs(rng, n, 4, v)
        jobs.append((Job(E, None, tokens, draft, target, u, v), tokens, draft, target))
    graphs = [W.Graph(lambda s, j=j: j.run(s)) for j, *_ in jobs]
    for _ in range(3):
        for (j, tokens, draft, target), g in zip(jobs, graphs):
            u = rng.random((j.n, 5), dtype=np.float32)
            j.bufs[4].upload(u)
            j.clear()
            g.launch()
            a, b = j.get()
            wa, wb = expect(None, tokens, draft, target, u, j.vocab)
            assert np.array_equal(a, wa) and np.array_equal(b, wb)
    for g in graphs:
        g.free()
