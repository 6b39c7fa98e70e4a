"""Log probabilities of given tokens, entropies and alternatives (eakv_token_logprobs_device)
against 64 bits.

Bounds, e = 2^-24 half a step of f32: a term's exponent (x - M) log2(e) is off by 2 e of it
(difference, product), so a term e^(x - M) by 2 e |x - M| + 2 e of itself, at most 1 e of the
sum where it counts (u e^-u <= 0.37), and with the adding of 64 values in a lane, 6 steps over a
wave and 4 waves (74 roundings of partial sums) ln S is off by at most 80 e.  A log
probability adds half a step of itself: 80 e + e |lp|.  T = sum p z is off by 84 e of sum
p |z|, and H = ln S - ln2 T / S by 80 e + (84 + 80) e H' + e H, H' = sum p |x - M| <= H."""
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


class Job:
    def __init__(self, E, x, vocab, tokens, top, bf16, shift=0, rows=None):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.vocab, self.k, self.bf16 = E, vocab, top, bf16
        self.n, self.ld = x.shape
        u = W.to_bf16(x) if bf16 else np.ascontiguousarray(x, np.float32)
        if bf16:
            u = np.where(np.isnan(x), np.uint16(0x7fc0), u)
        self.x = W.from_bf16(u) if bf16 else u
        self.size, self.shift = u.itemsize, shift
        pad = np.full(8, 0x7fc0 if bf16 else np.nan, u.dtype)
        self.dx = DeviceArray.from_host(np.concatenate([pad[:shift], u.reshape(-1), pad]))
        self.tokens = np.asarray(tokens, np.int32)
        self.dt = DeviceArray.from_host(self.tokens)
        self.out = [DeviceArray((self.n + 1,)), DeviceArray((self.n + 1,)),
                    DeviceArray((self.n * top + 1,), np.int32), DeviceArray((self.n * top + 1,))]
        self.need = E.lib().eakv_token_logprobs_work_bytes(self.n, vocab, top)
        self.work = DeviceArray((self.need + 16,), np.uint8)

    def run(self, stream=None, want=(1, 1, 1)):
        for o in self.out:
            o.upload(np.full(o.shape, -7, o.dtype))
        self.call(stream, want)

    def call(self, stream=None, want=(1, 1, 1)):
        p = [o.ptr for o in self.out]
        rc = self.E.lib().eakv_token_logprobs_device(
            self.n, self.vocab, self.dx.ptr + self.shift * self.size, 1 if self.bf16 else 0, self.ld,
            self.dt.ptr if want[0] else None, self.k if want[2] else 0, p[0] if want[0] else None,
            p[1] if want[1] else None, p[2], p[3], self.work.ptr, self.need, stream)
        assert rc == 0, self.E.last_error()

    def check(self, want=(1, 1, 1)):
        from eakv_amd import hipmem
        hipmem.synchronize()
        lp, ent, tok, tlp = [o.download() for o in self.out]
        for o in (lp, ent, tok, tlp):
            assert o[-1] == -7
        if not want[0]:
            assert (lp == -7).all()
        if not want[1]:
            assert (ent == -7).all()
        x = self.x[:, :self.vocab].astype(np.float64)
        for r in range(self.n):
            with np.errstate(all="ignore"):
                m = x[r].max()
                z = x[r] - m
                s = np.exp(z).sum()
                ls = np.log(s)
                h1 = -np.where(z > -np.inf, np.exp(z) * z, 0).sum() / s
            t = int(self.tokens[r])
            if want[0]:
                want_lp = z[t] - ls if 0 <= t < self.vocab else -np.inf
                self.near(lp[r], want_lp, 80 * E32)
            if want[1]:
                self.near(ent[r], ls + h1, (80 + 164 * h1) * E32)
            if want[2] and self.k:
                ok = np.nonzero(x[r] > -np.inf)[0]
                order = ok[np.argsort(-x[r, ok], kind="stable")][:self.k]
                row = tok[r * self.k:(r + 1) * self.k]
                assert np.array_equal(row[:len(order)], order), (r, row, order)
                assert (row[len(order):] == -1).all()
                got = tlp[r * self.k:(r + 1) * self.k]
                for a, i in zip(got, order):
                    self.near(a, z[i] - ls, 80 * E32)
                assert (got[len(order):] == -np.inf).all()

    @staticmethod
    def near(got, want, tol):
        if np.isnan(want):
            assert np.isnan(got), (got, want)
        elif np.isinf(want):
            assert got == want, (got, want)
        else:
            assert abs(float(got) - want) <= tol + E32 * abs(want), (got, want)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,vocab,ld,top,shift", [
    (1, 1, 1, 1, 0), (3, 2, 7, 5, 1), (4, 63, 63, 32, 0), (5, 1000, 1003, 7, 3), (2, 16377, 16377, 20, 7),
    (2, 16384, 16384, 20, 0), (2, 16385, 16391, 32, 5), (3, 50257, 50257, 0, 0), (5, 151665, 151665, 20, 0),
    (1, 700001, 700001, 32, 2)])
def test_logprobs(E, rng, bf16, n, vocab, ld, top, shift):
    x = (rng.standard_normal((n, ld)) * 3).astype(np.float32)
    j = Job(E, x, vocab, rng.integers(0, vocab, n), top, bf16, shift)
    j.run()
    j.check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", [300, 40000])
def test_rows_of_all_kinds(E, rng, bf16, vocab):
    """Equal values, ties at the bound, one allowed token, some, none, NaN, infinities, sharp rows, far
    offsets, values sorted so that one lane has the largest, both zeros."""
    n = 14
    x = rng.standard_normal((n, vocab)).astype(np.float32)
    x[0] = 0.0
    x[1] = np.round(x[1])
    x[2] = -np.inf
    x[2, vocab // 2] = 1.5
    x[3, rng.random(vocab) < 0.99] = -np.inf
    x[4] = -np.inf
    x[5, vocab - 1] = np.nan
    x[6, 7] = np.inf
    x[7, 11] = 60.0
    x[8] += 1000.0
    x[9] -= 3e4
    x[10, :] = 0.0
    x[10, 4 if not bf16 else 8::1024 if not bf16 else 2048] = 5.0 + np.arange(len(x[10, 4 if not bf16 else 8::1024 if not bf16 else 2048]))
    x[11] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[12] = -np.abs(x[12]) * 1e30
    x[13] *= 1e-20
    tokens = rng.integers(0, vocab, n)
    tokens[0], tokens[1], tokens[3] = -1, vocab, 1 << 30
    tokens[2] = vocab // 2
    tokens[7] = 11
    j = Job(E, x, vocab, tokens, 32, bf16)
    j.run()
    j.check()


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)])
def test_some_results(E, rng, want):
    j = Job(E, rng.standard_normal((3, 20000)).astype(np.float32), 20000, [1, 2, 3], 5, False)
    j.run(want=want)
    j.check(want)


def test_in_a_graph_and_with_many_equal_values(E, rng):
    from eakv_amd import hipmem
    j = Job(E, rng.standard_normal((4, 33000)).astype(np.float32), 33000, [5, 6, 7, 8], 20, True)
    j.run()
    hipmem.synchronize()
    g = W.Graph(lambda st: j.call(st))
    for k in range(3):
        x = np.round(rng.standard_normal((4, 33000)) * (10 ** k)).astype(np.float32)
        u = W.to_bf16(x)
        j.x = W.from_bf16(u)
        j.dx.upload(np.concatenate([u.reshape(-1), np.full(8, 0x7fc0, np.uint16)]))
        hipmem.synchronize()
        g.launch()
        j.check()
        first = [o.download() for o in j.out]
        j.run()
        j.check()
        for a, b in zip(first, j.out):
            assert np.array_equal(a, b.download())
    g.free()


def test_answers_of_the_target_beside_its_verification(E, rng):
    """The tokens that a verification keeps, with their log probabilities: one set of logits, its softmax to
    eakv_verify_drafts_device and itself here."""
    from eakv_amd import hipmem
    from eakv_amd.hipmem import DeviceArray
    n, k, v = 3, 4, 5000
    logits = (rng.standard_normal((n, k + 1, v)) * 4).astype(np.float32)
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p = (p / p.sum(-1, keepdims=True)).astype(np.float32)
    tokens = logits[:, :k].argmax(-1).astype(np.int32)
    u = rng.random((n, k + 1), dtype=np.float32)
    d = [DeviceArray.from_host(a) for a in (tokens, p, u)]
    kept, nxt = DeviceArray((n,), np.int32), DeviceArray((n,), np.int32)
    size = E.lib().eakv_verify_drafts_work_bytes(n, k, v)
    work = DeviceArray((size,), np.uint8)
    assert E.lib().eakv_verify_drafts_device(n, k, v, None, d[0].ptr, None, 0, d[1].ptr, v, d[2].ptr, kept.ptr,
                                             nxt.ptr, work.ptr, size, None) == 0
    hipmem.synchronize()
    a, nx = kept.download(), nxt.download()
    given = np.concatenate([tokens, nx[:, None]], 1)
    given[np.arange(n), a] = nx
    j = Job(E, logits.reshape(-1, v), v, given.reshape(-1), 3, False)
    j.run()
    j.check()
    lp = j.out[0].download()[:-1].reshape(n, k + 1)
    for s in range(n):
        for i in range(a[s] + 1):
            assert abs(lp[s, i] - np.log(p[s, i, given[s, i]].astype(np.float64))) < 1e-5
