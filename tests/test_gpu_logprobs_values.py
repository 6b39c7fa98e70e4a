"""Log probabilities where their sums are hardest.

Bounds, e = 2^-24, H the row's entropy: (24 + 4 H) e and half a step for ln p, (24 + 128 H) e and half
a step for H.  A term is off by 2 e (its exponential), e u 1.3 (its exponent's rounding and that of
log2(e); u = M - x) or, by differences, e u 2.3, and e u 1 by its segment's factor, itself 2 e off.  A
lane adds 8 terms 8 times, then 3, 6 and 2 steps: 18 roundings.  sum p u <= H, so ln S is off by
(18 + 2 + 2 + 3.3 H) e.  T, the sum of p u, by (18 + 1 + 2 + 2 + 1) e H and 3.3 e sum p u^2, and as 2^30
terms beyond u = 30 hold less than 1e-3, sum p u^2 <= 30 H and little: together
(22 + (3.3 + 24 + 99) H) e."""
import numpy as np
import pytest

from test_gpu_logprobs import Job
from windows import E32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", [300, 20000])
@pytest.mark.parametrize("rest", [-np.inf, -200.0, -17.0])
def test_no_probability_above_one(E, rng, bf16, vocab, rest):
    """The largest logit's own term is 1, so that S >= 1: no ln p above 0, no entropy below."""
    n = 400
    top = rng.uniform(-40.0, 40.0, n).astype(np.float32)
    at = rng.integers(0, vocab, n)
    x = np.full((n, vocab), rest, np.float32)
    if np.isfinite(rest):
        x += top[:, None]
    x[np.arange(n), at] = top
    j = Job(E, x, vocab, at, 3, bf16)
    j.run()
    j.check()
    lp, ent, _, tlp = [o.download()[:-1] for o in j.out]
    assert (lp <= 0.0).all(), float(lp.max())
    assert (tlp <= 0.0).all(), float(tlp.max())
    assert (ent >= 0.0).all(), float(ent.min())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", [16001, 130001])
@pytest.mark.parametrize("away", [0.0, 3e6])
def test_many_equal_logits_below_the_largest(E, rng, bf16, vocab, away):
    """Terms whose roundings are all alike, within what the header says; also of rows far from 0."""
    n = 64
    x = np.empty((n, vocab), np.float32)
    top = rng.uniform(-30.0, 30.0, n) + away
    x[:] = (top - rng.uniform(7.0, 14.0, n))[:, None]
    at = rng.integers(0, vocab, n)
    x[np.arange(n), at] = top
    tokens = np.where(np.arange(n) % 2, at, (at + 1) % vocab)
    j = Job(E, x, vocab, tokens, 2, bf16)
    j.run()
    j.check()
    lp, ent = [o.download()[:-1].astype(np.float64) for o in j.out[:2]]
    y = j.x.astype(np.float64)
    z = y - y.max(1, keepdims=True)
    p = np.exp(z)
    s = p.sum(1)
    want, h = z[np.arange(n), tokens] - np.log(s), np.log(s) - (p * z).sum(1) / s
    assert (np.abs(lp - want) <= ((24 + 4 * h) + np.abs(want)) * E32).all()
    assert (np.abs(ent - h) <= ((24 + 128 * h) + h) * E32).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", [65 * 16384 - 7, 2150001])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_rows_of_many_segments(E, rng, bf16, vocab, top):
    """More segments than a wave has lanes (65 and 132): the largest and the given token behind the
    64th, segments of nothing but -inf before and behind it."""
    seg = 16384
    x = (rng.standard_normal((3, vocab)) * 3).astype(np.float32)
    tokens = np.array([64 * seg + 77, 5, vocab - 1])
    x[0, tokens[0]] = 30.0                              # the largest and the given one: behind the 64th
    x[1, 64 * seg + 1000] = 40.0
    x[1, 2 * seg - 50:9 * seg + 50] = -np.inf
    x[2, :64 * seg + 100] = -np.inf                     # all there is is behind the 64th
    x[2, 40 * seg] = 1.0
    j = Job(E, x, vocab, tokens, top, bf16)
    j.run()
    j.check()
