"""Log probabilities where their sums are hardest.  Bounds: test_gpu_logprobs.py."""
import numpy as np
import pytest

from test_gpu_logprobs import Job

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
