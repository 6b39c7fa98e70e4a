"""Verification of drafts whose distributions hold negative values, NaN and infinities
(eakv_verify_drafts_device): negative values and NaN count as 0."""
import numpy as np
import pytest

from test_gpu_verify import E, Job, expect, inputs  # noqa: F401  (E: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [700, 12288, 12289, 70001])
def test_values_that_count_as_nothing(E, rng, vocab):
    n, k = 24, 3
    tokens, draft, target, u = inputs(rng, n, k, vocab)
    pick = rng.random(draft.shape)
    # weights that, if taken as they stand, would decide most of the drawn tokens
    draft[pick < 0.3] = -0.5
    draft[(pick >= 0.3) & (pick < 0.5)] = np.nan
    pick = rng.random(target.shape)
    target[pick < 0.2] = -0.5
    target[(pick >= 0.2) & (pick < 0.3)] = np.nan
    tokens[:8, 0] = np.argmax(np.isnan(draft[:8, 0]), 1)          # q(x) NaN: 0, kept where p(x) > 0
    tokens[8:16, 0] = np.argmax(draft[8:16, 0] < 0, 1)
    job = Job(E, None, tokens, draft, target, u, vocab)
    job.clear()
    job.run()
    a, b = job.get()
    with np.errstate(invalid="ignore"):
        q, p = np.where(draft > 0, draft, np.float32(0)), np.where(target > 0, target, np.float32(0))
    wa, wb = expect(None, tokens, q, p, u, vocab)
    assert np.array_equal(a, wa) and np.array_equal(b, wb), (a, wa, b, wb)
    # what a token is drawn from is positive
    assert (p[np.arange(n), a, b] > 0).all()
