"""The choice of kept tokens on either side of where its kernels change: 4096 tokens and 8192 of one
launch, and the heads that a thread takes at once."""
import numpy as np
import pytest

from test_gpu_evict import Choice, weights_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "any"])
@pytest.mark.parametrize("heads,kept", [(3, True), (4, True), (5, True), (8, True), (9, True), (17, True), (9, False)])
@pytest.mark.parametrize("n,first,recent,keep", [
    ([4096], 4, 32, [3000]), ([4097, 10], 0, 0, [4096, 1]), ([8191, 4096, 0, 300], 7, 500, [600, 4000, 0, 300]),
    ([8192, 5000], 4, 64, [8192, 4999]), ([8192], 0, 0, [1]), ([8193, 70], 4, 64, [5000, 68])])
def test_select_where_kernels_change(E, rng, kind, heads, kept, n, first, recent, keep):
    c = Choice(E, weights_of(rng, kind, len(n), heads, max(n) + 1), n, first, recent, keep, kept)
    c.clear()
    c.run()
    c.check()
