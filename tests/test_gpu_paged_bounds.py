"""Calls over pages at the ends of what their 32-bit counts hold.  Refusals are made on the host:
addresses stand for buffers and nothing is launched."""
import ctypes as C

import pytest

from test_gpu_paged_evict_refusals import BASE, N_KV, batch

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


@pytest.mark.parametrize("d", [64, 128])
def test_append_of_the_most_rows(E, d):
    """2^31 - 1 rows are an error of the call's, no arithmetic fault on the host."""
    pool = E.Cache(1, N_KV, d, 4096)
    s = batch(E, n_new=INT_MAX, max_new=INT_MAX)
    rc = E.lib().eakv_append_paged_device(pool.h, C.addressof(s), 0, BASE + (1 << 24), BASE + (2 << 24), 1, N_KV * d,
                                          None)
    assert rc < 0 and E.last_error()[0] == rc and E.last_error()[1]
    E.lib().eakv_clear_error()
