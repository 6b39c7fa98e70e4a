"""Calls over pages at the ends of what their 32-bit counts hold.  Refusals are made on the host:
addresses stand for buffers and nothing is launched."""
import ctypes as C

import pytest

from test_gpu_paged_evict_refusals import BASE, N_KV, batch, refused

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


@pytest.mark.parametrize("d,most", [(64, 2 ** 29 - 32), (128, 2 ** 28 - 16)])
def test_append_of_too_many_rows_is_refused(E, d, most):
    """As an argument, before streams are ordered (a NULL K behind it is refused too, but later)."""
    pool = E.Cache(1, N_KV, d, 4096)
    for n in (most + 1, INT_MAX):
        s = batch(E, n_new=n, max_new=n)
        for k in (BASE + (1 << 24), None):
            rc = E.lib().eakv_append_paged_device(pool.h, C.addressof(s), 0, k, BASE + (2 << 24), 1, N_KV * d, None)
            assert "rows" in E.last_error()[1] and refused(E, rc)
    s = batch(E, n_new=most, max_new=most)
    rc = E.lib().eakv_append_paged_device(pool.h, C.addressof(s), 0, None, BASE + (2 << 24), 1, N_KV * d, None)
    assert "NULL" in E.last_error()[1] and refused(E, rc)
