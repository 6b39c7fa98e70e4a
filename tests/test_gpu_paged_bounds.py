"""Calls over pages at the ends of what their 32-bit counts hold.  Refusals are made on the host:
addresses stand for buffers and nothing is launched."""
import ctypes as C

import numpy as np
import pytest

import paging as P
import windows as W
from test_gpu_paged_evict_refusals import BASE, D, N_KV, N_Q, ROOM, batch, refused

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


@pytest.mark.parametrize("max_len,n_new", [(INT_MAX, 1), (2 ** 31 - 65535, 1), (16, INT_MAX)])
def test_positions_that_pass_32_bits_are_refused(E, max_len, n_new):
    """A bound so near 2^31 that the places looked up behind a sequence's end are not 32 bits."""
    pool = E.Cache(1, N_KV, D, ROOM)
    L = E.lib()
    s = batch(E, n_seqs=1, n_new=n_new, max_new=1, max_len=max_len, ld=1 << 30)
    assert L.eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, N_KV, N_KV) == 0
    assert refused(E, E.EAKV_ERR_INVALID)
    a = BASE + (1 << 40)
    assert refused(E, L.eakv_attention_paged_device(pool.h, C.addressof(s), 0, a, N_Q * D, 1, N_KV, N_KV, a, N_Q * D, None,
                                                    0, None))
    assert refused(E, L.eakv_append_paged_device(pool.h, C.addressof(s), 0, a, a, 1, N_KV * D, None))


def test_the_longest_bound_is_accepted(E):
    pool = E.Cache(1, N_KV, D, ROOM)
    s = batch(E, n_seqs=1, n_new=1, max_new=1, max_len=2 ** 31 - 65536, ld=1 << 30)
    assert E.lib().eakv_attention_paged_work_bytes(pool.h, C.addressof(s), 1, N_KV, N_KV) > 0
    assert E.lib().eakv_last_error() == E.EAKV_OK


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [2, 64, 70, 300])
@pytest.mark.parametrize("large", [False, True])
def test_rows_of_a_list_that_falls_are_left_alone(E, rng, bf16, n, large):
    """Its sequences would share rows, and their work together might be more than the call counts
    (2048 sequences of 4096 new tokens each: a line of 2.8e9 tiles)."""
    from eakv_amd.hipmem import DeviceArray
    p = P.Pool(E, rng, [40] * n, [4] * n, 16, 2, 64, ld_more=(1 << 22) // (4 * n) if large else 0)
    p.fill(P.contents(rng, p))
    c = P.Call(p, 8, 2, bf16)
    c.put(rng.standard_normal((p.rows, 8, 64)).astype(np.float32))
    kw = dict(max_len=(1 << 24) // p.rows + 1, max_new=p.rows) if large else {}
    lists = [np.arange(n + 1) % 2 * p.rows, np.arange(n, -1, -1), p.first + (np.arange(n + 1) == n - 1) * p.rows]
    for x in lists:
        first = DeviceArray.from_host(x.astype(np.int32))
        c.run(batch=p.make(d_first=first.ptr, **kw))
        got = c.get()
        guard = np.frombuffer(bytes([c.GUARD]) * 4, np.float32)[0] if not bf16 else W.from_bf16(
            np.array([c.GUARD * 257], np.uint16))[0]
        assert (got == guard).all()
    c.run()                                             # (the pool's own list)
    assert np.isfinite(c.get()).all()
