"""Gathers whose pairs differ: in place beside another cache, with lists of every length."""
import numpy as np
import pytest

from test_gpu_move import E, filled, planes  # noqa: F401  (E: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [(1500, 1500, 700), (0, 1400, 3), (1, 0, 2000), (2000, 513, 0)])
def test_in_place_beside_another_cache(E, rng, d, n):
    """One pair in place (ascending), two into other caches (any order, positions twice)
    from sources that are shared."""
    from eakv_amd.hipmem import DeviceArray
    room = 2100
    a, b, c, e = (filled(E, rng, 2, 2, d, room) for _ in range(4))
    print("gather mixed", d, n, flush=True)
    lists = [np.sort(rng.choice(np.arange(30, room), n[0], replace=False)).astype(np.int32),
             rng.integers(0, room, n[1]).astype(np.int32), rng.integers(0, room, n[2]).astype(np.int32)]
    at = (30, 0, 5)
    srcs, dsts = [a, b, b], [a, c, e]
    before = [planes(x) for x in (a, b, c, e)]
    pa, pb, pc, pe = (x.copy() for x in before)
    pa[:, :, :, 30:30 + n[0]] = before[0][:, :, :, lists[0]]
    pc[:, :, :, :n[1]] = before[1][:, :, :, lists[1]]
    pe[:, :, :, 5:5 + n[2]] = before[1][:, :, :, lists[2]]
    di = DeviceArray.from_host(np.concatenate(lists))
    assert E.lib().eakv_cache_gather_batch_device(E.handles(srcs), E.handles(dsts), 3, E.ints(at), di.ptr,
                                                  E.ints(n), None) == 0, E.last_error()
    a.sync()
    for x, want in zip((a, b, c, e), (pa, pb, pc, pe)):
        assert np.array_equal(planes(x), want)


def test_compact_to_the_recent_tokens(E, rng):
    """The commonest list: the first tokens and the last, longer than what lies between."""
    c = filled(E, rng, 1, 2, 128, 5000)
    p = planes(c)
    keep = np.concatenate([np.arange(4), np.arange(1000, 5000)])
    c.compact(keep)
    assert c.seq_len == 4004
    assert np.array_equal(planes(c)[:, :, :, :4004], p[:, :, :, keep])
