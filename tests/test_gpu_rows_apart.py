"""Rows of weights that are parts of larger ones (a layer's of [head][layer][token]): what lies behind the
last of a call's rows is another buffer's."""
import numpy as np
import pytest

import test_gpu_evict as EV
import windows as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


LAYERS = 3


def test_choice_from_a_layer_s_weights(E, rng):
    """The list stands right behind the weights of all layers, the kept weights behind it."""
    from eakv_amd import hipmem
    heads, n, keep = 2, 512, 100
    w = rng.random((heads, LAYERS, n), dtype=np.float32)
    room = w.nbytes + keep * 4 + heads * keep * 4
    buf = hipmem.DeviceArray.from_host(np.concatenate([w.reshape(-1).view(np.uint8),
                                                       np.full(room - w.nbytes, 0x7b, np.uint8)]))
    for layer in range(LAYERS):
        rc = E.lib().eakv_evict_select_device(
            1, heads, buf.ptr + layer * n * 4, LAYERS * n, E.ints([n]), 4, 16, E.ints([keep]), buf.ptr + w.nbytes,
            buf.ptr + w.nbytes + keep * 4, keep, None, 0, None)
        assert rc == 0, (layer, E.last_error())
        hipmem.synchronize()
        host = buf.download()
        want = EV.choose(w[:, layer], n, 4, 16, keep)
        assert np.array_equal(host[w.nbytes:w.nbytes + keep * 4].view(np.int32), want)
        kept = host[w.nbytes + keep * 4:].view(np.float32).reshape(heads, keep)
        assert np.array_equal(kept, w[:, layer][:, want])
        assert np.array_equal(host[:w.nbytes].view(np.float32), w.reshape(-1))


def test_weights_of_a_layer(E, rng):
    """The queries stand right behind the weights of all layers."""
    from eakv_amd import hipmem
    n_q, n_kv, d, room = 4, 2, 64, 128
    caches = W.build(E, rng, [100, 60], n_kv, d, room)
    w = rng.random((2, n_kv, LAYERS, room), dtype=np.float32)
    q = rng.standard_normal((2, n_q, d)).astype(np.float32)
    buf = hipmem.DeviceArray.from_host(np.concatenate([w.reshape(-1), q.reshape(-1)]))
    plan = E.WeightsPlan(caches, [1, 1], n_q, n_kv, starts=[99, 59])
    for layer in range(LAYERS):
        plan.run(0, buf.ptr + w.nbytes, buf.ptr + layer * room * 4, LAYERS * room, 0.5)
    caches[0].sync()
    host = buf.download()
    got = host[:w.size].reshape(w.shape)
    assert np.array_equal(host[w.size:], q.reshape(-1))
    for i, n in enumerate((100, 60)):
        want, tol = EV.exact(caches[i], 0, q[i:i + 1], n - 1, n_q, n_kv)
        for layer in range(LAYERS):
            y = want + 0.5 * w[i, :, layer, :n].astype(np.float64)
            assert (np.abs(got[i, :, layer, :n] - y) <= tol + 3 * W.E32 * np.abs(y)).all()
            assert np.array_equal(got[i, :, layer, n:], w[i, :, layer, n:])
