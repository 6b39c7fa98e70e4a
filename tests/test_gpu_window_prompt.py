"""Windows of so many rows that K and V are expanded into matrix operands first
(eakv_attention_window_batch_device), against the exact attention of the cache's own
planes in 64 bits, of a sample of the heads; bounds in windows.py."""
import numpy as np
import pytest

import windows as W
from test_gpu_window import E  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


class Head:
    """One kv head of a cache, as windows.values reads one."""

    def __init__(self, cache, k):
        self.cache, self.k = cache, k
        self.n_heads, self.max_seq_len, self.head_dim = 1, cache.max_seq_len, cache.head_dim

    def read_planes(self, layer, kv):
        n = self.max_seq_len * self.head_dim // 64
        return tuple(x[self.k * n:(self.k + 1) * n] for x in self.cache.read_planes(layer, kv))


def expanded(call, wins, n_kv):
    """Whether the call's workspace holds f16 operands of every token."""
    tokens = sum((s + m + 31) // 32 * 32 for s, m in wins if m > 64)
    return call.plan.work_bytes >= tokens * n_kv * call.d * 4


def compare(E, rng, d, n_kv, n_q, wins, bf16, layers=1, layer=0, shift=0, scale=None):
    caches = W.build(E, rng, [s + m for s, m in wins], n_kv, d, max(s + m for s, m in wins) + 5, layers,
                     scale)
    ms = [m for _, m in wins]
    call = W.Call(E, caches, ms, n_q, n_kv, bf16, [s for s, _ in wins], None, shift)
    assert expanded(call, wins, n_kv)
    q = call.put(rng.standard_normal((sum(ms), n_q, d), dtype=np.float32))
    print("expanded", d, n_kv, n_q, wins, "bf16" if bf16 else "f32", "work", call.plan.work_bytes, flush=True)
    call.run(layer)
    got = call.get()
    call.run(layer)
    assert np.array_equal(call.get().view(np.uint32), got.view(np.uint32))     # the same bits
    g, row = n_q // n_kv, 0
    for c, (s, m) in zip(caches, wins):
        for k in sorted({0, n_kv - 1}):
            heads = sorted({k * g, k * g + g - 1})
            sub = np.ascontiguousarray(q[row:row + m][:, heads])
            want, tol, half = W.attend(Head(c, k), layer, sub, s, len(heads), 1, wide=True)
            if m:
                print("  rel", W.check(got[row:row + m][:, heads], want, tol, half, bf16), flush=True)
        row += m
    for c in caches:
        c.free()


# (d, kv heads, q heads, [(start, tokens)])
SHAPES = [
    (128, 8, 128, [(16, 80), (0, 97), (200, 65)]),
    (64, 8, 128, [(16, 80), (0, 97), (200, 65), (31, 66)]),
    # contexts in chunks
    (128, 4, 64, [(1500, 512)]),
    (64, 4, 64, [(1500, 512)]),
    # beside windows of few rows, empty ones and one token
    (128, 8, 64, [(31, 300), (700, 1), (33, 0), (90, 290), (5, 40)]),
    # one q head per kv head, rows that end inside a block
    (128, 32, 32, [(0, 1000), (5, 777)]),
    (64, 16, 48, [(0, 700), (64, 701)]),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_causal(E, rng, shape, bf16):
    compare(E, rng, *shape, bf16)


@pytest.mark.parametrize("shape", [(128, 8, 128, [(3000, 70)] * 3), (64, 4, 64, [(6000, 140)] * 3)])
def test_more_chunks(E, rng, shape):
    """(f32 windows of these sizes are not expanded)"""
    compare(E, rng, *shape, True)


@pytest.mark.parametrize("bf16", [False, True])
def test_layer_and_odd_addresses(E, rng, bf16):
    compare(E, rng, 128, 8, 128, [(16, 80), (0, 97), (200, 65)], bf16, layers=3, layer=1, shift=1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("scale", [1e-12, 1e-4, 3e4, 1e12])
def test_magnitudes(E, rng, scale, bf16):
    """V far from f16's range (K stays, so that the softmax is one)."""
    s = np.ones((1, 2, 1, 1, 1), np.float32)
    s[0, 1] = scale
    compare(E, rng, 128, 8, 128, [(40, 66)] * 3, bf16, scale=s)


@pytest.mark.parametrize("bf16", [False, True])
def test_outlier_channels(E, rng, bf16):
    s = np.ones((1, 1, 1, 1, 128), np.float32)
    s[..., [5, 70, 71]] = 30.0
    compare(E, rng, 128, 8, 128, [(90, 66)] * 3, bf16, scale=s)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_nonfinite(E, rng, d, bf16):
    """NaN and infinities in tokens that a row does not see leave it alone; where it
    sees them, K gives a row of NaN and V NaN in its 64 dims."""
    n_kv, n_q, start, m, n = 8, 128, 30, 80, 4
    x = rng.standard_normal((1, 2, n_kv, 128, d), dtype=np.float32)
    q = rng.standard_normal((n * m, n_q, d), dtype=np.float32)
    caches = [E.Cache(1, n_kv, d, 128) for _ in range(n)]
    got = []
    for bad in (False, True):
        if bad:
            x[0, 0, 3, start + 70, 0] = np.nan
            x[0, 1, 3, start + 40, d - 64] = np.inf
            x[0, :, :, start + m:] = np.nan
        for c in caches:
            c.clear()
            c.load_raw(x, 128)
            c.restore(start + m)
        call = W.Call(E, caches, [m] * n, n_q, n_kv, bf16, [start] * n)
        assert expanded(call, [(start, m)] * n, n_kv)
        call.put(q)
        call.run()
        got.append(call.get())
    nan = np.isnan(got[1])
    want = np.zeros((n, m, n_kv, n_q // n_kv, d), bool)
    want[:, 70:, 3] = True
    want[:, 40:, 3, :, d - 64:] = True
    want = want.reshape(nan.shape)
    assert np.array_equal(nan, want)
    assert np.array_equal(got[0][~want].view(np.uint32), got[1][~want].view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
def test_recorded_in_graphs(E, rng, bf16):
    """Two graphs over the same caches with workspaces of their own, replayed in turn
    with eager calls between; each replay against the eager result's bits."""
    from eakv_amd.hipmem import DeviceArray
    caches = W.build(E, rng, [2012], 4, 128, 2020)
    calls = [W.Call(E, caches, [m], 64, 4, bf16, [2012 - m]) for m in (512, 500)]
    works = [DeviceArray((c.plan.work_bytes,), np.uint8) for c in calls]
    graphs = [W.Graph(lambda s, c=c, w=w: c.run(stream=s, work=w.ptr, work_bytes=w.nbytes,
                                                clear=False)) for c, w in zip(calls, works)]
    for k in range(3):
        for c, g in zip(calls, graphs):
            assert expanded(c, [(1500, 512)], 4)
            c.put(rng.standard_normal((c.total, 64, 128), dtype=np.float32))
            c.run()
            want = c.get()
            c.do.upload(np.full(c.do.nbytes, c.GUARD, np.uint8))
            g.launch()
            assert np.array_equal(c.get(sync=False).view(np.uint32), want.view(np.uint32)), k
    for g in graphs:
        g.free()
