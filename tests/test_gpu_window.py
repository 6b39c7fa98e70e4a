"""Attention of several new tokens of each sequence over the packed cache
(eakv_attention_window_batch_device) against the exact attention of the cache's own
planes in 64 bits; bounds in windows.py."""
import numpy as np
import pytest

import windows as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


def say(*a):
    print(*a, flush=True)


def tree_words(rng, m, masks=False):
    """Ancestors and self of a random tree, or (masks) any bits, some rows empty."""
    words = []
    for i in range(m):
        if masks:
            words.append(int(rng.integers(0, 1 << min(m, 62))) if rng.random() < 0.8 else 0)
        else:
            up = int(rng.integers(-1, i)) if i else -1
            words.append((words[up] if up >= 0 else 0) | 1 << i)
    return words


def compare(E, rng, d, n_kv, n_q, wins, bf16, tree=None, layers=1, layer=0, shift=0, room=None,
            starts_given=True, scale=None):
    lens = [s + m for s, m in wins]
    room = room or max(lens) + 5
    caches = W.build(E, rng, lens, n_kv, d, room, layers, scale)
    ms = [m for _, m in wins]
    words = None
    if tree:
        words = [w for m in ms for w in tree_words(rng, m, tree == "masks")]
    if not starts_given:
        for c, (s, _) in zip(caches, wins):
            c.restore(s)                    # appended, not advanced
    call = W.Call(E, caches, ms, n_q, n_kv, bf16, [s for s, _ in wins] if starts_given else None,
                  words, shift)
    q = call.put(rng.standard_normal((sum(ms), n_q, d), dtype=np.float32))
    say("window", d, n_kv, n_q, wins[:4], len(wins), "bf16" if bf16 else "f32", tree,
        "work", call.plan.work_bytes)
    call.run(layer)
    got = call.get()
    call.run(layer)
    assert np.array_equal(call.get().view(np.uint32), got.view(np.uint32))     # the same bits
    row = 0
    for c, (s, m) in zip(caches, wins):
        want, tol, half = W.attend(c, layer, q[row:row + m], s, n_q, n_kv,
                                   None if words is None else words[row:row + m])
        if m:
            rel = W.check(got[row:row + m], want, tol, half, bf16)
            say("  rel", rel)
        row += m
    for c in caches:
        c.free()


# (d, kv heads, q heads, [(start, tokens)]): rows (tokens x q heads per kv head) on
# both sides of 32, 64, 128 and 256, contexts around tiles of 32 to 256 tokens
SHAPES = [
    (128, 2, 8, [(0, 1)]),
    (128, 1, 1, [(0, 2)]),
    (128, 2, 8, [(31, 2)]),
    (64, 4, 32, [(100, 4), (0, 3), (255, 1)]),
    (128, 8, 32, [(500, 8)]),
    (128, 2, 8, [(63, 9)]),
    (128, 2, 10, [(777, 7), (5, 0), (0, 7)]),
    (64, 3, 3, [(1000, 33)]),
    (128, 2, 8, [(300, 17)]),
    (128, 2, 2, [(129, 65), (2, 64)]),
    (64, 1, 16, [(60, 9)]),
    (128, 1, 8, [(250, 33)]),
    (64, 2, 8, [(0, 257)]),
    (128, 1, 3, [(40, 171)]),
    (128, 2, 2, [(0, 300), (700, 1), (33, 0), (90, 200)]),
    (64, 2, 40, [(511, 5)]),
    # many blocks of rows
    (128, 2, 8, [(33, 65)]),
    (128, 1, 16, [(100, 140)]),
    (64, 1, 32, [(0, 70), (500, 3), (95, 97)]),
    (128, 1, 32, [(1, 65)]),
    (64, 1, 16, [(1500, 130)]),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_causal(E, rng, shape, bf16):
    compare(E, rng, *shape, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["tree", "masks"])
@pytest.mark.parametrize("d,n_kv,n_q,wins", [
    (128, 2, 8, [(0, 1), (0, 5), (7, 24)]),
    (64, 2, 2, [(0, 64), (321, 64), (40, 1)]),
    (128, 1, 8, [(200, 64), (0, 33)]),
])
def test_tree(E, rng, d, n_kv, n_q, wins, kind, bf16):
    compare(E, rng, d, n_kv, n_q, wins, bf16, tree=kind)


@pytest.mark.parametrize("bf16", [False, True])
def test_chunks_and_ragged_batch(E, rng, bf16):
    """Long contexts in chunks beside short ones in one, and 32 sequences."""
    compare(E, rng, 128, 1, 4, [(9000, 6), (0, 1), (100, 8), (4001, 3)], bf16)
    compare(E, rng, 64, 2, 4, [(int(97 * 1.13 ** i), 1 + i % 5) for i in range(32)], bf16)
    compare(E, rng, 128, 1, 2, [(2500, 150)], bf16)
    compare(E, rng, 64, 1, 24, [(6000, 100), (6100, 0), (3, 88)], bf16)


def test_long_context(E, rng):
    """70,000 tokens, hundreds of chunks of a unit joined."""
    compare(E, rng, 128, 1, 4, [(70000, 3)], False)


@pytest.mark.parametrize("bf16", [False, True])
def test_layer_pending_tokens_and_odd_addresses(E, rng, bf16):
    """Layer 2 of 3, windows at seq_len of tokens appended but not advanced, buffers
    one element off 16-byte alignment."""
    compare(E, rng, 128, 2, 8, [(64, 6), (200, 2)], bf16, layers=3, layer=2, starts_given=False)
    compare(E, rng, 64, 2, 4, [(90, 21)], bf16, shift=1)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 3e4, 1e12])
def test_magnitudes(E, rng, scale):
    """V far from f16's range (K stays, so that the softmax is one)."""
    s = np.ones((1, 2, 1, 1, 1), np.float32)
    s[0, 1] = scale
    for bf16 in (False, True):
        compare(E, rng, 128, 2, 4, [(100, 9)], bf16, scale=s)
        compare(E, rng, 128, 1, 32, [(40, 66)], bf16, scale=s)


def test_outlier_channels(E, rng):
    """Groups with an outlier: scale and bias far above the other values."""
    s = np.ones((1, 1, 1, 1, 128), np.float32)
    s[..., [5, 70, 71]] = 30.0
    for bf16 in (False, True):
        compare(E, rng, 128, 2, 8, [(333, 8)], bf16, scale=s)
        compare(E, rng, 128, 1, 32, [(90, 66)], bf16, scale=s)


def test_beyond_32_bit_offsets(E, rng):
    """A layer whose planes pass 4 GiB: the last head's bytes lie beyond 2^32."""
    n_kv, d, room = 8, 128, 9_700_000
    c = E.Cache(1, n_kv, d, room)
    x = rng.standard_normal((1, 2, n_kv, 100, d), dtype=np.float32)
    c.load_raw(x, 100)
    small = E.Cache(1, n_kv, d, 128)
    small.load_raw(x, 100)
    q = rng.standard_normal((6, 16, d), dtype=np.float32)
    outs = []
    for cc in (c, small):
        call = W.Call(E, [cc], [6], 16, n_kv, False, [94])
        call.put(q)
        call.run()
        outs.append(call.get())
    assert np.array_equal(outs[0].view(np.uint32), outs[1].view(np.uint32))
    c.free()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_nonfinite_many_rows(E, rng, d, bf16):
    """As below for windows of many rows."""
    n_kv, n_q, start, m = 1, 8 if bf16 else 32, 30, 80
    c = E.Cache(1, n_kv, d, 128)
    x = rng.standard_normal((1, 2, n_kv, 128, d), dtype=np.float32)
    q = rng.standard_normal((m, n_q, d), dtype=np.float32)
    got = []
    for bad in (False, True):
        if bad:
            x[0, 0, 0, start + 70, 0] = np.nan
            x[0, 1, 0, start + 40, d - 64] = np.nan
            x[0, :, :, start + m:] = np.nan
        c.clear()
        c.load_raw(x, 128)
        c.restore(start + m)
        call = W.Call(E, [c], [m], n_q, n_kv, bf16, [start])
        call.put(q)
        call.run()
        got.append(call.get())
    nan = np.isnan(got[1])
    want = np.zeros_like(nan)
    want[70:] = True
    want[40:, :, d - 64:] = True
    assert np.array_equal(nan, want)
    assert np.array_equal(got[0][~want].view(np.uint32), got[1][~want].view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_nonfinite(E, rng, d, bf16):
    """NaN and infinities in tokens that a row does not see (later drafts, other
    branches, the room behind) leave it alone; where it sees them, K gives a row of
    NaN and V NaN in its 64 dims."""
    n_kv, n_q, start, m = 2, 8, 70, 12
    c = E.Cache(1, n_kv, d, 128)
    x = rng.standard_normal((1, 2, n_kv, 128, d), dtype=np.float32)
    c.load_raw(x, 128)
    c.restore(start + m)
    words = [1 << i for i in range(m)]
    words[5] |= 1 << 3
    words[7] |= 1 << 2
    q = rng.standard_normal((m, n_q, d), dtype=np.float32)

    def run(tree):
        call = W.Call(E, [c], [m], n_q, n_kv, bf16, [start], words if tree else None)
        call.put(q)
        call.run()
        return call.get()

    clean = {t: run(t) for t in (False, True)}
    y = x.copy()
    y[0, 0, 0, start + 3, 0] = np.nan            # K of kv head 0, token 3 (a group's first value)
    y[0, 1, 1, start + 2, d - 1] = np.inf        # V of kv head 1, token 2, last group
    y[0, :, :, start + m:] = np.nan              # behind the last token
    c.clear()
    c.load_raw(y, 128)
    c.restore(start + m)
    for t in (False, True):
        got = run(t)
        for i in range(m):
            see = [j for j in range(m) if (words[i] >> j & 1 if t else j <= i)]
            for h in range(n_q):
                bad = np.zeros(d, bool)
                if h < 4 and 3 in see:
                    bad[:] = True
                if h >= 4 and 2 in see:
                    bad[d - 64:] = True
                assert np.array_equal(np.isnan(got[i, h]), bad), (t, i, h)
                assert np.array_equal(got[i, h][~bad].view(np.uint32),
                                      clean[t][i, h][~bad].view(np.uint32)), (t, i, h)
    # non-finite queries: their own rows alone
    q2 = q.copy()
    q2[4, 3, 0] = np.nan
    q2[6, 1, 5] = np.inf
    c.clear()
    c.load_raw(x, 128)
    call = W.Call(E, [c], [m], n_q, n_kv, False, [start])
    call.put(q2)
    call.run()
    got = call.get()
    assert np.isnan(got[4, 3]).all() and np.isnan(got[6, 1]).all()
    assert np.isfinite(np.delete(got.reshape(-1, d), [4 * n_q + 3, 6 * n_q + 1], 0)).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_one_cache_in_several_windows(E, rng, bf16):
    """The same cache named three times, its windows overlapping."""
    c = W.build(E, rng, [400], 2, 128, 410)[0]
    starts, ms = [390, 100, 385], [10, 40, 12]
    call = W.Call(E, [c, c, c], ms, 8, 2, bf16, starts)
    q = call.put(rng.standard_normal((sum(ms), 8, 128), dtype=np.float32))
    call.run()
    got = call.get()
    row = 0
    for s, m in zip(starts, ms):
        want, tol, half = W.attend(c, 0, q[row:row + m], s, 8, 2)
        W.check(got[row:row + m], want, tol, half, bf16)
        row += m


@pytest.mark.parametrize("tree", [None, "tree", "masks"])
@pytest.mark.parametrize("bf16", [False, True])
def test_large_groups(E, rng, bf16, tree):
    """Hundreds of q heads to one kv head: many blocks of rows for a few tokens."""
    compare(E, rng, 64, 1, 300, [(33, 2), (0, 1)], bf16, tree)
    compare(E, rng, 128, 1, 40, [(290, 64)], bf16, tree)


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_without_tokens(E, rng, bf16):
    c = W.build(E, rng, [40], 2, 64, 48)[0]
    call = W.Call(E, [c], [3], 4, 2, bf16, [0], [0, 2, 0])
    call.put(rng.standard_normal((3, 4, 64), dtype=np.float32))
    call.run()
    got = call.get()
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[1] != 0).any()
    # an empty call and one with empty windows only
    call = W.Call(E, [c], [0], 4, 2, bf16, [0])
    call.run()
    call.get()


def test_one_token_is_the_decode_launch(E, rng):
    from eakv_amd.hipmem import DeviceArray
    caches = W.build(E, rng, [700, 33, 5000], 4, 128, 5001)
    q = rng.standard_normal((3, 16, 128), dtype=np.float32)
    call = W.Call(E, caches, [1, 1, 1], 16, 4, False, [699, 32, 4999])
    call.put(q)
    dq, do = DeviceArray.from_host(q), DeviceArray((3, 16, 128))
    assert E.lib().eakv_attention_fused_batch_device(E.handles(caches), 3, 0, dq.ptr, 16, 4, do.ptr,
                                                     None) == 0
    caches[0].sync()
    want = do.download()
    call.run()
    assert np.array_equal(call.get().view(np.uint32), want.view(np.uint32))
    # with a workspace of its own: the same bits
    n = call.plan.work_bytes
    w = DeviceArray((n + 16,), np.uint8)
    call.run(work=w.ptr, work_bytes=n)
    assert np.array_equal(call.get().view(np.uint32), want.view(np.uint32))


def test_streams_and_workspaces(E, rng):
    """A batched append on the shared stream, then calls over the appended tokens on two
    callers' streams with workspaces of their own, and one with the cache's."""
    from eakv_amd.hipmem import DeviceArray, Stream
    caches = W.build(E, rng, [6000, 6000], 2, 128, 6100)
    x = rng.standard_normal((2, 1, 2, 2, 8, 128), dtype=np.float32)
    dx = DeviceArray.from_host(x)
    calls = [W.Call(E, caches, [8, 8], 8, 2, bf16, None) for bf16 in (False, True, False)]
    qs = [c.put(rng.standard_normal((16, 8, 128), dtype=np.float32)) for c in calls]
    sizes = [c.plan.work_bytes for c in calls]
    works = [DeviceArray((max(n, 16),), np.uint8) for n in sizes[:2]] + [None]
    streams = [Stream(), Stream(), None]
    for c in calls:
        c.do.upload(np.full(c.do.nbytes, c.GUARD, np.uint8))
    assert sizes[0] > 0
    assert E.lib().eakv_append_batch_device(E.handles(caches), 2, dx.ptr, 8, None) == 0
    for c, s, w, n in zip(calls, streams, works, sizes):
        c.run(stream=s and s.s, work=w and w.ptr, work_bytes=n if w else 0, clear=False)
    for s in streams[:2]:
        s.synchronize()
    caches[0].sync()
    for c, q, bf16 in zip(calls, qs, (False, True, False)):
        got = c.get()
        for i, cache in enumerate(caches):
            want, tol, half = W.attend(cache, 0, q[8 * i:8 * i + 8], 6000, 8, 2)
            W.check(got[8 * i:8 * i + 8], want, tol, half, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_recorded_in_graphs(E, rng, bf16):
    """Two graphs over the same caches with workspaces of their own, replayed in turn
    with eager calls between; each replay against the eager result's bits."""
    from eakv_amd.hipmem import DeviceArray
    caches = W.build(E, rng, [3000, 500], 2, 128, 3010)
    calls = [W.Call(E, caches, [m, m], 8, 2, bf16, [3000 - m, 500 - m]) for m in (5, 9)]
    works = [DeviceArray((max(c.plan.work_bytes, 16),), np.uint8) for c in calls]
    graphs = [W.Graph(lambda s, c=c, w=w: c.run(stream=s, work=w.ptr, work_bytes=w.nbytes,
                                                clear=False)) for c, w in zip(calls, works)]
    for k in range(3):
        for c, g in zip(calls, graphs):
            c.put(rng.standard_normal((c.total, 8, 128), dtype=np.float32))
            c.run()
            want = c.get()
            c.do.upload(np.full(c.do.nbytes, c.GUARD, np.uint8))
            g.launch()
            assert np.array_equal(c.get(sync=False).view(np.uint32), want.view(np.uint32)), k
    # without a workspace of its own a captured call that needs one is refused
    with pytest.raises(E.EakvError) as e:
        W.Graph(lambda s: calls[0].run(stream=s, clear=False))
    assert e.value.code == E.EAKV_ERR_INVALID
    for g in graphs:
        g.free()


def test_refusals(E, rng):
    from eakv_amd.hipmem import DeviceArray
    a, b = W.build(E, rng, [100, 100], 2, 128, 120)
    other = E.Cache(1, 2, 128, 121)
    odd = E.Cache(1, 2, 96, 120)
    buf = DeviceArray((1 << 16,))
    L = E.lib()

    def call(caches=(a,), layer=0, starts=(96,), n=(4,), q=None, dtype=0, n_q=8, n_kv=2, tree=None,
             out=None, work=None, work_bytes=0):
        hs = E.handles(caches)
        return L.eakv_attention_window_batch_device(
            hs, len(caches), layer, E.ints(starts) if starts else None, E.ints(n) if n else None,
            buf.ptr if q is None else q, dtype, n_q, n_kv, tree,
            buf.ptr + 4096 if out is None else out, work, work_bytes, None)

    assert call() == 0
    a.sync()
    for kw in (dict(layer=1), dict(layer=-1), dict(starts=(-1,)), dict(starts=(101,)),
               dict(starts=(100,), n=(21,)), dict(n=(-1,)), dict(n=None), dict(dtype=2),
               dict(n_q=7), dict(n_kv=3), dict(n_q=0), dict(q=buf.ptr + 2), dict(out=buf.ptr + 1),
               dict(q=0), dict(out=0), dict(tree=buf.ptr + 4), dict(tree=buf.ptr, starts=(0,), n=(65,)),
               dict(caches=(a, other), starts=(0, 0), n=(1, 1)), dict(caches=(odd,), starts=(0,), n=(1,)),
               dict(work=buf.ptr + 8, work_bytes=1 << 12), dict(caches=(a,) * 33, starts=(0,) * 33,
                                                               n=(1,) * 33)):
        L.eakv_clear_error()
        assert call(**kw) == E.EAKV_ERR_INVALID, kw
        assert L.eakv_last_error() == E.EAKV_ERR_INVALID
    # a workspace that is too small
    big = W.build(E, rng, [9000], 1, 128, 9000)[0]
    p = E.WindowPlan([big], [4], 4, 1, starts=[8996])
    assert p.work_bytes > 16
    with pytest.raises(E.EakvError):
        p.run(0, buf.ptr, buf.ptr + 8192, None, buf.ptr, 16)
    # the same cache twice in a batch, at two positions: allowed, it is only read
    call2 = W.Call(E, [a, a], [3, 2], 8, 2, False, [97, 10])
    q = call2.put(rng.standard_normal((5, 8, 128), dtype=np.float32))
    call2.run()
    got = call2.get()
    for r, s, m in ((0, 97, 3), (3, 10, 2)):
        want, tol, half = W.attend(a, 0, q[r:r + m], s, 8, 2)
        W.check(got[r:r + m], want, tol, half, False)
