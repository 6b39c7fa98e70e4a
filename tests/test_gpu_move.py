"""Tokens moved between and within caches (copy, gather, fork, compact): planes bit for
bit, everything else as it was; and the loop of serving with drafts."""
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


def planes(c):
    """Every block's planes as [layers][2][n_kv][room][bytes of a token]."""
    out = []
    for layer in range(c.n_layers):
        for kv in (0, 1):
            w, s, b = c.read_planes(layer, kv)
            sh = (c.n_heads, c.max_seq_len, -1)
            out.append(np.concatenate([x.view(np.uint8).reshape(sh) for x in (w, s, b)], 2))
    return np.stack(out).reshape((c.n_layers, 2) + out[0].shape)


def filled(E, rng, layers, n_kv, d, room, n=None):
    c = E.Cache(layers, n_kv, d, room)
    n = room if n is None else n
    if n:
        c.load_raw(rng.standard_normal((layers, 2, n_kv, n, d), dtype=np.float32), n)
    return c


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,src_pos,dst_pos,room_s,room_d,n_dst", [
    (1, 0, 0, 5, 7, 1), (3, 2, 1, 9, 64, 2), (511, 0, 0, 600, 511, 3), (513, 7, 5, 1500, 700, 1),
    (1025, 3, 0, 1100, 1031, 32), (2600, 0, 100, 2600, 3001, 2)])
def test_copy(E, rng, d, n, src_pos, dst_pos, room_s, room_d, n_dst):
    from eakv_amd.hipmem import Stream
    print("copy", d, n, src_pos, dst_pos, n_dst, flush=True)
    src = filled(E, rng, 2, 3, d, room_s)
    dsts = [filled(E, rng, 2, 3, d, room_d) for _ in range(n_dst)]
    before = [planes(c) for c in dsts]
    from_ = planes(src)
    st = Stream()
    for stream in (None, st.s):
        assert E.lib().eakv_cache_copy_batch_device(src.h, src_pos, E.handles(dsts), n_dst, dst_pos, n,
                                                    stream) == 0, E.last_error()
        st.synchronize()
        for c, b in zip(dsts, before):
            want = b.copy()
            want[:, :, :, dst_pos:dst_pos + n] = from_[:, :, :, src_pos:src_pos + n]
            assert np.array_equal(planes(c), want)
            assert c.seq_len == room_d
    assert np.array_equal(planes(src), from_)


def test_copy_within_a_cache(E, rng):
    c = filled(E, rng, 1, 2, 128, 400)
    a = planes(c)
    assert E.lib().eakv_cache_copy_batch_device(c.h, 300, E.handles([c]), 1, 200, 100, None) == 0
    c.sync()
    a[:, :, :, 200:300] = a[:, :, :, 300:400]
    assert np.array_equal(planes(c), a)
    for s, d, n in ((300, 201, 100), (100, 100, 1), (0, 399, 2)):
        assert E.lib().eakv_cache_copy_batch_device(c.h, s, E.handles([c]), 1, d, n,
                                                    None) == E.EAKV_ERR_INVALID


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 511, 512, 513, 1024, 1025, 2500])
def test_gather_to_another_cache(E, rng, d, n):
    """Any list: in no order, positions twice, and (clamped) outside the room."""
    from eakv_amd.hipmem import DeviceArray
    srcs = [filled(E, rng, 2, 2, d, 1600) for _ in range(2)]
    dsts = [filled(E, rng, 2, 2, d, 2600) for _ in range(2)]
    index = rng.integers(0, 1600, (2, n)).astype(np.int32)
    index[0, 0], index[1, -1] = -5, 1 << 30
    di = DeviceArray.from_host(index)
    before = [planes(c) for c in dsts]
    assert E.lib().eakv_cache_gather_batch_device(E.handles(srcs), E.handles(dsts), 2, E.ints([3, 0]),
                                                  di.ptr, E.ints([n, n]), None) == 0, E.last_error()
    srcs[0].sync()
    for s, c, b, i, at in zip(srcs, dsts, before, index, (3, 0)):
        b[:, :, :, at:at + n] = planes(s)[:, :, :, np.clip(i, 0, 1599)]
        assert np.array_equal(planes(c), b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at,n,room", [(0, 1, 4), (0, 4, 4), (90, 7, 114), (0, 700, 1500),
                                       (4, 2500, 4000), (100, 3500, 3700)])
def test_gather_in_place(E, rng, d, at, n, room):
    from eakv_amd.hipmem import DeviceArray
    print("gather in place", d, at, n, room, flush=True)
    caches = [filled(E, rng, 1, 2, d, room) for _ in range(3)]
    lists = [np.sort(rng.choice(np.arange(at, room), n, replace=False)).astype(np.int32)
             for _ in caches]
    lists[2] = lists[2][:n // 2]
    di = DeviceArray.from_host(np.concatenate(lists))
    want = [planes(c) for c in caches]
    for w, i in zip(want, lists):
        w[:, :, :, at:at + i.size] = w[:, :, :, i]
    hs = E.handles(caches)
    assert E.lib().eakv_cache_gather_batch_device(hs, hs, 3, E.ints([at] * 3), di.ptr,
                                                  E.ints([i.size for i in lists]), None) == 0
    caches[0].sync()
    for c, w in zip(caches, want):
        assert np.array_equal(planes(c), w)


def test_fork_and_compact(E, rng):
    src = filled(E, rng, 2, 2, 64, 300, 250)
    p = planes(src)
    for n, room in ((250, 300), (0, 1), (17, 17), (249, 1000)):
        f = src.fork(n, room)
        assert (f.seq_len, f.max_seq_len, f.n_layers, f.head_dim) == (n, room, 2, 64)
        q = planes(f)
        assert np.array_equal(q[:, :, :, :n], p[:, :, :, :n]) and not q[:, :, :, n:].any()
        f.free()
    keep = np.sort(rng.choice(np.arange(10, 250), 100, replace=False))
    src.compact(keep, 10)
    assert src.seq_len == 110
    q = planes(src)
    assert np.array_equal(q[:, :, :, 10:110], p[:, :, :, keep])
    assert np.array_equal(q[:, :, :, :10], p[:, :, :, :10])
    src.compact(np.arange(20, 60), 20)               # all in place already
    assert src.seq_len == 60 and np.array_equal(planes(src), q)
    src.compact([], 30)
    assert src.seq_len == 30
    for keep, start in (([5, 5], 0), ([7, 6], 0), ([30], 0), ([-1], 0), ([3], 4), ([0], 31), ([0], -1)):
        with pytest.raises(E.EakvError):
            src.compact(keep, start)
        assert src.seq_len == 30
    for n, room in ((31, 40), (-1, 40), (10, 9), (0, 0)):
        with pytest.raises(E.EakvError):
            src.fork(n, room)


def test_refusals(E, rng):
    from eakv_amd.hipmem import DeviceArray
    L = E.lib()
    a, b, c = (filled(E, rng, 1, 2, 128, 50, 20) for _ in range(3))
    wide, layers, odd = E.Cache(1, 2, 64, 50), E.Cache(2, 2, 128, 50), E.Cache(1, 2, 96, 50)
    roomy = E.Cache(1, 2, 128, 60)
    di = DeviceArray.from_host(np.arange(64, dtype=np.int32))

    def copy(dsts, s=0, d=0, n=5, src=a):
        return L.eakv_cache_copy_batch_device(src.h, s, E.handles(dsts), len(dsts), d, n, None)

    for kw in (dict(dsts=[wide]), dict(dsts=[layers]), dict(dsts=[b, b]), dict(dsts=[b, roomy]),
               dict(dsts=[b], s=-1), dict(dsts=[b], s=46), dict(dsts=[b], d=21), dict(dsts=[b], d=-1),
               dict(dsts=[b], d=20, n=31), dict(dsts=[b], n=-1), dict(dsts=[odd], src=odd)):
        assert copy(**kw) == E.EAKV_ERR_INVALID, kw
    assert copy([b], n=0) == 0 and copy([b], s=45) == 0

    def gather(srcs, dsts, at=(0,), n=(5,), index=di.ptr):
        return L.eakv_cache_gather_batch_device(E.handles(srcs), E.handles(dsts), len(dsts), E.ints(at),
                                                index, E.ints(n), None)

    two = dict(at=(0, 0), n=(1, 1))
    for srcs, dsts, kw in (([a], [wide], {}), ([a, a], [b, b], two), ([a, b], [b, c], two),
                           ([a, c], [a, a], two), ([a], [b], dict(at=(21,))), ([a], [b], dict(at=(-1,))),
                           ([a], [b], dict(n=(-1,))), ([a], [b], dict(at=(20,), n=(31,))),
                           ([a], [b], dict(index=0)), ([a], [b], dict(index=di.ptr + 2)),
                           ([odd], [odd], {}), ([a, roomy], [b, c], two)):
        assert gather(srcs, dsts, **kw) == E.EAKV_ERR_INVALID, (kw,)
    assert gather([a], [b], n=(0,), index=0) == 0
    assert gather([a, a], [b, c], **two) == 0            # one source twice
    a.sync()
    # not recorded in graphs
    for f in (lambda s: E._check(L.eakv_cache_copy_batch_device(a.h, 0, E.handles([b]), 1, 0, 5, s)),
              lambda s: E._check(L.eakv_cache_gather_batch_device(E.handles([a]), E.handles([b]), 1,
                                                                  E.ints([0]), di.ptr, E.ints([5]), s))):
        with pytest.raises(E.EakvError) as e:
            W.Graph(f)
        assert e.value.code == E.EAKV_ERR_INVALID


def test_shared_stream_that_records_a_graph(E, rng):
    """Copies, gathers and windows without scratch of their own are refused on the
    caches' shared stream too while it records."""
    import ctypes as C
    from eakv_amd import hipmem
    from eakv_amd.hipmem import DeviceArray
    a, b = W.build(E, rng, [3000, 100], 2, 128, 3010)
    buf = DeviceArray((1 << 16,))
    index = DeviceArray.from_host(np.arange(4, dtype=np.int32))
    L, h = E.lib(), hipmem.hip()
    shared = L.eakv_cache_stream(a.h)
    a.sync()
    hipmem.check(h.hipStreamBeginCapture(C.c_void_p(shared), 2), "begin")
    try:
        copy = L.eakv_cache_copy_batch_device(a.h, 0, E.handles([b]), 1, 0, 4, None)
        gather = L.eakv_cache_gather_batch_device(E.handles([a]), E.handles([b]), 1, E.ints([0]),
                                                  index.ptr, E.ints([4]), None)
        window = L.eakv_attention_window_batch_device(E.handles([a]), 1, 0, None, E.ints([4]), buf.ptr,
                                                      0, 8, 2, None, buf.ptr, None, 0, None)
    finally:
        graph = C.c_void_p()
        rc = h.hipStreamEndCapture(C.c_void_p(shared), C.byref(graph))
    hipmem.check(rc, "end")
    h.hipGraphDestroy(graph)
    assert (copy, gather, window) == (E.EAKV_ERR_INVALID,) * 3
    # and work again afterwards
    assert L.eakv_cache_copy_batch_device(a.h, 0, E.handles([b]), 1, 0, 4, None) == 0
    a.sync()
    for x, y in zip(a.read_planes(0, 0), b.read_planes(0, 0)):
        n, m = 3010 * 2, 3010 * 2
        assert np.array_equal(x[:8], y[:8]) and np.array_equal(x[n:n + 8], y[m:m + 8])


def test_orders_with_other_streams(E, rng):
    """A copy on a caller's stream right behind an append on the shared stream, then an
    append to the source on the shared stream and a host call on the copy."""
    from eakv_amd.hipmem import DeviceArray, Stream
    n_kv, d, n = 4, 128, 5000
    src = filled(E, rng, 1, n_kv, d, 2 * n, 1)
    dst = E.Cache(1, n_kv, d, 2 * n)
    x = rng.standard_normal((2, 1, 2, n_kv, n, d), dtype=np.float32)
    dx = DeviceArray.from_host(x)
    st = Stream()
    one = x[0].nbytes
    assert E.lib().eakv_append_batch_device(E.handles([src]), 1, dx.ptr, n, None) == 0
    assert E.lib().eakv_cache_copy_batch_device(src.h, 0, E.handles([dst]), 1, 0, n + 1, st.s) == 0
    # overwrites the tokens that the copy reads
    assert E.lib().eakv_append_batch_device(E.handles([src]), 1, dx.ptr + one, n, None) == 0
    got = planes(dst)
    ref = E.Cache(1, n_kv, d, 2 * n)
    ref.advance(1)
    for kv in (0, 1):
        ref.append(x[0, 0, kv], 0, kv, n)
    assert np.array_equal(got[:, :, :, 1:n + 1], planes(ref)[:, :, :, 1:n + 1])


@pytest.mark.parametrize("bf16", [False, True])
def test_drafts_loop(E, rng, bf16):
    """Serving with drafts, two steps for two sequences forked from one prompt: append
    the drafts layer by layer, attend, verify against a target computed from the
    attention's outputs, keep what was accepted.  At the end the caches hold what
    appending the kept tokens one after the other gives, and a tree's kept path attends
    as a chain does."""
    from eakv_amd.hipmem import DeviceArray, Stream
    layers, n_kv, n_q, d, room, k, vocab = 2, 2, 8, 64, 400, 6, 50
    prompt = filled(E, rng, layers, n_kv, d, room, 130)
    seqs = [prompt.fork(), E.Cache(layers, n_kv, d, room)]
    assert E.lib().eakv_cache_copy_batch_device(prompt.h, 0, E.handles(seqs[1:]), 1, 0, 130, None) == 0
    seqs[1].advance(130)
    plain = [prompt.fork() for _ in seqs]
    emb = rng.standard_normal((vocab, layers, 2, n_kv, d), dtype=np.float32)
    head = rng.standard_normal((n_q * d, vocab)) * 0.3
    hs = E.handles(seqs)
    kept_tokens = [[], []]
    for step in range(2):
        drafts = rng.integers(0, vocab, (2, k)).astype(np.int32)
        q = rng.standard_normal((2 * (k + 1), n_q, d), dtype=np.float32)
        # the window: the last kept token's successor is not known, so its first token is the
        # step's own start token; then the drafts
        first = rng.integers(0, vocab, 2)
        toks = np.concatenate([first[:, None], drafts], 1)
        x = emb[toks].transpose(0, 2, 3, 4, 1, 5).copy()        # [seq][layer][2][n_kv][k+1][d]
        dx = DeviceArray.from_host(x)
        assert E.lib().eakv_append_batch_device(hs, 2, dx.ptr, k + 1, None) == 0
        call = W.Call(E, seqs, [k + 1, k + 1], n_q, n_kv, bf16)
        qq = call.put(q)
        out = None
        for layer in range(layers):
            call.run(layer)
            out = call.get()
            for s, c in enumerate(seqs):
                rows = slice(s * (k + 1), (s + 1) * (k + 1))
                want, tol, half = W.attend(c, layer, qq[rows], c.seq_len, n_q, n_kv)
                W.check(out[rows], want, tol, half, bf16)
        logits = out.reshape(2, k + 1, -1).astype(np.float64) @ head
        target = np.exp(logits - logits.max(-1, keepdims=True))
        target = (target / target.sum(-1, keepdims=True)).astype(np.float32)
        target[0, 0] = 0.0                                        # the first draft certainly kept
        target[0, 0, drafts[0, 0]] = 1.0
        u = rng.random((2, k + 1), dtype=np.float32)
        bufs = [DeviceArray.from_host(a) for a in (drafts, target, u)]
        kept, nxt = DeviceArray((2,), np.int32), DeviceArray((2,), np.int32)
        n = E.lib().eakv_verify_drafts_work_bytes(2, k, vocab)
        work = DeviceArray((n,), np.uint8)
        st = Stream()
        E._check(E.lib().eakv_verify_drafts_device(2, k, vocab, None, bufs[0].ptr, None, 0, bufs[1].ptr,
                                                   vocab, bufs[2].ptr, kept.ptr, nxt.ptr, work.ptr, n,
                                                   st.s))
        st.synchronize()
        a = kept.download()
        assert a[0] >= 1 and (0 <= nxt.download()).all()
        for s, c in enumerate(seqs):
            c.advance(1 + int(a[s]))                              # a chain's prefix stays
            kept_tokens[s] += toks[s, :1 + a[s]].tolist()
    for s, c in enumerate(plain):
        for t in kept_tokens[s]:
            for layer in range(layers):
                for kv in (0, 1):
                    c.append(emb[t, layer, kv][:, None], layer, kv, 1)
            c.advance(1)
        n = c.seq_len
        assert n == seqs[s].seq_len
        assert np.array_equal(planes(c)[:, :, :, :n], planes(seqs[s])[:, :, :, :n])
    # a tree on sequence 0: nodes 0-1-4-6 are a path; keep it, attend with a chain's mask
    parent = [-1, 0, 0, 1, 1, 2, 4, 4]
    words = []
    for i, up in enumerate(parent):
        words.append((words[up] if up >= 0 else 0) | 1 << i)
    path = [0, 1, 4, 6]
    toks = rng.integers(0, vocab, 8)
    c, base = seqs[0], seqs[0].seq_len
    dx = DeviceArray.from_host(emb[toks].transpose(1, 2, 3, 0, 4).copy())
    assert E.lib().eakv_append_batch_device(E.handles([c]), 1, dx.ptr, 8, None) == 0
    q = rng.standard_normal((8, n_q, d), dtype=np.float32)
    call = W.Call(E, [c], [8], n_q, n_kv, bf16, None, words)
    call.put(q)
    call.run(1)
    tree = call.get()
    di = DeviceArray.from_host(np.array([base + i for i in path], np.int32))
    h1 = E.handles([c])
    assert E.lib().eakv_cache_gather_batch_device(h1, h1, 1, E.ints([base]), di.ptr, E.ints([4]),
                                                  None) == 0
    c.advance(4)
    call = W.Call(E, [c], [4], n_q, n_kv, bf16, [base])
    qq = call.put(q[path])
    call.run(1)
    chain = call.get()
    want, tol, half = W.attend(c, 1, qq, base, n_q, n_kv)
    W.check(chain, want, tol, half, bf16)
    W.check(tree[path], want, tol, half, bf16)
