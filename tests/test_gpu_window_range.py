"""Windows (eakv_attention_window_batch_device) at values where an operand of 16 bits would
show: K on an offset, tokens of very different magnitudes side by side, queries of zeros and
near the end of f32's range; against the exact attention of the cache's own planes in 64
bits, by both ways that a window takes (kernels of few rows, expanded operands).  Bounds in
windows.py, and K exact (wide=False) in all of them."""
import numpy as np
import pytest

import windows as W
from test_gpu_window import E  # noqa: F401  (the fixture)
from test_gpu_window_prompt import Head, expanded

pytestmark = pytest.mark.gpu

# (kv heads, q heads, [(start, tokens)]): few rows per kv head; many, expanded
FEW = (2, 4, [(40, 12)])
MANY = (8, 128, [(40, 72)] * 3)
WAYS = [FEW, MANY]


def data(rng, way, d):
    """Caches' K and V [1][2][n_kv][t][d] and queries, of normal values."""
    n_kv, n_q, wins = way
    xs = [rng.standard_normal((1, 2, n_kv, s + m, d), dtype=np.float32) for s, m in wins]
    return xs, rng.standard_normal((sum(m for _, m in wins), n_q, d), dtype=np.float32)


def attend(E, way, d, xs, q, bf16, words=None):
    """Outputs [rows][n_q][d] and the queries as the kernel reads them, with the caches."""
    n_kv, n_q, wins = way
    caches = []
    for x in xs:
        c = E.Cache(1, n_kv, d, x.shape[3] + 5)
        c.load_raw(x, x.shape[3])
        caches.append(c)
    call = W.Call(E, caches, [m for _, m in wins], n_q, n_kv, bf16, [s for s, _ in wins], words)
    assert way is not MANY or expanded(call, wins, n_kv)
    q = call.put(q)
    call.run()
    return call.get(), q, caches


def sample(n_kv, n_q):
    """(kv head, q head) pairs to look at."""
    g = n_q // n_kv
    return sorted({(k, k * g + i) for k in (0, n_kv - 1) for i in (0, g - 1)})


def exact(cache, q, start, k, words=None):
    return W.attend(Head(cache, k), 0, np.ascontiguousarray(q[:, None]), start, 1, 1, words, wide=False)


def verify(way, got, q, caches, bf16, words=None, rows=None):
    """The sampled heads of every window, or of its `rows` (bool by token)."""
    n_kv, n_q, wins = way
    at = 0
    for c, (s, m) in zip(caches, wins):
        pick = np.ones(m, bool) if rows is None else rows
        for k, h in sample(n_kv, n_q):
            want, tol, half = exact(c, q[at:at + m, h], s, k, words)
            rel = W.check(got[at:at + m, h][pick], want[pick, 0], tol[pick, 0], half[pick, 0], bf16)
        print("  rel", rel, flush=True)
        at += m


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_keys_on_an_offset(E, rng, way, d, bf16):
    """K = 100 + normal values: rounded to f16 (steps of 1/16) the scores are off by
    1/16/sqrt(12) = 0.018 each, and the output by as much of its norm.  Exact K: c * sum(q)
    in three pieces each is off by some 2^-23 * 100 * |sum(q)| / sqrt(d) = 1e-5, in f32 four
    times the norm's bound at scores of normal data: 4e-5 is asked for."""
    xs, q = data(rng, way, d)
    for x in xs:
        x[:, 0] += 100.0
    got, q, caches = attend(E, way, d, xs, q, bf16)
    at = 0
    n_kv, n_q, wins = way
    for c, (s, m) in zip(caches, wins):
        for k, h in sample(n_kv, n_q):
            want, tol, half = exact(c, q[at:at + m, h], s, k)
            err = np.abs(got[at:at + m, h] - want[:, 0])
            lim = tol[:, 0] + (half[:, 0] + W.O16 * np.abs(want[:, 0]) if bf16 else 0.0)
            assert (err <= lim).all()
            rel = np.linalg.norm(err) / np.linalg.norm(want)
            print("  rel", rel, flush=True)
            assert rel <= (2 * W.O16 / 3 if bf16 else 4e-5)
        at += m


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e12, 1e18])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_magnitude_of_a_token_not_seen(E, rng, way, d, size, bf16):
    """Later tokens of the window with K and V of `size`, in the same 32 tokens as those
    that the earlier rows see: the same bits as with tokens of ordinary size."""
    n_kv, n_q, wins = way
    xs, q = data(rng, way, d)
    plain = attend(E, way, d, xs, q, bf16)[0]
    for x, (s, m) in zip(xs, wins):
        x[:, 1, :, s + m - 4] *= size
        x[:, :, :, s + m - 2] *= size
    got, q, caches = attend(E, way, d, xs, q, bf16)
    m = wins[0][1]
    rows = np.arange(m) < m - 4
    verify(way, got, q, caches, bf16, rows=rows)
    every = np.tile(rows, len(wins))
    assert np.array_equal(got[every].view(np.uint32), plain[every].view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e12])
@pytest.mark.parametrize("d", [64, 128])
def test_magnitude_of_another_branch(E, rng, d, size, bf16):
    """A tree's node with K and V of `size`, seen by its own row alone."""
    n_kv, n_q, wins = FEW
    (s, m), = wins
    words = [(1 << i + 1) - 1 & ~(1 << 5) for i in range(m)]
    words[5] |= 1 << 5
    xs, q = data(rng, FEW, d)
    xs[0][:, :, :, s + 5] *= size
    got, q, caches = attend(E, FEW, d, xs, q, bf16, words)
    verify(FEW, got, q, caches, bf16, words, rows=np.arange(m) != 5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_magnitude_of_a_token_without_weight(E, rng, way, d, size, bf16):
    """A token with a score some 100 below the others' (weight e^-100) and V of `size`."""
    xs, q = data(rng, way, d)
    q += 1.0
    for x in xs:
        x[:, 0, :, 17] = -16.0 if d == 64 else -12.0
        x[:, 1, :, 17] *= size
    got, q, caches = attend(E, way, d, xs, q, bf16)
    verify(way, got, q, caches, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e-3, 1e3])
@pytest.mark.parametrize("way", WAYS)
def test_magnitudes_that_vary(E, rng, way, size, bf16):
    """V's size changes from token to token over 18 powers of ten around `size`; the
    largest decide the outputs."""
    xs, q = data(rng, way, 128)
    for x in xs:
        x[:, 1] *= (size * 10.0 ** rng.uniform(-9, 9, x.shape[3])).astype(np.float32)[:, None]
    got, q, caches = attend(E, way, 128, xs, q, bf16)
    verify(way, got, q, caches, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-3, 1.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_queries_of_zeros(E, rng, way, d, size, bf16):
    """Rows of zeros (and of values far below the normal f16) give the mean of the V that
    they see, whatever K's size; planes of zeros as a new cache has them among those."""
    xs, q = data(rng, way, d)
    for x in xs:
        x[:, 0] *= size
    q[::2] = 0.0
    q[1::4] *= 1e-36
    got, q, caches = attend(E, way, d, xs, q, bf16)
    verify(way, got, q, caches, bf16)


@pytest.mark.parametrize("way", WAYS)
def test_room_of_a_new_cache(E, rng, way):
    """K and V never written, all zeros: zeros come out, for zero queries too."""
    n_kv, n_q, wins = way
    for bf16 in (False, True):
        caches = [E.Cache(1, n_kv, 128, s + m) for s, m in wins]
        for c, (s, m) in zip(caches, wins):
            c.advance(s + m)
        call = W.Call(E, caches, [m for _, m in wins], n_q, n_kv, bf16, [s for s, _ in wins])
        q = rng.standard_normal((call.total, n_q, 128), dtype=np.float32)
        q[::3] = 0.0
        call.put(q)
        call.run()
        assert (call.get() == 0.0).all()


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("d", [64, 128])
def test_queries_near_the_end_of_the_range(E, rng, way, d):
    """bf16 queries beyond 2^121 against K of 2^-116: scores of standard deviation 16.  (The
    third piece of K's biases lies below bf16's range: 2^-16 of them is lost, 2e-4 of a
    score, far below the bound.)"""
    xs, q = data(rng, way, d)
    for x in xs:
        x[:, 0] *= 2.0 ** -116
    q *= np.float32(2.0 ** 120)
    got, q, caches = attend(E, way, d, xs, q, True)
    verify(way, got, q, caches, True)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("way", [(2, 8, [(9000, 6)]), (4, 64, [(1500, 512)])])
def test_nonfinite_value_in_a_chunk_without_weight(E, rng, way, bf16):
    """NaN in V of a token whose whole chunk lies hundreds of powers of two below the rows'
    maximum: NaN in its 64 dims as anywhere else, and nowhere else."""
    n_kv, n_q, ((s, m),) = way
    d = 128
    x = rng.standard_normal((1, 2, n_kv, s + m, d), dtype=np.float32)
    x[:, 0, :, :s - 100] = -24.0
    x[0, 1, 0, 33, 64] = np.nan                  # a group's first value: its scale and bias
    c = E.Cache(1, n_kv, d, s + m)
    c.load_raw(x, s + m)
    call = W.Call(E, [c], [m], n_q, n_kv, bf16, [s])
    call.put(rng.standard_normal((m, n_q, d), dtype=np.float32) * 0.5 + 1.0)
    call.run()
    nan = np.isnan(call.get())
    want = np.zeros_like(nan)
    want[:, :n_q // n_kv, 64:] = True
    assert np.array_equal(nan, want)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("way", [(2, 8, [(9000, 6)]), (4, 64, [(1500, 512)])])
def test_nonfinite_queries_over_chunks(E, rng, way, bf16):
    """NaN and infinite queries: NaN in their own rows alone, whatever the chunks."""
    n_kv, n_q, ((s, m),) = way
    c = W.build(E, rng, [s + m], n_kv, 128, s + m)[0]
    call = W.Call(E, [c], [m], n_q, n_kv, bf16, [s])
    q = rng.standard_normal((m, n_q, 128), dtype=np.float32)
    want = np.zeros(q.shape, bool)
    for i, (row, head, x) in enumerate(((0, 1, np.nan), (3, 0, np.inf), (5, n_q - 1, -np.inf))):
        q[row, head, 17 * i] = x
        want[row, head] = True
    if bf16:
        bits = W.to_bf16(np.where(np.isnan(q), np.float32(1), q))
        call.put(q)
        bits[np.isnan(q)] = 0x7fc0
        host = np.full(call.dq.nbytes, call.GUARD, np.uint8)
        host[call.at:call.at + bits.nbytes] = bits.reshape(-1).view(np.uint8)
        call.dq.upload(host)
    else:
        call.put(q)
    call.run()
    assert np.array_equal(np.isnan(call.get()), want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way", [(2, 8, [(33, 65)]), (2, 2, [(0, 300)]), (1, 16, [(100, 140)]),
                                 (8, 128, [(16, 80), (0, 97), (200, 65)])])
def test_k_is_exact_for_bf16_windows_of_many_rows(E, rng, way, d):
    """The bound without a rounding of K, for windows of more than 256 rows per kv head, by
    whichever way they go, with outlier channels in K."""
    n_kv, n_q, wins = way
    xs, q = data(rng, way, d)
    for x in xs:
        x[:, 0, ..., [3, d - 9]] *= 10.0
    caches = [E.Cache(1, n_kv, d, max(s + m for s, m in wins)) for _ in wins]
    for c, x in zip(caches, xs):
        c.load_raw(x, x.shape[3])
    call = W.Call(E, caches, [m for _, m in wins], n_q, n_kv, True, [s for s, _ in wins])
    q = call.put(q)
    call.run()
    verify(way, call.get(), q, caches, True)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e19, 1e35, -3e38])
@pytest.mark.parametrize("way", WAYS)
def test_constant_groups_of_any_size(E, rng, way, size, bf16):
    """Groups of 64 equal values have scale 1 beside a bias of their size.  A token of such
    groups near the end of f32's range leaves the rows that do not see it alone, and the rows
    that do get their weight of it.

    The token's exponent e (f32: of 2^-24 of its values) is added to its scores, so that the
    3 roundings behind that are of sums of |e| + |score|, half a step each: up to 3 e 2^-24
    in log2 units, ln 2 of which is the weight's error, and the normalisation's at most as
    much again: 6 ln 2 e 2^-24 beside the norm's usual bound, 2.4e-5 at 1e35."""
    n_kv, n_q, wins = way
    xs, q = data(rng, way, 128)
    for x, (s, m) in zip(xs, wins):
        x[:, 1, :, s + m - 3] = size
    got, q, caches = attend(E, way, 128, xs, q, bf16)
    m = wins[0][1]
    verify(way, got, q, caches, bf16, rows=np.arange(m) < m - 3)
    bound = 2 * W.O16 / 3 if bf16 else 4e-6
    bound += 6 * np.log(2) * (np.log2(abs(size)) + 1 - (0 if bf16 else 24)) * W.E32
    at = 0
    for c, (s, m) in zip(caches, wins):
        for k, h in sample(n_kv, n_q):
            want = exact(c, q[at:at + m, h], s, k)[0][m - 3:, 0]
            rel = np.linalg.norm(got[at + m - 3:at + m, h] - want) / np.linalg.norm(want)
            assert rel <= bound, rel
        at += m
