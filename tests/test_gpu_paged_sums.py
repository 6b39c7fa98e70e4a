"""bf16 queries over pages where K's steps are large: keys with outliers, queries with one large dim.

Bound, beside that of paging.py: the matrix cores lose up to 2^-11 of a step times the largest operand
of a sum with subnormal nibbles.  A score may so be off by dS = sum over groups of 2^-11 s max|q| /
sqrt(d) more and a result by 2 dS times 2 max|v| (windows.py), or by 2^-11 max s of V, as the weights of
32 tokens are at most 1 together with the others'."""
import numpy as np
import pytest

import paging as P
import windows as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


def bound(p, q, n_q, n_kv):
    """What the sums may lose, f64 [rows][n_q][d]."""
    _, ks = W.values(p.pool, 0, 0)
    v, vs = W.values(p.pool, 0, 1)
    d, g = q.shape[2], n_q // n_kv
    more = np.zeros(q.shape)
    for s, (n, m) in enumerate(zip(p.lens, p.new)):
        at = p.place(s)
        for h in range(n_q):
            vm, sm = np.abs(v[h // g, at]).max(0), np.repeat(vs[h // g, at].max(0), 64)
            for i in range(m):
                r = p.first[s] + i
                top = np.abs(q[r, h]).reshape(-1, 64).max(1)
                ds = 2.0 ** -11 * (ks[h // g, at] * top).sum(1).max() / np.sqrt(d)
                more[r, h] = 2 * ds * 2 * vm + 2.0 ** -11 * sm
    return more


@pytest.mark.parametrize("n_q,n_kv,d,lens,new", [(8, 2, 128, [700, 90], [1, 1]), (4, 1, 64, [500], [9]),
                                                 (6, 2, 64, [300, 33], [40, 20])])
@pytest.mark.parametrize("k_top,q_top", [(1.0, 60.0), (40.0, 1.0), (12.0, 12.0)])
@pytest.mark.parametrize("large", [False, True])
def test_large_steps(E, rng, n_q, n_kv, d, lens, new, k_top, q_top, large):
    p = P.Pool(E, rng, lens, new, 16, n_kv, d, ld_more=(1 << 27) // (sum(new) * n_q) // 16 + 2 if large else 0)
    x = P.contents(rng, p)
    for y in x:
        y[0][:, :, 7] *= k_top                  # one dim of each key, and of each query
    p.fill(x)
    c = P.Call(p, n_q, n_kv, True)
    q = rng.standard_normal((p.rows, n_q, d)).astype(np.float32)
    q[:, :, 9] *= q_top
    q = c.put(q)
    c.run(batch=p.make(max_len=(1 << 27) // (p.rows * n_q) + 1) if large else None)
    want, tol, half = P.attend(p, 0, q, n_q, n_kv)
    err = np.abs(c.get().astype(np.float64) - want)
    lim = tol + half + W.O16 * np.abs(want) + bound(p, q, n_q, n_kv)
    assert (err <= lim).all(), float((err / lim).max())
