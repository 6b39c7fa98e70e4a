"""Shared by the tests of sequences in pages: a pool with tables, the exact attention of its
packed planes in 64 bits, and the bounds of results.

Bounds: those of windows.py (e = 2^-24, h = 2^-11, o = 2^-8, each half a step).  bf16: x = p s
(n the nibble, z the one nearest 0), p and c are rounded to f16, x once in both of the sums of x n
and x z, so that its error is of x (n - z): h (|v - c| + 2 |c|), and a product with a nibble comes
out to 2^-17: 2^-17 15 s < h s / 4; together h (3 max|v| + 2 max s), |c| <= s or |v|."""
import numpy as np

import windows as W
from windows import E32, H16


class Pool:
    """Sequences of given lengths in a pool's pages, in any order of pages; places of the
    tables behind a sequence's last page hold numbers outside the pool."""

    def __init__(self, E, rng, lens, new, page, n_kv, d, layers=1, spare=3, ld_more=0, ragged=True,
                 bad=()):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.lens, self.new, self.page = E, list(lens), list(new), page
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        self.pool = E.Cache(layers, n_kv, d, self.n_pages * page + page // 2)
        self.ld = max(need + [1]) + ld_more
        self.table = np.full((len(lens), self.ld), 1 << 30, np.int32)
        order = rng.permutation(self.n_pages)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = order[at:at + k]
            at += k
        for s, k, p in bad:                     # pages that hold nothing
            self.table[s, k] = p
        self.first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.first[-1])
        self.d_table = DeviceArray.from_host(self.table)
        self.d_lens = DeviceArray.from_host(np.asarray(list(lens) + [0], np.int32))
        self.d_first = DeviceArray.from_host(self.first)
        self.max_new, self.max_len = max(list(new) + [0]), max(list(lens) + [0])
        self.batch = self.make(ragged)

    def make(self, ragged=True, **kw):
        a = dict(max_len=self.max_len, max_new=self.max_new,
                 d_first=self.d_first.ptr if ragged else None, n_new=self.rows)
        a.update(kw)
        return self.E.PagedBatch(self.pool, self.page, self.d_table.ptr, self.ld, self.d_lens.ptr,
                                 len(self.lens), **a)

    def place(self, s):
        """Pool tokens of sequence s's positions, -1 where it has none."""
        t = np.arange(self.lens[s])
        p = self.table[s, t // self.page] if len(t) else t
        return np.where((p >= 0) & (p < self.n_pages), p * self.page + t % self.page, -1)

    def fill(self, x, layer=0):
        """x: per sequence f32 [2][n_kv][len][d], appended whole through the pages."""
        from eakv_amd.hipmem import DeviceArray
        rows = [np.ascontiguousarray(y.transpose(0, 2, 1, 3)) for y in x]
        kv = [DeviceArray.from_host(np.concatenate([r[j] for r in rows])) for j in (0, 1)]
        first = DeviceArray.from_host(np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32))
        b = self.make(d_first=first.ptr, n_new=sum(self.lens), max_new=self.max_len)
        b.append(layer, kv[0].ptr, kv[1].ptr)
        self.pool.sync()
        return kv, first


def contents(rng, pool, scale=1.0):
    c = pool.pool
    return [(rng.standard_normal((2, c.n_heads, n, c.head_dim)) * scale).astype(np.float32)
            for n in pool.lens]


def attend(pool, layer, q, n_q, n_kv):
    """Exact outputs f64 [rows][n_q][d] and the bounds of their f32 and their f16 parts."""
    kk, ks = W.values(pool.pool, layer, 0)
    vv, vs = W.values(pool.pool, layer, 1)
    d, g = q.shape[2], n_q // n_kv
    out, tol, half = (np.zeros(q.shape) for _ in range(3))
    for s, (n, m) in enumerate(zip(pool.lens, pool.new)):
        at = pool.place(s)
        pos = np.nonzero(at >= 0)[0]
        at = at[pos]
        for h in range(n_q):
            k, v = kk[h // g, at], vv[h // g, at]
            kc, sm = np.repeat(ks[h // g, at], 64, 1), np.repeat(vs[h // g, at], 64, 1)
            qs = q[pool.first[s]:pool.first[s + 1], h].astype(np.float64)
            sc = qs @ k.T / np.sqrt(d)
            a = np.abs(qs) @ (2 * np.abs(k) + 2 * kc).T / np.sqrt(d)
            for i in range(m):
                see = int(np.searchsorted(pos, n - m + i, side="right"))
                if see == 0:
                    continue
                p = np.exp(sc[i, :see] - sc[i, :see].max())
                r = pool.first[s] + i
                out[r, h] = p @ v[:see] / p.sum()
                vm, s_ = np.abs(v[:see]).max(0), sm[:see].max(0)
                tol[r, h] = (80 * E32 * a[i, :see].max() + 4 * E32) * 2 * vm + 40 * E32 * (vm + s_)
                half[r, h] = H16 * (3 * vm + 2 * s_)
    return out, tol, half


class Call:
    """One attention call: buffers with guard rows each side, any distance between tokens."""
    GUARD = 0x7b

    def __init__(self, pool, n_q, n_kv, bf16, more=(0, 0), shift=0):
        from eakv_amd.hipmem import DeviceArray
        self.p, self.n_q, self.n_kv, self.bf16 = pool, n_q, n_kv, bf16
        self.d = pool.pool.head_dim
        self.size = 2 if bf16 else 4
        self.width = n_q * self.d
        self.ld = [self.width + m for m in more]
        self.shift = shift
        self.buf = [DeviceArray(((pool.rows + 2) * ld * self.size + 64,), np.uint8) for ld in self.ld]
        self.dtype = "bf16" if bf16 else "f32"

    def at(self, j):
        return self.buf[j].ptr + (self.ld[j] + self.shift) * self.size

    def _rows(self, j, host):
        t = np.uint16 if self.bf16 else np.float32
        x = host[(self.ld[j] + self.shift) * self.size:]
        x = x[:self.p.rows * self.ld[j] * self.size].view(t).reshape(self.p.rows, self.ld[j])
        return x[:, :self.width]

    def put(self, q):
        host = np.full(self.buf[0].nbytes, self.GUARD, np.uint8)
        u = W.to_bf16(q) if self.bf16 else np.ascontiguousarray(q, np.float32)
        self._rows(0, host)[:] = u.reshape(self.p.rows, -1)
        self.buf[0].upload(host)
        return W.from_bf16(u) if self.bf16 else u

    def run(self, layer=0, batch=None, clear=True, **kw):
        if clear:
            self.buf[1].upload(np.full(self.buf[1].nbytes, self.GUARD, np.uint8))
        (batch or self.p.batch).attend(layer, self.at(0), self.at(1), self.n_q, self.n_kv, self.dtype,
                                       ld_q=self.ld[0], ld_out=self.ld[1], **kw)

    def get(self, sync=True):
        if sync:
            self.p.pool.sync()
        host = self.buf[1].download()
        rows = self._rows(1, host)
        got = rows.copy()
        rows[:] = np.frombuffer(
            bytes([self.GUARD]) * self.size, rows.dtype)[0]
        assert (host == self.GUARD).all()       # everything around the rows is as it was
        x = W.from_bf16(got) if self.bf16 else got
        return x.reshape(self.p.rows, self.n_q, self.d)
