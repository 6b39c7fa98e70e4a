"""Shared by the tests of the window attention: the exact attention of a cache's
packed planes in 64 bits, and the bounds that f32 and bf16 results are held to.

Bounds, with e = 2^-24 (f32), h = 2^-11 (f16), o = 2^-8 (bf16), each half a step:

  Scores.  A score is the sum of d products of the query's two f16 parts with
  whole numbers, scaled by s, and of c * sum(q): a chain of at most d/8 matrix steps
  of 8 products and two parts each (32 f32 additions at d = 128), and 8 further
  roundings (scaling, the bias' pieces, the split of q, sum(q), the softmax scale and
  its exponent).  Each rounds a partial sum of at most
      A = sum_i |q_i| (|k_i| + |c| + |k_i - c|) / sqrt(d) <= sum |q_i| (2|k_i| + 2|c|),
  |c| <= s or |k_i|.  So |dS| <= 40 e A.
  Weights.  p is off by a factor within exp(2|dS|) after normalisation, and by
  4 e more (exp2, its argument, the sum), so the output is off by at most
      (2 max|dS| + 4e) * max|v - out| <= (80 e A + 4e) * 2 max|v|
  and by 40 e max(|v| + |c|) in the weighted sum (chain of tiles, joined in a tree).
  bf16.  V's operand rounds s, c and the value to f16, p is rounded once:
  h (|n - z| s + |c| + |v| + |v|) <= h (3 max|v| + 2 max s), and the result to bf16:
  o |out|.  Windows of many rows (k16) have K rounded to f16 too: |dS| grows by
  h sum_i |q_i| |k_i| / sqrt(d), the output by 2 |dS| * 2 max|v|.

The 2-norm over a case is held to a third of that scale, as roundings of random
sign: 4e-6 of the norm for f32 (A is about 15 for the normal data used: 40 roundings
of rms e/sqrt(3)*A/3 each give 1e-6; four times that)."""
import ctypes as C

import numpy as np

E32, H16, O16 = 2.0 ** -24, 2.0 ** -11, 2.0 ** -8


def values(cache, layer, kv):
    """(f64 values [n_kv][room][d], f64 scales [n_kv][room][d/64])."""
    w, s, b = cache.read_planes(layer, kv)
    n_kv, room, d = cache.n_heads, cache.max_seq_len, cache.head_dim
    n = np.concatenate([w & 15, w >> 4], 1).astype(np.float64)
    x = n * s[:, None].astype(np.float64) + b[:, None].astype(np.float64)
    return x.reshape(n_kv, room, d), s.astype(np.float64).reshape(n_kv, room, d // 64)


def visible(start, m, words=None):
    """bool [m][start + m]"""
    see = np.tril(np.ones((m, start + m), bool), start)
    if words is not None:
        for i in range(m):
            for j in range(m):
                see[i, start + j] = bool((int(words[i]) >> j) & 1)
    return see


def k16(m, n_q, n_kv):
    """Whether a bf16 window of m tokens may have K rounded to f16."""
    return m > 64 and m * (n_q // n_kv) > 256


def attend(cache, layer, q, start, n_q, n_kv, words=None, wide=None):
    """Exact outputs f64 [m][n_q][d] and the bound of each output's f32 part.
    wide: whether K is rounded to f16 (of more rows than q has)."""
    m, _, d = q.shape
    wide = k16(m, n_q, n_kv) if wide is None else wide
    k, ks = values(cache, layer, 0)
    v, vs = values(cache, layer, 1)
    see = visible(start, m, words)
    out = np.zeros((m, n_q, d))
    tol = np.zeros((m, n_q, d))
    half = np.zeros((m, n_q, d))
    g = n_q // n_kv
    for h in range(n_q):
        kh, vh = k[h // g, :start + m], v[h // g, :start + m]
        sh = np.repeat(vs[h // g, :start + m], 64, 1)
        kc = np.repeat(ks[h // g, :start + m], 64, 1)
        for i in range(m):
            t = see[i]
            if not t.any():
                continue
            qi = q[i, h].astype(np.float64)
            s = kh[t] @ qi / np.sqrt(d)
            p = np.exp(s - s.max())
            out[i, h] = p @ vh[t] / p.sum()
            a = (np.abs(qi) * (2 * np.abs(kh[t]) + 2 * kc[t])).sum(1).max() / np.sqrt(d)
            vm = np.abs(vh[t]).max(0)
            sm = sh[t].max(0)
            tol[i, h] = (80 * E32 * a + 4 * E32) * 2 * vm + 40 * E32 * (vm + sm)
            half[i, h] = H16 * (3 * vm + 2 * sm)
            if wide:
                half[i, h] += 4 * H16 * (np.abs(kh[t]) @ np.abs(qi)).max() / np.sqrt(d) * vm
    return out, tol, half


def check(got, want, tol, half, bf16):
    got, want = got.astype(np.float64), np.asarray(want)
    lim = tol + (half + O16 * np.abs(want) if bf16 else 0.0) + 1e-30
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= lim).all(), (float((err / lim).max()), np.argwhere(err > lim)[:3].tolist())
    norm = np.linalg.norm(want)
    rel = np.linalg.norm(err) / norm if norm else 0.0
    assert rel <= (2 * O16 / 3 if bf16 else 4e-6), rel
    return rel


def to_bf16(x):
    """f32 -> the nearest bf16's bits (ties to even; finite x)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def build(E, rng, lens, n_kv, d, room, layers=1, scale=None):
    caches = []
    for n in lens:
        c = E.Cache(layers, n_kv, d, room)
        if n:
            x = rng.standard_normal((layers, 2, n_kv, n, d), dtype=np.float32)
            if scale is not None:
                x *= scale
            c.load_raw(x, n)
        caches.append(c)
    return caches


class Call:
    """One window call: device buffers with guard rows, one canary row each side."""
    GUARD = 0x7b

    def __init__(self, E, caches, n_tokens, n_q, n_kv, bf16, starts=None, words=None, shift=0):
        from eakv_amd.hipmem import DeviceArray
        self.E, self.caches, self.bf16, self.shift = E, caches, bf16, shift
        self.total, self.n_q, self.d = sum(n_tokens), n_q, caches[0].head_dim
        self.plan = E.WindowPlan(caches, n_tokens, n_q, n_kv, starts=starts,
                                 dtype="bf16" if bf16 else "f32")
        self.size = 2 if bf16 else 4
        self.row = n_q * self.d * self.size
        # shift: elements that the buffers are moved off their alignment
        self.dq = DeviceArray(((self.total + 2) * self.row + 64,), np.uint8)
        self.do = DeviceArray(((self.total + 2) * self.row + 64,), np.uint8)
        self.dt = None if words is None else DeviceArray.from_host(np.asarray(words, np.uint64))
        self.at = self.row + shift * self.size

    def put(self, q):
        u = to_bf16(q) if self.bf16 else np.ascontiguousarray(q, np.float32)
        host = np.full(self.dq.nbytes, self.GUARD, np.uint8)
        host[self.at:self.at + u.nbytes] = u.reshape(-1).view(np.uint8)
        self.dq.upload(host)
        return from_bf16(u) if self.bf16 else u

    def run(self, layer=0, stream=None, work=None, work_bytes=0, clear=True):
        if clear:
            self.do.upload(np.full(self.do.nbytes, self.GUARD, np.uint8))
        self.plan.run(layer, self.dq.ptr + self.at, self.do.ptr + self.at,
                      None if self.dt is None else self.dt.ptr, work, work_bytes, stream)

    def get(self, sync=True):
        if sync:
            self.caches[0].sync()
        host = self.do.download()
        n = self.total * self.row
        inner = host[self.at:self.at + n]
        # rows before and behind the windows' stay as they were
        assert (host[:self.at] == self.GUARD).all() and (host[self.at + n:] == self.GUARD).all()
        u = inner.copy().view(np.uint16 if self.bf16 else np.float32)
        x = from_bf16(u) if self.bf16 else u
        return x.reshape(self.total, self.n_q, self.d)


class Graph:
    """A HIP graph recorded from the calls that `record` makes on a stream."""

    def __init__(self, record):
        from eakv_amd import hipmem
        self.h = h = hipmem.hip()
        self.st = hipmem.Stream()
        for n, a in (("hipStreamBeginCapture", [C.c_void_p, C.c_int]),
                     ("hipStreamEndCapture", [C.c_void_p, C.c_void_p]),
                     ("hipGraphInstantiate", [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                              C.c_size_t]),
                     ("hipGraphLaunch", [C.c_void_p, C.c_void_p]),
                     ("hipGraphExecDestroy", [C.c_void_p]), ("hipGraphDestroy", [C.c_void_p])):
            f = getattr(h, n)
            f.argtypes, f.restype = a, C.c_int
        hipmem.check(h.hipStreamBeginCapture(self.st.s, 2), "begin")     # relaxed
        self.graph = C.c_void_p()
        try:
            record(self.st.s)
        finally:
            rc = h.hipStreamEndCapture(self.st.s, C.byref(self.graph))
        hipmem.check(rc, "end")
        self.exe = C.c_void_p()
        hipmem.check(h.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, 0),
                     "instantiate")

    def launch(self):
        from eakv_amd import hipmem
        hipmem.check(self.h.hipGraphLaunch(self.exe, self.st.s), "launch")
        self.st.synchronize()

    def free(self):
        self.h.hipGraphExecDestroy(self.exe)
        self.h.hipGraphDestroy(self.graph)
