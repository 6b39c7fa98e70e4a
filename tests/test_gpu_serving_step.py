"""Steps of a server over pages: a prompt beside single tokens, then single tokens; in each step
the new K and V are appended and attended to layer by layer, the last rows' logits give the
next tokens and their log probabilities.  Every part is checked against 64 bits by the bounds of
its own tests."""
import numpy as np
import pytest

import paging as P
import windows as W
from windows import E32

pytestmark = pytest.mark.gpu

LAYERS, N_Q, N_KV, D, VOCAB, TOP, PAGE = 2, 6, 2, 64, 20001, 4, 16


@pytest.fixture(scope="module")
def E():
    import eakv_amd
    from eakv_amd import hipmem
    if hipmem.device_count() < 1:
        pytest.fail("no HIP device visible")
    return eakv_amd


@pytest.mark.parametrize("bf16", [False, True])
def test_steps(E, bf16):
    from eakv_amd import hipmem
    from eakv_amd.hipmem import DeviceArray
    rng = np.random.default_rng(5)
    held = [300, 0, 45]                                 # the second sequence is new
    new = [1, 21, 1]
    total = [a + b for a, b in zip(held, new)]
    steps = 4
    # room in the tables for the steps to come
    p = P.Pool(E, rng, [n + steps for n in total], new, PAGE, N_KV, D, layers=LAYERS)
    p.lens = held
    for layer in range(LAYERS):
        p.fill(P.contents(rng, p), layer)
    emb = rng.standard_normal((VOCAB, 32)).astype(np.float32)
    proj = {x: rng.standard_normal((LAYERS, 32, n * D)).astype(np.float32) / 6 for x, n in
            (("q", N_Q), ("k", N_KV), ("v", N_KV))}
    head = (rng.standard_normal((LAYERS * N_Q * D, VOCAB)) / 4).astype(np.float32)
    rows = [rng.integers(0, VOCAB, m) for m in new]
    for step in range(steps):
        p.new, p.lens = [len(r) for r in rows], [a + len(r) for a, r in zip(held, rows)]
        p.first = np.concatenate([[0], np.cumsum(p.new)]).astype(np.int32)
        p.rows = int(p.first[-1])
        p.d_first.upload(p.first)
        p.d_lens.upload(np.asarray(p.lens + [0], np.int32))
        p.max_new, p.max_len = max(p.new), max(p.lens)
        p.batch = p.make()
        x = emb[np.concatenate(rows)]
        outs = []
        for layer in range(LAYERS):
            kv = [np.ascontiguousarray(x @ proj[c][layer]) for c in "kv"]
            kv = [DeviceArray.from_host(W.to_bf16(y) if bf16 else y) for y in kv]
            c = P.Call(p, N_Q, N_KV, bf16)
            q = c.put((x @ proj["q"][layer]).reshape(p.rows, N_Q, D))
            p.batch.append(layer, kv[0].ptr, kv[1].ptr, "bf16" if bf16 else "f32")
            c.run(layer)
            got = c.get()
            W.check(got, *P.attend(p, layer, q, N_Q, N_KV), bf16)
            outs.append(got)
        last = p.first[1:] - 1
        z = np.concatenate([o[last].reshape(len(held), -1) for o in outs], 1) @ head
        z = W.to_bf16(z) if bf16 else z
        dz, n = DeviceArray.from_host(z), len(held)
        given = np.asarray([r[-1] for r in rows], np.int32)
        dt, lp, ent = DeviceArray.from_host(given), DeviceArray((n,)), DeviceArray((n,))
        tt, tl = DeviceArray((n, TOP), np.int32), DeviceArray((n, TOP))
        need = E.lib().eakv_token_logprobs_work_bytes(n, VOCAB, TOP)
        work = DeviceArray((need + 16,), np.uint8)
        hipmem.synchronize()
        assert E.lib().eakv_token_logprobs_device(n, VOCAB, dz.ptr, 1 if bf16 else 0, VOCAB, dt.ptr, TOP, lp.ptr,
                                                  ent.ptr, tt.ptr, tl.ptr, work.ptr, need, None) == 0
        hipmem.synchronize()
        z = (W.from_bf16(z) if bf16 else z).astype(np.float64)
        ln = z - z.max(1, keepdims=True)
        ln -= np.log(np.exp(ln).sum(1, keepdims=True))
        order = np.argsort(-z, axis=1, kind="stable")[:, :TOP]
        tops = tt.download()
        assert np.array_equal(tops, order)
        for got, want in ((tl.download(), np.take_along_axis(ln, order, 1)),
                          (lp.download(), ln[np.arange(n), given])):
            assert (np.abs(got - want) <= 80 * E32 + 2 * E32 * np.abs(want)).all()
        h1 = -(np.exp(ln) * ln).sum(1)
        assert (np.abs(ent.download() - h1) <= (80 + 165 * h1) * E32).all()
        held, rows = p.lens, [[int(t)] for t in tops[:, 0]]
