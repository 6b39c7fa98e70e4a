"""Window calls whose buffers touch one another, and the workspace's size."""
import numpy as np
import pytest

import windows as W
from test_gpu_window import E  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
def test_overlapping_buffers(E, rng, bf16):
    """Scratch over queries, outputs or a tree's words, and outputs over those words, are
    refused; outputs in the queries' own place give the same bits."""
    from eakv_amd.hipmem import DeviceArray
    caches = W.build(E, rng, [9000, 80], 2, 128, 9000)
    ms, n_q = [6, 70], 64
    call = W.Call(E, caches, ms, n_q, 2, bf16, [8994, 10])
    q = rng.standard_normal((call.total, n_q, 128), dtype=np.float32)
    call.put(q)
    call.run()
    want = call.get()
    rows, need = call.total * call.row, call.plan.work_bytes
    assert need > 16
    buf = DeviceArray((2 * rows + need + 64,), np.uint8)
    a = buf.ptr

    def run(q, out, tree, work, plan=call.plan):
        with pytest.raises(E.EakvError) as e:
            plan.run(0, q, out, tree, work, need)
        assert e.value.code == E.EAKV_ERR_INVALID

    far = a + (2 * rows + 63) // 64 * 64
    run(a, a + rows, None, a + rows - 16)
    run(a, a + rows, None, a + 2 * rows - 16)
    run(a, a + rows, None, a)
    small = E.WindowPlan(caches, [3, 3], n_q, 2, starts=[8994, 10], dtype="bf16" if bf16 else "f32")
    run(a, a + rows, a + rows, far, small)
    run(a, a + rows, far + 8, far, small)
    host = W.to_bf16(q) if bf16 else q
    same = DeviceArray.from_host(host.reshape(-1))
    call.plan.run(0, same.ptr, same.ptr, None, far, need)
    caches[0].sync()
    got = same.download()
    got = W.from_bf16(got) if bf16 else got
    assert np.array_equal(got.reshape(want.shape).view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d,n_kv,ctx,seqs", [(128, 8, 1_000_000, 1), (64, 16, 120_000, 32)])
def test_workspace_is_bounded(E, d, n_kv, ctx, seqs, bf16):
    """Operands of every token would take more than 4 GiB: the call goes without them."""
    caches = [E.Cache(1, n_kv, d, ctx) for _ in range(seqs)]
    for c in caches:
        c.advance(ctx)
    for m in (130, 2000):
        p = E.WindowPlan(caches, [m] * seqs, n_kv * 8, n_kv, starts=[ctx - m] * seqs,
                         dtype="bf16" if bf16 else "f32")
        assert p.work_bytes <= (4 << 30) + seqs * m * n_kv * 8 * (d + 2) * 4 * 64
    short = E.WindowPlan(caches, [2000] * seqs, n_kv * 8, n_kv, starts=[0] * seqs,
                         dtype="bf16" if bf16 else "f32")
    assert short.work_bytes >= seqs * 2000 // 32 * n_kv * d * 128       # expanded
    for c in caches:
        c.free()
