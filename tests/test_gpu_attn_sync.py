"""What a synchronisation costs once attention-side calls were made, and that it still reports."""
import statistics
import time

import numpy as np
import pytest

import moe_rocm as M

pytestmark = pytest.mark.gpu


def idle_sync(ctx):
    """Microseconds of a synchronisation with nothing to wait for: the middle of 400."""
    t = []
    for _ in range(400):
        a = time.perf_counter()
        ctx.sync()
        t.append(time.perf_counter() - a)
    return statistics.median(t) * 1e6


def test_a_sync_costs_no_copy_after_attention_calls():
    """A copy of a few bytes from the device takes 12 us here, a synchronisation of an idle stream half of one. 4 us
    lie between them by a factor of three at least on both sides."""
    used, fresh = M.Context(0), M.Context(0)
    kv = M.KvCache(used, M.KV_MXFP4, 4, 64, 2, 64)
    x, slots = used.to_device(np.zeros((2, 2, 64), np.float32)), used.to_device(np.array([3, 4 * 64], np.int32))
    h = M.Heads(x.ptr, 2)
    for n in (1, 2):
        kv.write(h, h, n, slots)
        if n == 2:  # the second slot is behind the last page
            with pytest.raises(M.MoeRocmError) as ei:
                used.sync()
            assert ei.value.status == M.MR_E_INVAL and "slots" in ei.value.message
        used.sync()
        assert idle_sync(used) <= idle_sync(fresh) + 4.0
    x.free(), slots.free(), kv.close()
    used.close(), fresh.close()


def test_errors_of_one_context_are_not_anothers():
    a, b = M.Context(0), M.Context(0)
    kv = [M.KvCache(c, M.KV_MXFP4, 4, 64, 2, 64) for c in (a, b)]
    rows = [(c.to_device(np.zeros((1, 2, 64), np.float32)), c.to_device(np.array([s], np.int32))) for c, s in ((a, 1000), (b, 3))]
    for k, (x, s) in zip(kv, rows):
        k.write(M.Heads(x.ptr, 2), M.Heads(x.ptr, 2), 1, s)
    b.sync()
    with pytest.raises(M.MoeRocmError):
        a.sync()
    a.sync(), b.sync()
    for k, (x, s) in zip(kv, rows):
        x.free(), s.free(), k.close()
    a.close(), b.close()
