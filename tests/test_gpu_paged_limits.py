"""Steps of moe_model_step_paged that cannot be done whole: the requests' state stays as it was, and what failed is not
told of the calls after it."""
import numpy as np
import pytest

import oracle as O
import paged_cases as C

pytestmark = pytest.mark.gpu


def test_failed_call_and_the_next(moehip):
    """Memory that is not there is refused once; the call after it is done."""
    M = moehip
    x, w = np.linspace(-1, 1, 64, dtype=np.float32), np.ones(64, np.float32)
    bufs = [M.DeviceBuffer.from_array(a) for a in (x, w, np.zeros(64, np.float32))]
    with pytest.raises(M.MoeError, match="emory"):
        M.DeviceBuffer(1 << 42)
    M.check(M.lib().moe_rmsnorm_dev(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, 1, 64, 1e-6), "rmsnorm")
    np.testing.assert_array_equal(bufs[2].download((64,), np.float32), O.rmsnorm(x.reshape(1, 64), w)[0])


def _model(M, dff):
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=dff, E=8, top_k=8, V=97, seed=5)
    return tm, M.model_from_tiny(tm)


def _state(c):
    return [c.array(n, k) for n, k in (("held", c.n_req), ("ring_at", 2), ("ring", 24), ("tables", 12), ("status", 1))]


def test_memory_that_is_not_there(moehip):
    """Scratch of half a terabyte for the experts: the step fails before its plan, and the next one is done."""
    M = moehip
    tm, m = _model(M, 8192)
    c = M.PagedCache(tm.L, tm.nkv, tm.hd, 24, 8, 2, 6, 4)
    c.set_step([2, 1], [1, 2, 3])
    before = _state(c)
    rows = 4_000_000
    # arrays of that many rows for the plan alone: the step does not get as far as using them
    big = {n: M.DeviceBuffer(4 * rows) for n in ("req", "pos", "slot", "ids")}
    plan = type(c.plan).from_buffer_copy(c.plan)
    plan.max_tokens, plan.req, plan.pos, plan.slot = rows, big["req"].ptr, big["pos"].ptr, big["slot"].ptr
    lg, nx = M.DeviceBuffer(2 * tm.V * 4), M.DeviceBuffer(8)
    print("paged step of", rows, "rows", flush=True)
    assert M.lib().moe_model_step_paged(m.h, C.ref(plan), c.layers, big["ids"].ptr, lg.ptr, nx.ptr) == 1
    assert b"emory" in M.lib().moe_last_error()
    for a, b in zip(_state(c), before):
        np.testing.assert_array_equal(a, b)
    got, _ = m.step_paged(c, [2, 1], [1, 2, 3])
    assert c.status == 0 and np.isfinite(got).all()
    np.testing.assert_array_equal(c.array("held", 2), [2, 1])
    m.close()
