"""Paged attention on the smallest numbers of the pages' types: keys and values below their normal ranges count in full
(bound: paged_cases.attend)."""
import numpy as np
import pytest

import test_gpu_paged_attn as A
import paged_cases as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,shift", [("f16", 18), ("f16", 22), ("e4m3", 7), ("e4m3", 9), ("bf16", 60), ("f32", 60)])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("T,hd,ps", [(3, 64, 16), (6, 128, 7)])   # 6 rows of 3 requests: shared tiles
def test_subnormals(moehip, kind, shift, side, T, hd, ps):
    dtype = C.TYPES[kind]
    b = A.Batch(moehip, dtype, [40, 300, 1], 8, 2, hd, ps, seed=51)
    pool, f = getattr(b.pool, side), b.pool.factor("kv".index(side))
    for r, n in enumerate(b.lens):
        p = np.arange(n)
        slot = (b.tables[r][p // ps], p % ps)
        pool[slot] = C.encode((b.rng.standard_normal((n, 2, hd)) * 2.0 ** -shift).astype(np.float32), dtype)
    b.pool.upload()
    q = b.rng.standard_normal((T, b.ld)).astype(np.float32)
    if side == "k":   # scores of ordinary size all the same
        q *= np.float32(2.0 ** shift / f.mean())
    req, pos = [0, 1, 2, 1, 1, 0][:T], [39, 299, 0, 298, 150, 38][:T]
    out, q = b.run(req=req, pos=pos, T=T, q=q)
    for t in range(T):
        k, v = b.pool.rows(b.tables[req[t]], pos[t] + 1)
        want, tol = C.attend(q[t].astype(np.float64), k, v, b.scale)
        got = out[t].reshape(b.nq, hd)
        assert (np.abs(got - want) <= tol).all(), f"row {t}: {np.max(np.abs(got - want) / tol):.2f} times the bound"
