"""The 64-bit model and its bound (model64.py) against the fp32 oracle, which is the reference's model bit for bit.  CPU
only."""
import numpy as np
import pytest

import model64
import oracle as O


@pytest.mark.parametrize("experts,seed,nq,nkv,bias", [(False, 1, 4, 2, False), (False, 2, 4, 2, True), (False, 3, 16, 2, False), (True, 1, 4, 2, False),
                                                      (True, 2, 4, 2, True)])
def test_oracle_within_the_bound(experts, seed, nq, nkv, bias):
    tm = model64.plain_model(O, seed, 1, experts, nq=nq, nkv=nkv, bias=bias)
    ids = np.random.default_rng(seed).integers(0, tm.V, 60)
    tables = O.rope_tables(tm.hd, tm.theta, 64)
    want, tol = model64.forward(tm, ids, tables)
    held = np.isfinite(tol).all(-1)
    assert held.mean() > 0.5 and np.median(tol[held]) < (5e-3 if experts else 1e-3)
    cache, at = tm.new_cache(64), 0
    for k in (25, 1, 1, 8, 1, 4, *[1] * 20):
        at += k
        got = tm.forward_kv(ids[at - k:at], at - k, cache)
        assert not held[at - 1] or (np.abs(got - want[at - 1]) <= tol[at - 1]).all()
    # the bound tells other tokens, a lost position and a shifted one from what is right
    last = int(np.flatnonzero(held)[-1])
    shifted = [np.concatenate([a[:30], a[31:]]) for a in tables]
    for x in (model64.forward(tm, np.roll(ids, 1), tables)[0][last], model64.forward(tm, ids[1:last + 1], tables)[0][-1],
              model64.forward(tm, ids, shifted)[0][last]):
        assert (np.abs(x - want[last]) > 2 * tol[last]).mean() > 0.5
