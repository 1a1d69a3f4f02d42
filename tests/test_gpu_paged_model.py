"""moe_model_step_paged and moe_model_forward over prompts and decode steps, each against the 64-bit model and its bound
(model64.py): every request at positions of its own, in steps with somewhat more rows than requests."""
import numpy as np
import pytest

import model64
import oracle as O
import paged_cases as C

pytestmark = pytest.mark.gpu

MODELS = [(False, 11, 4, 2, False), (False, 12, 4, 2, True), (False, 13, 16, 2, False), (True, 14, 4, 2, False), (True, 15, 4, 2, True)]


def _within(got, want, tol, where):
    """-> whether the bound says anything here"""
    if not np.isfinite(tol).all():
        return 0
    assert (np.abs(got - want) <= tol).all(), f"{where}: {np.max(np.abs(got - want) / tol):.2f} times the bound"
    return 1


@pytest.mark.parametrize("experts,seed,nq,nkv,bias", MODELS)
def test_forward(moehip, experts, seed, nq, nkv, bias):
    tm = model64.plain_model(O, seed, 1, experts, nq=nq, nkv=nkv, bias=bias)
    ids = np.random.default_rng(seed).integers(0, tm.V, 130)
    want, tol = model64.forward(tm, ids, O.rope_tables(tm.hd, tm.theta, 256))
    m, at, told = moehip.model_from_tiny(tm, 256), 0, 0
    for k in (100, 1, 1, 7, *[1] * 21):
        at += k
        got, _ = m.forward(ids[at - k:at])
        told += _within(got, want[at - 1], tol[at - 1], f"position {at - 1}")
    assert told >= 12
    m.close()


@pytest.mark.parametrize("kind,experts,seed,nq,nkv,bias", [("f32", *x) for x in MODELS] + [("f16", *x) for x in MODELS if not x[0]])
@pytest.mark.parametrize("n,rows,ps", [(16, 17, 16), (10, 13, 8), (30, 33, 32)])
def test_steps(moehip, kind, experts, seed, nq, nkv, bias, n, rows, ps):
    """Prompts of about 100 tokens, decode steps padded to `rows`, one with a few tokens of a request, one that ends."""
    print("paged model", kind, experts, nq, nkv, n, rows, ps, flush=True)
    M, dtype = moehip, C.TYPES[kind]
    tm = model64.plain_model(O, seed, 1, experts, nq=nq, nkv=nkv, bias=bias)
    m = M.model_from_tiny(tm, 256)
    rng = np.random.default_rng(100 + seed)
    ids = [rng.integers(0, tm.V, 120) for _ in range(n)]
    stored = (0.0, 0.0) if dtype == C.F32 else (C.HALF[dtype], C.TINY[dtype])
    wants = [model64.forward(tm, i, O.rope_tables(tm.hd, tm.theta, 256), stored) for i in ids]
    c = M.PagedCache(1, nkv, tm.hd, n * (256 // ps), ps, n, 256 // ps, 110 * n, dtype)
    held, told, seen = np.zeros(n, int), 0, 0

    def step(fresh):
        nonlocal told, seen
        new = [ids[r][held[r]:held[r] + k] for r, k in enumerate(fresh) if k > 0]
        lg, nx = m.step_paged(c, fresh, np.concatenate(new))
        assert c.status == 0
        for r, k in enumerate(fresh):
            held[r] = held[r] + k if k >= 0 else 0
            if k <= 0:
                assert nx[r] == -1 and not lg[r].any()
                continue
            assert np.isfinite(lg[r]).all() and nx[r] == O.greedy(lg[r])
            want, tol = wants[r]
            told += _within(lg[r], want[held[r] - 1], tol[held[r] - 1], f"request {r} at position {held[r] - 1}")
            seen += 1
        np.testing.assert_array_equal(c.array("held", n), held)

    step(rng.integers(90, 108, n))
    c.plan.max_tokens = c.max_tokens = rows   # steps of a fixed size from here on
    ones = np.ones(n, int)
    for i in range(3):
        step(ones)
    some = ones.copy()
    some[n // 2] += rows - n
    step(some)
    some = ones.copy()
    some[[0, n // 3]] = 0, -1
    step(some)
    some[n // 3] = 2
    step(some)
    step(ones)
    assert told > seen // 2
    m.close()
