"""Batches with somewhat more rows than requests: a decode step of a fixed size that is not full, or one with a short
prompt in it, over tables of a few hundred positions.  Each row against a 64-bit evaluation (paged_cases.attend)."""
import numpy as np
import pytest

import test_gpu_paged_attn as A
import paged_cases as C

pytestmark = pytest.mark.gpu


def _widen(b, positions):
    """tables of `positions` positions"""
    width = positions // b.ps
    tables = np.full((len(b.lens), width), -7, np.int32)
    tables[:, :min(width, b.width)] = b.tables[:, :width]
    b.tables, b.width = tables, width


def _check(b, req, pos):
    T = len(req)
    out, q = b.run(req=req, pos=pos, T=T)
    for fill in (0, 0x3C):   # whatever `work` held
        again, _ = b.run(req=req, pos=pos, T=T, q=q.reshape(T, -1), work_from=fill)
        np.testing.assert_array_equal(out.view(np.uint32), again.view(np.uint32))
    for t in range(T):
        if req[t] < 0:
            assert (out[t] == 7).all(), f"row {t} of no request was written"
        else:
            b.check(out, q, t, int(req[t]), int(pos[t]) + 1)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("n,T,length,positions,nq,nkv,hd,ps", [
    (16, 17, 100, 256, 32, 4, 128, 16), (32, 40, 60, 256, 32, 4, 128, 16), (16, 18, 700, 768, 32, 4, 128, 24), (10, 11, 500, 512, 32, 4, 128, 16),
    (16, 18, 512, 512, 32, 4, 128, 32), (16, 17, 2048, 2048, 8, 1, 64, 16), (60, 63, 250, 256, 8, 8, 64, 16), (5, 6, 1, 256, 4, 2, 16, 8),
    (40, 44, 300, 384, 6, 2, 256, 16)])
def test_padded_decode(moehip, kind, n, T, length, positions, nq, nkv, hd, ps):
    print("paged attention padded", kind, n, T, length, positions, nq, nkv, hd, flush=True)
    b = A.Batch(moehip, C.TYPES[kind], [length] * n, nq, nkv, hd, ps, "head", seed=n + T)
    _widen(b, positions)
    _check(b, [*range(n)] + [-1] * (T - n), [length - 1] * n + [-1] * (T - n))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [(1, 2, 1), (1, 1, 3, 1, 1, 1), (2, 1, 1, 1, 1, 1, 1, 1), (1,) * 20 + (5,) + (1,) * 9])
def test_short_prompt_beside_decode(moehip, kind, tokens):
    """A request's rows on both sides of a border between groups of shared columns."""
    n = len(tokens)
    print("paged attention short prompt", kind, tokens, flush=True)
    b = A.Batch(moehip, C.TYPES[kind], [250 - r for r in range(n)], 32, 4, 128, 16, seed=n)
    _widen(b, 256)
    req = [r for r, k in enumerate(tokens) for _ in range(k)]
    pos = [b.lens[r] - k + i for r, k in enumerate(tokens) for i in range(k)]
    _check(b, req, pos)


@pytest.mark.parametrize("seed", range(32))
def test_drawn(moehip, seed):
    """Batches of any make: rows of one request in stretches or apart, lengths to the table's end, rows of no request."""
    rng = np.random.default_rng(900 + seed)
    kind = list(C.TYPES)[seed % 4]
    nq, nkv, hd = [(8, 1, 64), (4, 4, 32), (32, 4, 128), (6, 2, 80), (10, 2, 48), (3, 1, 256), (9, 3, 64), (24, 2, 64)][rng.integers(8)]
    ps, n = int(rng.choice([1, 7, 16, 24, 64])), int(rng.integers(1, 40))
    positions = max(1, int(rng.integers(20, 1500)) // ps) * ps
    lens = [positions if rng.random() < 0.5 else int(rng.integers(0, positions + 1)) for _ in range(n)]
    req, pos = [], []
    T = n + int(rng.integers(0, 30))
    while len(req) < T:
        r = int(rng.integers(-1, n))
        k = int(rng.integers(1, 12)) if rng.random() < 0.4 else 1
        at = int(rng.integers(-1, lens[r])) if r >= 0 and lens[r] and rng.random() < 0.5 else (lens[r] if r >= 0 else 0) - 1
        req += [r] * k
        pos += [max(at - i, -1) for i in range(k)][::-1]
    print("paged attention drawn", seed, kind, nq, nkv, hd, ps, n, positions, T, flush=True)
    b = A.Batch(moehip, C.TYPES[kind], lens, nq, nkv, hd, ps, ["slot", "head"][seed % 2], seed=seed)
    _widen(b, positions)
    _check(b, req[:T], pos[:T])
