"""moe_paged_heads_dev against a 64-bit evaluation (bound: paged_cases.turn_head, and half a step of the cache's type)."""
import numpy as np
import pytest

import paged_cases as C

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _run(M, pool, qkv, nq, pos, slot, qn, kn, cos, sin, rope_dim, q_out=None, ldq=None):
    T, ld = qkv.shape
    b = {n: M.DeviceBuffer.from_array(x) for n, x in dict(qkv=qkv, pos=np.asarray(pos, np.int32), slot=np.asarray(slot, np.int32)).items()}
    opt = [None if x is None else M.DeviceBuffer.from_array(x) for x in (qn, kn, cos, sin)]
    ptr = [None if x is None else x.ptr for x in opt]
    ob = b["qkv"] if q_out is None else M.DeviceBuffer.from_array(q_out)
    h = M.PagedHeads(b["qkv"].ptr, ld, T, nq, b["pos"].ptr, b["slot"].ptr, ptr[0], ptr[1], EPS, ptr[2], ptr[3], 0 if cos is None else len(cos),
                     rope_dim, ob.ptr, ld if q_out is None else ldq)
    pool.upload()
    M.check(M.lib().moe_paged_heads_dev(C.ref(h), C.ref(pool.pages)), "paged_heads")
    before = pool.raw.copy()
    pool.download()
    shape = qkv.shape if q_out is None else q_out.shape
    return ob.download(shape, np.float32), before


def _check_pages(pool, before, slot, kd, kt, vd):
    """Written slots within the bounds, every other byte as it was."""
    ps = pool.ps
    raw = pool.raw.copy()
    for t, s in enumerate(slot):
        if not 0 <= s < pool.n_pages * ps:
            continue
        for side, (view, x, tol) in enumerate(((pool.k, kd[t], kt[t]), (pool.v, vd[t], 0.0))):
            f = pool.factor(side)
            x, tol = x / f, tol / f + np.abs(x / f) * (2 * C.U if pool.scales[side] is not None else 0)
            got = C.decode(np.ascontiguousarray(view[s // ps, s % ps]), pool.dtype)
            if pool.dtype == C.E4M3:
                x = np.clip(x, -448, 448)
            lim = tol * (1 + C.HALF[pool.dtype]) + np.maximum(np.abs(x) * C.HALF[pool.dtype], C.TINY[pool.dtype])
            if pool.dtype == C.F32:
                lim = tol + 1e-38
            assert (np.abs(got - x) <= lim).all(), f"row {t}, {'kv'[side]}: {np.max(np.abs(got - x) / lim):.2f} times the bound"
    # put the old bytes back into the written slots: the rest must be untouched
    now, pool.raw[...] = raw, before
    old = [(pool.k[s // ps, s % ps].copy(), pool.v[s // ps, s % ps].copy()) for s in slot if 0 <= s < pool.n_pages * ps]
    pool.raw[...] = now
    for (k, v), s in zip(old, [s for s in slot if 0 <= s < pool.n_pages * ps]):
        pool.k[s // ps, s % ps], pool.v[s // ps, s % ps] = k, v
    np.testing.assert_array_equal(pool.raw.view(np.uint8), before.view(np.uint8))


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("T,nq,nkv,hd,ps,order,rope_dim,norm,extra", [
    (1, 32, 4, 128, 16, "slot", 128, "qk", 0), (33, 8, 8, 64, 32, "head", 64, "qk", 0), (7, 6, 2, 80, 24, "shared", 80, "qk", 3),
    (50, 16, 1, 256, 64, "slot", 256, "qk", 4), (5, 3, 3, 16, 1, "head", 16, "q", 0), (9, 4, 2, 96, 16, "slot", 32, "qk", 0),
    (9, 4, 2, 96, 16, "slot", 38, "k", 1), (4, 2, 1, 128, 8, "shared", 0, "qk", 0), (12, 4, 4, 48, 16, "slot", 48, "", 0),
    (400, 32, 4, 128, 16, "slot", 128, "qk", 0), (3, 2, 2, 64, 16, "slot", 62, "qk", 0)])
def test_shapes(moehip, kind, T, nq, nkv, hd, ps, order, rope_dim, norm, extra):
    print("paged heads", kind, T, nq, nkv, hd, ps, order, rope_dim, norm, flush=True)
    dtype = C.TYPES[kind]
    rng = np.random.default_rng(T + hd + rope_dim)
    scales = [0.01 + 0.02 * rng.random(nkv) for _ in "kv"] if kind == "e4m3" else [None, None]
    pool = C.Pool(moehip, dtype, -(-2 * T // ps) + 2, ps, nkv, hd, order, *scales)
    H = nq + 2 * nkv
    qkv = rng.standard_normal((T, H * hd + extra)).astype(np.float32) * 3
    pos = rng.integers(0, 200, T)
    slot = rng.permutation(pool.n_pages * ps)[:T].astype(np.int32)
    if T > 4:
        slot[T // 2] = -1
    qn, kn = (rng.uniform(0.5, 1.5, hd).astype(np.float32) if c in norm else None for c in "qk")
    cos, sin = C.rope_tables(200, rope_dim) if rope_dim else (None, None)
    old = rng.standard_normal((T, nq * hd + extra)).astype(np.float32)
    got, before = _run(moehip, pool, qkv, nq, pos, slot, qn, kn, cos, sin, rope_dim, old, nq * hd + extra)
    x = qkv[:, :H * hd].reshape(T, H, hd).astype(np.float64)
    cs = [None, None] if not rope_dim else [a[pos][:, None].astype(np.float64) for a in (cos, sin)]
    qd, qt = C.turn_head(x[:, :nq], None if qn is None else qn.astype(np.float64), EPS, *cs, rope_dim)
    kd, kt = C.turn_head(x[:, nq:nq + nkv], None if kn is None else kn.astype(np.float64), EPS, *cs, rope_dim)
    for t in range(T):
        if slot[t] < 0:
            np.testing.assert_array_equal(got[t], old[t])
            continue
        g = got[t, :nq * hd].reshape(nq, hd)
        assert (np.abs(g - qd[t]) <= qt[t] + 1e-38).all(), f"row {t}"
        np.testing.assert_array_equal(got[t, nq * hd:], old[t, nq * hd:])
    _check_pages(pool, before, slot.tolist(), kd, kt, x[:, nq + nkv:])


def test_in_place_and_unaligned(moehip):
    """Queries back into qkv; rows an odd number of floats apart."""
    M = moehip
    rng = np.random.default_rng(3)
    T, nq, nkv, hd = 6, 4, 2, 64
    for extra in (0, 1):
        pool = C.Pool(M, C.F32, 4, 16, nkv, hd)
        qkv = rng.standard_normal((T, (nq + 2 * nkv) * hd + extra)).astype(np.float32)
        pos, slot = np.arange(T), np.array([3, 40, -1, 17, 63, 0], np.int32)
        qn, kn = np.ones(hd, np.float32), np.ones(hd, np.float32)
        cos, sin = C.rope_tables(T, hd)
        got, before = _run(M, pool, qkv, nq, pos, slot, qn, kn, cos, sin, hd)
        x = qkv[:, :(nq + 2 * nkv) * hd].reshape(T, -1, hd).astype(np.float64)
        cs = [a[pos][:, None].astype(np.float64) for a in (cos, sin)]
        qd, qt = C.turn_head(x[:, :nq], 1.0, EPS, *cs, hd)
        kd, kt = C.turn_head(x[:, nq:nq + nkv], 1.0, EPS, *cs, hd)
        for t in range(T):
            if slot[t] < 0:
                np.testing.assert_array_equal(got[t], qkv[t])
                continue
            assert (np.abs(got[t, :nq * hd].reshape(nq, hd) - qd[t]) <= qt[t]).all()
            np.testing.assert_array_equal(got[t, nq * hd:], qkv[t, nq * hd:])   # keys and values stay in qkv
        _check_pages(pool, before, slot.tolist(), kd, kt, x[:, nq + nkv:])


@pytest.mark.parametrize("kind", list(C.TYPES))
def test_bad_places(moehip, kind):
    """Slots past the cache and positions past the rotation's tables: NaN queries, nothing outside written."""
    M, dtype = moehip, C.TYPES[kind]
    rng = np.random.default_rng(4)
    T, nq, nkv, hd, ps = 7, 4, 2, 64, 16
    pool = C.Pool(M, dtype, 4, ps, nkv, hd)
    qkv = rng.standard_normal((T, (nq + 2 * nkv) * hd)).astype(np.float32)
    slot = np.array([0, 64, 2 ** 31 - 1, -2 ** 31, 5, 6, 63], np.int32)
    pos = np.array([0, 1, 2, 3, 50, -1, 49], np.int32)
    cos, sin = C.rope_tables(50, hd)
    old = np.full((T, nq * hd), 7, np.float32)
    got, before = _run(M, pool, qkv, nq, pos, slot, None, None, cos, sin, hd, old, nq * hd)
    assert np.isnan(got[[1, 2, 4, 5]]).all() and (got[3] == 7).all() and np.isfinite(got[[0, 6]]).all()
    for s in (5, 6):   # the slot is right, the position is not: the key is NaN, the value is there
        assert np.isnan(C.decode(np.ascontiguousarray(pool.k[0, s]), dtype)).all()
        assert np.isfinite(C.decode(np.ascontiguousarray(pool.v[0, s]), dtype)).all()
    x = qkv.reshape(T, -1, hd).astype(np.float64)
    cs = [a[np.clip(pos, 0, 49)][:, None].astype(np.float64) for a in (cos, sin)]
    kd, kt = C.turn_head(x[:, nq:nq + nkv], None, EPS, *cs, hd)
    keep = pool.raw.copy()
    for s in (5, 6):
        pool.k[0, s], pool.v[0, s] = before.reshape(2, 4, ps, nkv, hd)[:, 0, s]
    _check_pages(pool, before, [0, -1, -1, -1, -1, -1, 63], kd, kt, x[:, nq + nkv:])
    assert keep.shape == pool.raw.shape


def test_values_at_the_types_edges(moehip):
    """Values through every type: saturation at 448, ties to even, subnormals, infinities, NaN."""
    M = moehip
    vals = np.array([0.0, -0.0, 448, 449, 464, 1e9, -1e9, np.inf, -np.inf, np.nan, 17, 18, 19, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 2 ** -11, -2 ** -7,
                     65504, 65519, 65520, 1 + 2 ** -8, 1 + 3 * 2 ** -8, 1 + 2 ** -11, 1 + 3 * 2 ** -11, 6e-8, 3e-8, 2.9e-8, 3.4e38, 1e-40, 240, 0.3],
                    np.float32)
    hd = 32
    for kind, dtype in C.TYPES.items():
        pool = C.Pool(M, dtype, 1, 16, 1, hd)
        qkv = np.zeros((1, 3 * hd), np.float32)
        qkv[0, 2 * hd:] = vals
        _run(M, pool, qkv, 1, [0], [4], None, None, None, None, 0, np.zeros((1, hd), np.float32), hd)
        got = C.decode(np.ascontiguousarray(pool.v[0, 4, 0]), dtype)
        with np.errstate(all="ignore"):
            want = C.decode(C.encode(np.nan_to_num(vals, nan=0.0) if dtype in (C.E4M3, C.BF16) else vals, dtype), dtype)
        want[np.isnan(vals)] = np.nan
        np.testing.assert_array_equal(got, want, err_msg=kind)
