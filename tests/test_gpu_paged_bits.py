"""How many bits of a query and of a weight attention over pages keeps, whichever call reads them: moe_paged_attn_dev and
moe_paged_attn_shared_dev, whose results are to be as close.

Scores here are exact in fp32: a key is 256 or 64 times a unit vector, so a score is one of its query's values times a power
of two, and scale * log2(e) rounds to 1.  What is left to go wrong is what a kernel makes of a query's 24 bits and of a weight's.
Bound, against sum p |v| / sum p: the hardware's exp2 2 U, of a part's weight and of its join; the sums over n positions
n + 32 half steps each for the numerator and the denominator; 8 U more for the rounding of the scale, whose difference from
ln 2 acts on scores' differences of at most 60."""
import ctypes

import numpy as np
import pytest

import paged_cases as C
from test_gpu_paged_shared import Batch

pytestmark = pytest.mark.gpu

U = C.U
SCALE = next(s for s in (np.nextafter(np.float32(np.log(2)), np.float32(d)) if d else np.float32(np.log(2)) for d in (None, 0, 1))
             if np.float32(s * np.float32(1.44269504088896340736)) == np.float32(1))


class Exact(Batch):
    """Every position's key is `size` times the unit vector of a dimension of its own, its value one of that dimension's."""

    def __init__(self, M, kind, groups, nq, nkv, hd, wide, size, seed):
        self.dim_of, self.size = np.random.default_rng(seed + 1), size
        self.values = self.dim_of.standard_normal((nkv, hd, hd)).astype(np.float32)
        super().__init__(M, kind, groups, nq, nkv, hd, 16, "head", seed=seed, wide=wide)
        if kind == "e4m3":   # (scales of 1)
            self.pool.pages.k_scale = self.pool.pages.v_scale = None
            self.pool.scales = [None, None]
        self.scale = float(SCALE)

    def put(self, page, off, d, v):
        k = np.zeros((self.nkv, self.hd), np.float32)
        k[np.arange(self.nkv), d] = self.size
        self.pool.put(page, off, k, v)

    def fill(self, page, n):
        had, self.pool.scales = self.pool.scales, [None, None]
        for off in range(n):
            d = self.dim_of.integers(1, self.hd, self.nkv)
            self.put(page, off, d, self.values[np.arange(self.nkv), d])
        self.pool.scales = had

    def bound(self, floor):
        """floor: what each weight may be off by besides, relative to its row's largest one"""
        out = self.b["out"].download((self.T, self.ldo), np.float32)[:, :self.nq * self.hd].reshape(self.T, self.nq, self.hd)
        worst = 0.0
        for t in range(self.T):
            k, v = self.pool.rows(self.tables[self.req[t]], int(self.pos[t]) + 1)
            g, n = self.nq // self.nkv, k.shape[0]
            for h in range(self.nq):
                s = self.scale * (k[:, h // g] @ self.q[t, h].astype(np.float64))
                p = np.exp(s - s.max())
                w, a = v[:, h // g], np.abs(v[:, h // g])
                tol = ((2 * (n + 32) + 16) * U * (p @ a) + floor * a.sum(0)) / p.sum() + 1e-30
                worst = max(worst, float(np.max(np.abs(out[t, h] - p @ w / p.sum()) / tol)))
        return worst

    def both(self, floor):
        M, L = self.M, self.M.lib()
        self.upload()
        self.calls()
        shared = self.bound(floor)
        need = L.moe_paged_attn_work_bytes(self.T, self.nq, self.nkv, self.hd)
        work = M.DeviceBuffer(need)
        a = M.PagedAttn(*[getattr(self.attn, f) for f, _ in M.PagedAttn._fields_])
        a.work, a.work_bytes = work.ptr, need
        M.check(L.moe_paged_attn_dev(ctypes.byref(a), ctypes.byref(self.pool.pages)))
        apart = self.bound(floor)
        assert shared <= 1 and apart <= 1, f"times the bound: shared {shared:.3g}, apart {apart:.3g}"


SHAPES = [([(4, 208, (1, 40)), (1, 0, (150, 150))], 8, 2, 64, False), ([(4, 208, (1, 40)), (3, 160, (20, 20))], 16, 1, 128, True), ([(10, 208, (1, 40))], 8, 1, 64, True),
          ([(3, 192, (0, 30))], 16, 1, 256, True), ([(9, 192, (0, 30))], 16, 2, 80, True)]


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_queries(moehip, kind, shape):
    """Scores near 179000 that differ by a few: two parts of 11 bits of a query move one by up to 2^-6, a weight by 1 %."""
    groups, nq, nkv, hd, wide = SHAPES[shape]
    print("bits of queries", kind, shape, flush=True)
    b = Exact(moehip, kind, groups, nq, nkv, hd, wide, 256.0, 40 + shape)
    b.q = (700.2 + 0.008 * b.rng.random(b.q.shape)).astype(np.float32)
    b.q.view(np.uint32)[...] |= 1   # 700, 0.2 to 11 bits and a last bit more
    b.both(0.0)


@pytest.mark.parametrize("kind,below", [(k, 22) for k in C.TYPES] + [(k, 60) for k in ("f32", "bf16", "e4m3")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_weights(moehip, kind, below, shape):
    """A first position that takes nearly all of the weight and whose value is zero: what is left is weights of 2^-below and
    less.  fp16 parts hold a weight to 2^-38 of the row's largest one."""
    groups, nq, nkv, hd, wide = SHAPES[shape]
    print("bits of weights", kind, below, shape, flush=True)
    b = Exact(moehip, kind, groups, nq, nkv, hd, wide, 64.0, 60 + shape)
    for t in range(b.T):
        b.put(int(b.tables[b.req[t], 0]), 0, 0, np.zeros((nkv, hd), np.float32))
    b.q = (700 - (below + b.rng.random(b.q.shape)) / 64).astype(np.float32)
    b.q[:, :, 0] = 700
    b.both(2.0 ** -38 if kind == "f16" else 0.0)
