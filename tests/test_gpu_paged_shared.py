"""moe_paged_share_dev against a simulation (whole numbers), and moe_paged_attn_shared_dev against attention in 64 bits on
what the pages hold, by the bound that moe_paged_attn_dev's tests use (paged_cases.attend)."""
import ctypes

import numpy as np
import pytest

import beam_cases as B
import paged_cases as C

pytestmark = pytest.mark.gpu


class Batch:
    """Rows in groups whose requests begin in the same pages.

    groups: [(rows, shared positions, (fewest, most) of a row's own)]; the rest of the pool holds NaNs and infinities.
    wide: tables of 32768 positions, whose shared items are not taken in sixteen columns only for being few."""

    def __init__(self, M, kind, groups, nq, nkv, hd, ps, order="slot", seed=0, listed=True, spare_rows=0, first=None, wide=False):
        self.M, self.nq, self.nkv, self.hd, self.ps = M, nq, nkv, hd, ps
        self.rng = rng = np.random.default_rng(seed)
        self.T = T = sum(g[0] for g in groups)
        plan, pages = [], 0
        for rows, shared, (lo, hi) in groups:
            plan.append((rows, shared // ps, [int(rng.integers(lo, hi + 1)) for _ in range(rows)]))
            pages += shared // ps + sum(-(-m // ps) for m in plan[-1][2])
        width = max(1, max(s + max(-(-m // ps) for m in mine) for _, s, mine in plan)) + 1
        if wide:
            width = max(width, 32768 // ps)
        self.n_pages = pages + 2
        order_of = iter(rng.permutation(self.n_pages).tolist())
        dtype = C.TYPES[kind]
        scales = [0.01 + 0.01 * rng.random(nkv) for _ in "kv"] if kind == "e4m3" else [None, None]
        self.pool = C.Pool(M, dtype, self.n_pages, ps, nkv, hd, order, *scales)
        self.n_req = T + spare_rows
        self.tables = rng.integers(-2, self.n_pages + 2, (self.n_req, width)).astype(np.int32)
        self.pos = np.empty(T, np.int32)
        where = rng.permutation(self.n_req)[:T] if listed else np.arange(T)   # rows' requests in no order
        self.req = where.astype(np.int32)
        t = 0
        for rows, shared, mine in plan:
            common = [next(order_of) for _ in range(shared)]
            for p in common:
                self.fill(p, ps)
            for m in mine:
                own = [next(order_of) for _ in range(-(-m // ps))]
                for i, p in enumerate(own):
                    self.fill(p, min(ps, m - i * ps))
                self.tables[where[t], :shared + len(own)] = common + own
                self.pos[t] = shared * ps + m - 1
                t += 1
        self.first = np.cumsum([0] + [g[0] for g in groups]).astype(np.int32) if first is None else np.asarray(first, np.int32)
        self.q = rng.standard_normal((T, nq, hd)).astype(np.float32)
        self.old = rng.standard_normal((T, nq * hd)).astype(np.float32)
        self.scale = float(np.float32(1 / np.sqrt(hd)))
        self.listed = listed

    def fill(self, page, n):
        f = [1.0 if s is None else 30 * s[:, None] for s in self.pool.scales]
        for off in range(n):
            self.pool.put(page, off, *[(self.rng.standard_normal((self.nkv, self.hd)) * x).astype(np.float32) for x in f])

    def upload(self, ldq=None, ldo=None):
        M, L = self.M, self.M.lib()
        self.pool.upload()
        buf = M.DeviceBuffer.from_array
        n = self.nq * self.hd
        self.ldq, self.ldo = ldq or n, ldo or n
        q = np.full((self.T, self.ldq), np.nan, np.float32)
        q[:, :n] = self.q.reshape(self.T, n)
        out = np.full((self.T, self.ldo), 3.5, np.float32)
        out[:, :n] = self.old
        self.b = {"q": buf(q), "req": buf(self.req), "pos": buf(self.pos), "tables": buf(self.tables), "first": buf(self.first), "out": buf(out),
                  "prefix": buf(np.full(max(1, len(self.first) - 1), -9, np.int32))}
        sizes = (self.T, len(self.first) - 1, self.nq, self.nkv, self.hd)
        plan, work = L.moe_paged_share_plan_bytes(*sizes), L.moe_paged_attn_shared_work_bytes(*sizes)
        assert plan and work
        self.b["plan"], self.b["work"] = (buf(np.full(x, 0xA5, np.uint8)) for x in (plan, work))
        p = {x: b.ptr for x, b in self.b.items()}
        req = p["req"] if self.listed else None
        self.share = M.PagedShare(self.T, self.n_req, self.tables.shape[1], self.ps, self.nq, self.nkv, self.hd, req, p["pos"], p["tables"], len(self.first) - 1, p["first"],
                                  p["prefix"], p["plan"], plan)
        self.attn = M.PagedAttn(p["q"], self.ldq, self.T, self.nq, req, p["pos"], p["tables"], self.n_req, self.tables.shape[1], self.scale, p["out"], self.ldo, p["work"], work)

    def calls(self, times=1):
        M, L = self.M, self.M.lib()
        M.check(L.moe_paged_share_dev(ctypes.byref(self.share)), "share")
        for _ in range(times):
            M.check(L.moe_paged_attn_shared_dev(ctypes.byref(self.attn), ctypes.byref(self.pool.pages), ctypes.byref(self.share)), "attn")

    def check(self, nan_rows=()):
        want = B.share(self.req if self.listed else None, self.pos, self.tables, self.first, self.ps)
        if want.size:
            np.testing.assert_array_equal(self.b["prefix"].download(want.shape, np.int32), want)
        out = self.b["out"].download((self.T, self.ldo), np.float32)
        n = self.nq * self.hd
        assert (out[:, n:] == 3.5).all()
        worst = 0.0
        for t in range(self.T):
            got = out[t, :n].reshape(self.nq, self.hd)
            r = int(self.req[t])
            if r < 0:
                np.testing.assert_array_equal(got.reshape(-1), self.old[t])
                continue
            if t in nan_rows:
                assert np.isnan(got).all(), f"row {t}"
                continue
            k, v = self.pool.rows(self.tables[r], int(self.pos[t]) + 1)
            ref, tol = C.attend(self.q[t].astype(np.float64), k, v, self.scale)
            err = np.abs(got - ref)
            assert (err <= tol).all(), f"row {t}: {np.max(err / tol):.2f} times the bound"
            worst = max(worst, float(np.max(err / tol)) if int(self.pos[t]) >= 0 else 0.0)
        return want, worst

    def run(self, **kw):
        self.upload(**kw)
        self.calls()
        return self.check()


GROUPS = [
    [(1, 0, (1, 1))],
    [(2, 16, (1, 3))],
    [(4, 130, (0, 40))],
    [(1, 200, (1, 50)), (5, 64, (1, 100)), (3, 0, (1, 30))],
    [(8, 700, (1, 60)), (8, 300, (1, 60)), (2, 1000, (1, 1))],
    [(33, 260, (0, 33))],
    [(6, 144, (0, 20)), (40, 128, (0, 40)), (1, 300, (1, 9)), (7, 145, (100, 150))],
]


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("nq,nkv,hd,ps,order", [(8, 2, 64, 16, "slot"), (32, 4, 128, 16, "head"), (15, 3, 80, 24, "slot"), (6, 6, 256, 7, "shared"), (40, 1, 16, 1, "head"), (4, 1, 192, 128, "head")])
@pytest.mark.parametrize("groups", range(len(GROUPS)))
@pytest.mark.parametrize("wide", [False, True])
def test_attention(moehip, kind, nq, nkv, hd, ps, order, groups, wide):
    print("shared attention", kind, nq, nkv, hd, ps, order, groups, wide, flush=True)
    b = Batch(moehip, kind, GROUPS[groups], nq, nkv, hd, ps, order, seed=hd + groups, listed=groups % 2 == 0, spare_rows=2 if groups % 2 == 0 else 0, wide=wide)
    b.run(ldq=nq * hd + 5 if groups == 2 else None, ldo=nq * hd + 3 if groups == 3 else None)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("nq,nkv,hd,groups", [(4, 1, 64, [(6, 6000, (1, 300)), (2, 3000, (900, 1000))]), (8, 2, 80, [(17, 4500, (0, 140))]), (2, 1, 256, [(33, 2700, (1, 600))]),
                                              (8, 8, 128, [(1, 9000, (5, 6))]), (32, 2, 16, [(3, 12000, (1, 2000))])])
@pytest.mark.parametrize("wide", [False, True])
def test_many_parts(moehip, kind, nq, nkv, hd, groups, wide):
    """Prefixes and rows of their own long enough that a head's sums come in tens of parts, up to more than a wave's lanes."""
    print("shared attention, many parts", kind, nq, nkv, hd, groups, wide, flush=True)
    Batch(moehip, kind, groups, nq, nkv, hd, 16, "head", seed=hd + 1, wide=wide).run()


def test_rows_of_no_request_and_empty_ones(moehip):
    """In a group, at its start, and a whole group of them; rows outside every group."""
    b = Batch(moehip, "bf16", [(6, 192, (1, 40)), (3, 160, (1, 20)), (4, 48, (2, 9))], 8, 2, 64, 16, seed=2, first=[1, 6, 9, 12])
    b.req[[1, 4, 6, 7, 8]] = -1
    b.pos[[2, 10]] = -1
    want, _ = b.run()
    assert want[0] == 192 and want[1] == 0 and want[2] >= 48
    b.pos[:] = -1
    b.run()
    b.req[:] = -5
    b.run()


@pytest.mark.parametrize("wide", [False, True])
def test_outside_and_bad_pages(moehip, wide):
    """A request or position outside the tables, a page that is none: NaN in the rows that attend it, none else."""
    b = Batch(moehip, "f16", [(6, 160, (1, 40)), (5, 80, (20, 20))], 24, 2, 64, 16, seed=3, spare_rows=1, wide=wide)
    b.req[1], b.pos[3] = b.n_req, b.tables.shape[1] * 16
    b.tables[b.req[8], 5] = b.n_pages      # a page of its own
    b.upload()
    b.calls()
    b.check(nan_rows=(1, 3, 8))
    b = Batch(moehip, "f32", [(6, 160, (1, 40)), (5, 80, (1, 40))], 24, 2, 64, 16, seed=4, wide=wide)
    for t in range(6):
        b.tables[b.req[t], 4] = -1         # a page that the group shares
    b.upload()
    b.calls()
    b.check(nan_rows=range(6))


@pytest.mark.parametrize("first", [[0, 4, 2, 9], [0, 10], [-1, 9], [9, 9, 9], [0, 0, 9, 9], [3, 3]], ids=str)
@pytest.mark.parametrize("wide", [False, True])
def test_firsts(moehip, first, wide):
    """Empty groups, groups that are none: every row has its attention all the same."""
    Batch(moehip, "bf16", [(9, 192, (1, 20))], 4, 2, 64, 16, seed=5, first=first).run()
    Batch(moehip, "bf16", [(9, 192, (1, 20))], 48, 2, 64, 16, seed=5, first=first, wide=wide).run()


def test_rows_of_one_request(moehip):
    """Several tokens of one request in a group (a prompt's end, tokens to be checked)."""
    b = Batch(moehip, "bf16", [(5, 0, (250, 250)), (4, 64, (30, 60))], 16, 2, 128, 16, seed=6, spare_rows=1)
    b.req[:5] = b.req[0]
    for pos, common in (([240, 241, 242, 243, 249], 240), ([140, 141, 142, 143, 149], 128)):
        b.pos[:5] = pos
        want, _ = b.run()
        assert want[0] == common


def test_as_the_unshared_call(moehip):
    """Against moe_paged_attn_dev on the same arguments: both within their bound of the same result."""
    M, L = moehip, moehip.lib()
    b = Batch(M, "f32", [(7, 300, (1, 90)), (3, 500, (1, 10))], 32, 4, 128, 16, "head", seed=7)
    b.run()
    need = L.moe_paged_attn_work_bytes(b.T, b.nq, b.nkv, b.hd)
    work = M.DeviceBuffer(need)
    b.attn.work, b.attn.work_bytes = work.ptr, need
    M.check(L.moe_paged_attn_dev(ctypes.byref(b.attn), ctypes.byref(b.pool.pages)))
    b.check()


def test_repeatable_and_graph(moehip):
    """The same bits every time; captured with its plan and replayed while the batch changes in device memory."""
    import test_gpu_paged_serving as G
    hip = G.Hip(moehip)
    groups = [(8, 400, (1, 60)), (3, 900, (1, 200)), (1, 50, (1, 5))]
    b = Batch(moehip, "bf16", groups, 32, 4, 128, 16, "head", seed=8)
    b.upload()
    graph = hip.capture(lambda: b.calls(2))
    for i in range(4):
        hip.launch(graph)
        moehip.synchronize()
        b.check()
        first = b.b["out"].download((b.T, b.ldo), np.float32)
        b.calls()
        np.testing.assert_array_equal(first, b.b["out"].download((b.T, b.ldo), np.float32))
        b.q = b.rng.standard_normal(b.q.shape).astype(np.float32)
        b.pos = np.maximum(b.pos - 37 * (i + 1), -1).astype(np.int32)
        b.b["q"].upload(b.q.reshape(b.T, -1))
        b.b["pos"].upload(b.pos)
    hip.destroy(graph)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0, 1e-6])
def test_scales(moehip, kind, scale):
    """Negative, no, sharp and flat scales."""
    b = Batch(moehip, kind, [(9, 256, (1, 70)), (2, 64, (1, 20))], 16, 2, 128, 16, "head", seed=12)
    b.scale = float(np.float32(scale))
    b.run()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_large_and_small_queries(moehip, kind):
    """Rows whose queries differ by many powers of two, in one product."""
    b = Batch(moehip, kind, [(8, 256, (1, 40))], 8, 1, 64, 16, seed=13)
    b.q *= (10.0 ** np.linspace(-30, 1, 8)).astype(np.float32)[:, None, None]
    b.q[3, 2] = 0
    b.run()


def test_no_rows_no_groups(moehip):
    M, L = moehip, moehip.lib()
    b = Batch(M, "f32", [(3, 32, (1, 5))], 4, 2, 64, 16, seed=9, first=[0])
    b.run()
    b.share.T = b.attn.T = 0
    M.check(L.moe_paged_share_dev(ctypes.byref(b.share)))
    M.check(L.moe_paged_attn_shared_dev(ctypes.byref(b.attn), ctypes.byref(b.pool.pages), ctypes.byref(b.share)))


def test_share_wide(moehip):
    """Long tables, many rows and groups of every size: the prefixes alone."""
    M, L = moehip, moehip.lib()
    rng = np.random.default_rng(10)
    sizes = [1, 2, 63, 64, 65, 300, 0, 500, 1]
    first = np.cumsum([3] + sizes).astype(np.int32)
    T, width, ps = int(first[-1]) + 4, 700, 8
    tables = rng.integers(0, 1 << 20, (T, width)).astype(np.int32)
    req = rng.permutation(T).astype(np.int32)
    pos = rng.integers(0, width * ps, T).astype(np.int32)
    for a, b in zip(first, first[1:]):
        if b > a:
            n = int(rng.integers(0, width))
            tables[req[a:b], :n] = tables[req[a], :n]
            pos[a:b] = rng.integers(max(0, n * ps - 600), width * ps, b - a)
    req[rng.integers(0, T, 30)] = -1
    pos[rng.integers(0, T, 30)] = -1
    buf = M.DeviceBuffer.from_array
    need = L.moe_paged_share_plan_bytes(T, len(sizes), 32, 4, 128)
    d = [buf(x) for x in (req, pos, tables, first, np.zeros(len(sizes), np.int32), np.full(need, 0xA5, np.uint8))]
    s = M.PagedShare(T, T, width, ps, 32, 4, 128, d[0].ptr, d[1].ptr, d[2].ptr, len(sizes), d[3].ptr, d[4].ptr, d[5].ptr, need)
    M.check(L.moe_paged_share_dev(ctypes.byref(s)))
    np.testing.assert_array_equal(d[4].download((len(sizes),), np.int32), B.share(req, pos, tables, first, ps))


@pytest.mark.parametrize("rows,groups", [(1500, 40), (1100, 1099), (400, 2000)])
def test_many_rows_and_groups(moehip, rows, groups):
    """More of either than the plan's block has threads."""
    rng = np.random.default_rng(rows)
    cuts = np.sort(rng.integers(0, rows + 1, groups - 1))
    first = np.concatenate([[0], cuts, [rows]]).astype(np.int32)
    sizes = [(int(b - a), 16 * int(rng.integers(0, 4)), (0, 20)) for a, b in zip(first, first[1:]) if b > a]
    Batch(moehip, "bf16", sizes, 2, 1, 64, 16, seed=14, first=first).run()
