"""moe_paged_fork_dev and moe_paged_copy_dev against simulations: whole numbers and bytes, so equal."""
import ctypes

import numpy as np
import pytest

import beam_cases as B
import paged_cases as C

pytestmark = pytest.mark.gpu


class Cache:
    """Requests over a ring of free pages, on the host and on the device."""

    def __init__(self, M, n_req, width, n_pages, page_size, max_copies=None, seed=0, in_place=True):
        self.M, self.n, self.width, self.n_pages, self.ps = M, n_req, width, n_pages, page_size
        self.copies = n_req if max_copies is None else max_copies
        self.rng = np.random.default_rng(seed)
        self.held = np.zeros(n_req, np.int32)
        self.tables = self.rng.integers(-5, n_pages + 5, (n_req, width)).astype(np.int32)   # what lies behind a request's pages
        self.ring = self.rng.permutation(n_pages).astype(np.int32)
        self.at = np.array([n_pages - 2 if n_pages > 2 else 0, n_pages], np.int32)
        buf = M.DeviceBuffer.from_array
        self.b = {n: buf(getattr(self, n)) for n in ("held", "tables", "ring")}
        self.b.update(ring_at=buf(self.at), parent=buf(np.zeros(n_req, np.int32)), copies=buf(np.full((self.copies, 3), 77, np.int32)), status=buf(np.full(1, 9, np.int32)))
        if in_place:
            self.b.update(held_out=self.b["held"], ring_at_out=self.b["ring_at"], tables_out=self.b["tables"])
        else:
            self.b.update(held_out=buf(self.held), ring_at_out=buf(self.at), tables_out=buf(self.tables + 1))
        need = M.lib().moe_paged_fork_work_bytes(n_req, width, n_pages)
        self.work = buf(np.full(need, 0xA5, np.uint8))
        self.args = M.PagedFork(n_req, width, n_pages, page_size, self.copies, *[self.b[n].ptr for n in (
            "parent", "held", "ring_at", "ring", "tables", "held_out", "ring_at_out", "tables_out", "copies", "status")], self.work.ptr, need)

    def grow(self, most):
        """New positions for every request, as a plan gives them."""
        for r in range(self.n):
            for _ in range(int(self.rng.integers(0, most + 1))):
                at = int(self.held[r])
                if at == self.width * self.ps or (at % self.ps == 0 and self.at[1] == 0):
                    break
                if at % self.ps == 0:
                    self.tables[r, at // self.ps] = self.ring[self.at[0]]
                    self.at[0], self.at[1] = (self.at[0] + 1) % self.n_pages, self.at[1] - 1
                self.held[r] += 1

    def upload(self, parent):
        for n, a in (("held", self.held), ("tables", self.tables), ("ring", self.ring), ("ring_at", self.at), ("parent", np.asarray(parent, np.int32))):
            self.b[n].upload(a)

    def check(self, parent):
        """What the call left against the simulation, which becomes the state."""
        want = B.fork(parent, self.held, self.tables, self.ring, self.at, self.ps, self.copies)
        shapes = {"tables": (self.n, self.width), "held": (self.n,), "ring": (self.n_pages,), "ring_at": (2,), "copies": (self.copies, 3), "status": (1,)}
        for n, shape in shapes.items():
            got = self.b[n + "_out" if n in ("tables", "held", "ring_at") else n].download(shape, np.int32)
            np.testing.assert_array_equal(got, np.reshape(want[n], shape), err_msg=n)
        if want["status"] == B.OK:
            self.tables, self.held, self.ring, self.at = want["tables"], want["held"], want["ring"], want["ring_at"].astype(np.int32)
            live = [int(p) for r in range(self.n) for p in self.tables[r, :-(-self.held[r] // self.ps)]]
            free = [int(self.ring[(self.at[0] + i) % self.n_pages]) for i in range(self.at[1])]
            assert len(set(free)) == len(free) and not set(free) & set(live) and len(set(free) | set(live)) == self.n_pages   # no page lost
        return want["status"]

    def step(self, parent):
        self.upload(parent)
        self.M.check(self.M.lib().moe_paged_fork_dev(ctypes.byref(self.args)), "fork")
        return self.check(parent)


def _parents(rng, n, group, ended):
    g = np.arange(n) // group * group
    p = g + np.minimum(rng.integers(0, group, n), rng.integers(0, group, n))
    p = np.where(p < n, p, np.arange(n))
    return np.where(rng.random(n) < ended, -1, p)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n,width,n_pages,ps,group", [(1, 3, 5, 4, 1), (8, 12, 60, 1, 8), (12, 30, 300, 7, 4), (64, 40, 1500, 16, 8), (300, 9, 2000, 3, 5), (1100, 20, 9000, 4, 16),
                                                      (4096, 5, 9000, 2, 64)])
def test_steps(moehip, n, width, n_pages, ps, group, in_place):
    """Requests that grow, fork, reorder and end, step after step."""
    print("paged fork", n, width, n_pages, ps, group, in_place, flush=True)
    c = Cache(moehip, n, width, n_pages, ps, seed=n + ps, in_place=in_place)
    done = 0
    for i in range(6 if n > 1000 else 12):
        c.grow(2 * ps)
        done += c.step(_parents(c.rng, n, group, 0.1 if i % 3 else 0.0)) == B.OK
    assert done >= 2   # (the largest run out of pages, as the simulation does)


def test_permutations(moehip):
    """Cycles and swaps in place: nothing is copied, nothing comes back."""
    c = Cache(moehip, 40, 25, 1200, 4, seed=3)
    for i in range(5):
        c.grow(20)
        assert c.step(c.rng.permutation(40)) == B.OK
        assert (c.b["copies"].download((40, 3), np.int32) == -1).all()


def test_all_end_and_all_from_one(moehip):
    c = Cache(moehip, 33, 10, 400, 5, seed=4)
    c.grow(30)
    assert c.step(np.full(33, 7)) == B.OK      # every other request is given up for copies of one
    c.grow(10)
    assert c.step(np.full(33, -1)) == B.OK and c.at[1] == 400
    assert c.step(np.arange(33)) == B.OK       # nothing held


def test_refused_states(moehip):
    """Too few pages, too many copies, broken states: nothing changes."""
    c = Cache(moehip, 8, 6, 30, 4, max_copies=3, seed=6)
    c.grow(14)
    one = next(r for r in range(8) if c.held[r] % 4)
    assert c.step([one] * 8) == B.TOO_MANY
    keep = c.at.copy()
    c.at[1] = 1
    assert c.step([one] * 3 + [r for r in range(8) if r != one][2:7]) == B.NO_PAGES
    c.at[:] = keep
    for parent in ([0, 8, 2, 3, 4, 5, 6, 7], [0, 1, -2, 3, 4, 5, 6, 7]):
        assert c.step(parent) == B.BAD
    for held in (-1, 6 * 4 + 1):
        was = c.held[3]
        c.held[3] = held
        assert c.step(np.arange(8)) == B.BAD
        c.held[3] = was
    for at in ([30, 2], [-1, 2], [0, 31], [0, -1]):
        c.at[:] = at
        assert c.step(np.arange(8)) == B.BAD
    c.at[:] = [keep[0], 30]                    # more would come back than there are pages
    assert c.step(np.full(8, -1)) == B.BAD


def test_entries_that_are_no_pages(moehip):
    """They are handed on and never given back."""
    c = Cache(moehip, 4, 5, 20, 4, seed=7)
    c.held[:] = [18, 9, 20, 3]
    pages = iter(c.rng.permutation(20))
    for r in range(4):
        for i in range(-(-c.held[r] // 4)):
            c.tables[r, i] = next(pages)
    c.tables[0, 1], c.tables[2, 3], c.tables[1, 2] = -3, 20, 1 << 30
    c.ring[:3], c.at[:] = list(pages)[:3], [0, 3]
    c.upload([0, 1, 1, -1])
    c.M.check(c.M.lib().moe_paged_fork_dev(ctypes.byref(c.args)))
    want = B.fork([0, 1, 1, -1], c.held, c.tables, c.ring, c.at, 4, 4)
    assert want["status"] == B.OK
    for n, shape in (("tables", (4, 5)), ("held", (4,)), ("ring", (20,)), ("ring_at", (2,)), ("copies", (4, 3))):
        np.testing.assert_array_equal(c.b[n].download(shape, np.int32), np.reshape(want[n], shape), err_msg=n)


def test_no_requests(moehip):
    M = moehip
    c = Cache(M, 1, 3, 5, 4, in_place=False)
    a = c.args
    a.n_req, a.parent, a.held, a.tables, a.held_out, a.tables_out = 0, None, None, None, None, None
    M.check(M.lib().moe_paged_fork_dev(ctypes.byref(a)))
    assert c.b["status"].download((1,), np.int32)[0] == 0 and c.b["ring_at_out"].download((2,), np.int32).tolist() == c.at.tolist()
    assert (c.b["copies"].download((1, 3), np.int32) == -1).all()


def test_graph(moehip):
    """Captured once, replayed over a state that changes in place, with uploads and downloads between."""
    import test_gpu_paged_serving as G
    hip = G.Hip(moehip)
    c = Cache(moehip, 24, 30, 500, 8, seed=12)
    graph = hip.capture(lambda: moehip.check(moehip.lib().moe_paged_fork_dev(ctypes.byref(c.args))))
    for i in range(6):
        c.grow(11)
        parent = _parents(c.rng, 24, 6, 0.1)
        c.upload(parent)
        hip.launch(graph)
        moehip.synchronize()
        assert c.check(parent) == B.OK
    hip.destroy(graph)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("order", ["slot", "head", "shared"])
@pytest.mark.parametrize("n_kv,hd,ps,layers,n", [(1, 16, 1, 1, 1), (3, 80, 7, 2, 5), (4, 128, 16, 3, 9), (2, 256, 33, 1, 4), (1, 32, 4, 70, 3)])
def test_copy(moehip, kind, order, n_kv, hd, ps, layers, n):
    if order == "shared" and layers > 3:
        pytest.skip("one pool for K and V: few layers will do")
    print("paged copy", kind, order, n_kv, hd, ps, layers, n, flush=True)
    M, dtype = moehip, C.TYPES[kind]
    rng = np.random.default_rng(n_kv * hd + ps)
    n_pages = 3 * n + 2
    scale = np.ones(n_kv) if kind == "e4m3" else None
    pools = [C.Pool(M, dtype, n_pages, ps, n_kv, hd, order, scale, scale) for _ in range(layers)]
    for p in pools:
        p.raw.view(np.uint8)[...] = rng.integers(0, 256, p.raw.view(np.uint8).shape)   # any bits
        p.upload()
    to = rng.permutation(n)
    copies = np.array([[rng.integers(n, n_pages), to[i], rng.integers(0, ps + 1)] for i in range(n)] + [[-1, -1, -1], [n_pages, 0, ps], [n, n_pages, ps], [n, -1, ps]], np.int32)
    copies[0, 2] = ps + 5   # a page's positions at most
    table = (M.Pages * layers)(*[p.pages for p in pools])
    dev = M.DeviceBuffer.from_array(copies)
    M.check(M.lib().moe_paged_copy_dev(dev.ptr, len(copies), table, layers))
    for p in pools:
        want = p.raw.copy()
        view = [np.lib.stride_tricks.as_strided(want.view(p.raw.dtype).reshape(-1)[(s.ctypes.data - p.raw.ctypes.data) // p.raw.itemsize:], s.shape, s.strides) for s in (p.k, p.v)]
        for src, dst, m in copies[:n]:
            for v in view:
                v[dst, :min(m, ps)] = v[src, :min(m, ps)].copy()
        p.download()
        np.testing.assert_array_equal(p.raw.view(np.uint8), want.view(np.uint8))
