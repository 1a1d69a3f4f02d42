"""moe_paged_plan_dev against a plain simulation of the cache's book-keeping: every output, every entry of the tables and
the ring, over steps that run in place and steps that cannot be done."""
import numpy as np
import pytest

import paged_cases as C

pytestmark = pytest.mark.gpu

OK, NO_PAGES, TOKENS, LONG, BAD = range(5)


class State:
    def __init__(self, n_req, width, n_pages, ps, tokens, seed=0, head=0):
        self.n_req, self.width, self.n_pages, self.ps, self.tokens = n_req, width, n_pages, ps, tokens
        rng = np.random.default_rng(seed)
        self.ring = rng.permutation(n_pages).astype(np.int32)
        self.at = np.array([head, n_pages], np.int32)
        self.held = np.zeros(n_req, np.int32)
        self.tables = np.full((n_req, width), -1, np.int32)

    def step(self, fresh):
        """-> starts, req, pos, slot, status; the state moves on if it is OK"""
        fresh = np.asarray(fresh, np.int64)
        ps, held = self.ps, self.held.astype(np.int64)
        head, count = (int(x) for x in self.at)
        old = -(-held // ps)
        add = np.maximum(fresh, 0)
        need = -(-(held + add) // ps) - old
        back = np.where(fresh < 0, old, 0)
        req, pos, slot = (np.full(self.tokens, -1, np.int32) for _ in range(3))
        starts = np.zeros(self.n_req + 1, np.int32)
        if (held < 0).any() or (fresh < -1).any() or not 0 <= head < self.n_pages or not 0 <= count <= self.n_pages or count + back.sum() > self.n_pages:
            return starts, req, pos, slot, BAD
        if (held > self.width * ps).any() or (held + add > self.width * ps).any():
            return starts, req, pos, slot, LONG
        if add.sum() > self.tokens:
            return starts, req, pos, slot, TOKENS
        if need.sum() > count:
            return starts, req, pos, slot, NO_PAGES
        ring = self.ring.copy()
        take = give = t = 0
        for r in range(self.n_req):
            for j in range(need[r]):
                self.tables[r, old[r] + j] = self.ring[(head + take) % self.n_pages]
                take += 1
            for j in range(back[r]):
                ring[(head + count + give) % self.n_pages] = self.tables[r, j]
                give += 1
            for i in range(add[r]):
                p = held[r] + i
                page = self.tables[r, p // ps]
                req[t], pos[t] = r, p
                slot[t] = page * ps + p % ps if 0 <= page < self.n_pages else self.n_pages * ps
                t += 1
            starts[r + 1] = t
        self.ring, self.at = ring, np.array([(head + take) % self.n_pages, count - take + give], np.int32)
        self.held = np.where(fresh < 0, 0, held + add).astype(np.int32)
        return starts, req, pos, slot, OK


class Device:
    def __init__(self, M, s, in_place=True):
        self.M, self.s = M, s
        new = lambda a: M.DeviceBuffer.from_array(np.ascontiguousarray(a, np.int32))  # noqa: E731
        self.b = {n: new(getattr(s, n)) for n in ("ring", "held", "tables")}
        self.b["at"] = new(s.at)
        self.b["held2"] = self.b["held"] if in_place else new(np.full(s.n_req, 9))
        self.b["at2"] = self.b["at"] if in_place else new([9, 9])
        for n, size in (("starts", s.n_req + 1), ("req", s.tokens), ("pos", s.tokens), ("slot", s.tokens), ("status", 1), ("fresh", s.n_req)):
            self.b[n] = new(np.full(max(size, 1), 55))
        p = {n: b.ptr for n, b in self.b.items()}
        self.args = M.PagedPlan(s.n_req, s.width, s.n_pages, s.ps, s.tokens, p["fresh"], p["held"], p["at"], p["ring"], p["tables"], p["held2"], p["at2"],
                                p["starts"], p["req"], p["pos"], p["slot"], p["status"])

    def get(self, n, *shape):
        return self.b[n].download(shape, np.int32)

    def step(self, fresh):
        s = self.s
        self.b["fresh"].upload(np.asarray(fresh, np.int32))
        self.M.check(self.M.lib().moe_paged_plan_dev(C.ref(self.args)), "paged_plan")
        want = s.step(fresh)
        for n, w in zip(("starts", "req", "pos", "slot"), want):
            np.testing.assert_array_equal(self.get(n, w.size), w, err_msg=n)
        assert self.get("status", 1)[0] == want[4]
        np.testing.assert_array_equal(self.get("held2", s.n_req), s.held)
        np.testing.assert_array_equal(self.get("at2", 2), s.at)
        np.testing.assert_array_equal(self.get("ring", s.n_pages), s.ring)
        np.testing.assert_array_equal(self.get("tables", s.n_req, s.width), s.tables)
        return want[4]


@pytest.mark.parametrize("n_req,width,n_pages,ps,tokens", [(1, 4, 4, 16, 64), (5, 8, 30, 7, 100), (64, 20, 1000, 16, 700), (1024, 6, 5000, 1, 3000),
                                                          (1025, 9, 4000, 24, 2500), (2100, 5, 9000, 16, 20000), (3, 700, 2100, 16, 9000)])
def test_steps(moehip, n_req, width, n_pages, ps, tokens):
    """A server's life: prompts, decode steps, requests that end and whose place is taken again."""
    print("paged plan", n_req, width, n_pages, ps, flush=True)
    rng = np.random.default_rng(n_req)
    s = State(n_req, width, n_pages, ps, tokens, seed=ps, head=n_pages - 1)
    d = Device(moehip, s)
    done = 0
    for step in range(14):
        room = min(tokens // n_req, width * ps)
        fresh = np.ones(n_req, np.int64)
        if step % 4 == 0:
            fresh = rng.integers(0, max(1, room // 2) + 1, n_req)
        fresh[rng.random(n_req) < 0.2] = -1
        fresh[rng.random(n_req) < 0.1] = 0
        if step == 5:
            fresh[:] = -1            # every request ends
        if step == 6:
            fresh[:] = 0             # nothing to do
        done += d.step(fresh) == OK
    assert done >= 5


def test_long_prompt_and_other_buffers(moehip):
    """One prompt of thousands of tokens over many pages; outputs beside the inputs leave those as they were."""
    s = State(40, 600, 3000, 16, 10000, seed=2, head=2990)
    d = Device(moehip, s, in_place=False)
    before = s.held.copy(), s.at.copy()
    assert d.step([1] * 20 + [9500] + [3] * 19) == OK
    np.testing.assert_array_equal(d.get("held", 40), before[0])
    np.testing.assert_array_equal(d.get("at", 2), before[1])


def test_steps_that_cannot_be_done(moehip):
    """Each refusal leaves the state as it was, and the next step that fits goes on from it."""
    s = State(4, 6, 12, 8, 40, seed=3, head=5)
    d = Device(moehip, s)
    assert d.step([20, 8, 0, 1]) == OK           # 3 + 1 + 0 + 1 pages
    assert d.step([28, 12, 1, 0]) == TOKENS
    assert d.step([29, 0, 0, 0]) == LONG         # 49 of 48 positions
    assert d.step([0, 33, 0, 0]) == OK           # 6 pages: 2 left... 10 in use
    assert d.step([0, 0, 24, 0]) == NO_PAGES     # 3 of 2
    assert d.step([0, 0, 24, -1]) == NO_PAGES    # pages given back serve the next step
    assert d.step([0, 0, 0, -2]) == BAD
    assert d.step([-1, 0, 16, -1]) == OK
    assert d.step([40, 0, 0, 0]) == NO_PAGES     # 5 of 4
    assert d.step([32, 0, 0, 0]) == OK


@pytest.mark.parametrize("at", [[-1, 3], [12, 3], [0, -1], [0, 13]])
def test_broken_ring(moehip, at):
    s = State(2, 4, 12, 8, 20, seed=4)
    s.at = np.array(at, np.int32)
    assert Device(moehip, s).step([1, 1]) == BAD


def test_negative_length_and_pages_that_are_none(moehip):
    s = State(3, 4, 12, 8, 20, seed=5)
    s.held = np.array([5, -3, 2], np.int32)
    assert Device(moehip, s).step([1, 1, 1]) == BAD
    s = State(3, 4, 12, 8, 20, seed=6)
    s.held = np.array([5, 8, 2], np.int32)
    s.at[1] = 9
    s.tables[:, 0] = [12, 3, -1]                 # no pages
    s.ring[1] = 77
    assert Device(moehip, s).step([1, 9, 2]) == OK


def test_no_requests_and_no_tokens(moehip):
    assert Device(moehip, State(0, 4, 12, 8, 5)).step([]) == OK
    assert Device(moehip, State(3, 4, 12, 8, 0)).step([0, -1, 0]) == OK
    assert Device(moehip, State(3, 4, 12, 8, 0)).step([0, 1, 0]) == TOKENS
