"""Beam searches as a program runs them: moe_model_step_beams step after step, and Model.beam_search.

Each step's choice is checked against the selection in 64 bits on the logits it had, its tables and pages against the
simulation, and its logits against the 64-bit model and its bound (model64.py) over each beam's own tokens; so a beam that
read another's pages, or a page that was not copied, shows."""
import ctypes

import numpy as np
import pytest

import beam_cases as B
import model64
import oracle as O
import paged_cases as C
import test_gpu_beam_select as S

pytestmark = pytest.mark.gpu


class Search:
    def __init__(self, M, m, prompts, n_beam, steps, kind, ps, eos, spare=0):
        self.M, self.m, self.G, self.K, self.eos = M, m, len(prompts), n_beam, eos
        self.R, self.V = self.G * n_beam, m.V
        R, V = self.R, self.V
        width = -(-(max(map(len, prompts)) + steps) // ps) + 1
        c = m.cfg
        self.c = M.PagedCache(c.n_layers, c.n_kv, c.head_dim, R * width, ps, R, width, max(R, sum(map(len, prompts))), C.TYPES[kind])
        fresh = np.zeros(R, np.int32)
        fresh[::n_beam] = [len(p) for p in prompts]
        self.c.set_step(fresh, np.concatenate(prompts))
        buf = M.DeviceBuffer.from_array
        self.logits = M.DeviceBuffer(R * V * 4)
        M.check(M.lib().moe_model_step_paged(m.h, ctypes.byref(self.c.plan), self.c.layers, self.c._b["ids"].ptr, self.logits.ptr, None))
        assert self.c.status == 0
        self.c.plan.max_tokens = R + spare if R + spare <= self.c.max_tokens else R
        self.score = np.where(np.arange(R) % n_beam == 0, 0, -np.inf).astype(np.float32)
        self.done = np.zeros(R, np.int32)
        self.seq = [list(p) for p in prompts for _ in range(n_beam)]   # of a row that holds any
        self.held = fresh.copy()
        self.b = {"score": buf(self.score), "done": buf(self.done), "parent": buf(np.zeros(R, np.int32)), "token": buf(np.zeros(R, np.int32))}
        need = M.lib().moe_beam_select_work_bytes(self.G, n_beam, V)
        self.work = M.DeviceBuffer(need)
        p = {n: x.ptr for n, x in self.b.items()}
        self.select = M.BeamSelect(self.G, n_beam, V, self.logits.ptr, V, p["score"], p["done"], None, eos, 0, p["parent"], p["token"], p["score"], p["done"],
                                   self.c._b["fresh"].ptr, self.work.ptr, need)
        self.fork = self.c.fork_args(p["parent"])

    def state(self):
        p = self.c.plan
        return [self.c.array(n, *s) for n, s in (("held", (p.n_req,)), ("tables", (p.n_req, p.max_pages)), ("ring", (p.n_pages,)), ("ring_at", (2,)))]

    def step(self):
        M, R = self.M, self.R
        logits = self.logits.download((R, self.V), np.float32)
        held, tables, ring, at = self.state()
        M.check(M.lib().moe_model_step_beams(self.m.h, ctypes.byref(self.select), ctypes.byref(self.fork), ctypes.byref(self.c.plan), self.c.layers, self.logits.ptr), "step")
        got = {n: self.b[n].download((R,), np.int32) for n in ("parent", "token", "done")}
        got.update(score=self.b["score"].download((R,), np.float32), fresh=self.c.array("fresh", R))
        S.check(got, logits, self.score, self.done, None, self.K, self.eos, 0)
        assert self.c.fork_status == 0 and self.c.status == 0
        want = B.fork(got["parent"], held, tables, ring, at, self.c.plan.page_size, R)
        assert want["status"] == B.OK
        np.testing.assert_array_equal(self.c.array("copies", R, 3), want["copies"])
        held, tables, ring, at = self.state()
        np.testing.assert_array_equal(held, want["held"] + got["fresh"])
        for r in range(R):   # (the plan then adds a page where one is full)
            used = -(-int(want["held"][r]) // self.c.plan.page_size)
            np.testing.assert_array_equal(tables[r, :used], want["tables"][r, :used])
        self.seq = [list(self.seq[p]) + ([int(t)] if f else []) if p >= 0 else [] for p, t, f in zip(got["parent"], got["token"], got["fresh"])]
        for r in range(R):
            if got["fresh"][r]:
                assert held[r] == len(self.seq[r])
        self.score, self.done = got["score"], got["done"]
        return got


@pytest.mark.parametrize("kind,experts,seed,nq,nkv", [("f32", False, 21, 4, 2), ("f16", False, 22, 16, 2), ("f32", True, 23, 4, 2)])
@pytest.mark.parametrize("G,K,ps,spare", [(1, 4, 16, 0), (3, 5, 4, 2), (2, 16, 8, 1), (2, 3, 8, 1)])
def test_steps(moehip, kind, experts, seed, nq, nkv, G, K, ps, spare):
    print("beam steps", kind, experts, nq, nkv, G, K, ps, flush=True)
    dtype = C.TYPES[kind]
    tm = model64.plain_model(O, seed, 1, experts, nq=nq, nkv=nkv)
    m = moehip.model_from_tiny(tm, 256)
    rng = np.random.default_rng(seed + K)
    lo, hi = (140, 200) if K == 3 else (20, 60)   # (on either side of what beams read together)
    prompts = [rng.integers(0, tm.V, int(rng.integers(lo, hi))) for _ in range(G)]
    rope = O.rope_tables(tm.hd, tm.theta, 256)
    stored = (0.0, 0.0) if dtype == C.F32 else (C.HALF[dtype], C.TINY[dtype])
    s = Search(moehip, m, prompts, K, 12, kind, ps, eos=int(rng.integers(0, tm.V)), spare=spare)
    told = seen = 0
    for _ in range(9):
        got = s.step()
        logits = s.logits.download((s.R, s.V), np.float32)
        for r in range(s.R):
            if not got["fresh"][r]:
                assert not logits[r].any()
                continue
            want, tol = model64.forward(tm, np.array(s.seq[r]), rope, stored)
            seen += 1
            if np.isfinite(tol[-1]).all():
                told += 1
                assert (np.abs(logits[r] - want[-1]) <= tol[-1]).all(), f"row {r}: {np.max(np.abs(logits[r] - want[-1]) / tol[-1]):.2f} times the bound"
    assert told > seen // 2
    m.close()


def _host_search(tm, rope, stored, prompt, n_beam, n_new, eos):
    """The same search on the 64-bit model -> (sequences, scores, whether every choice is clear): neighbours among the best
    n_beam + 1 candidates lie further apart than the scores may be off by, twice a step's logit bound for every step so far
    (the logit's own and the logarithm's)."""
    rows = [list(prompt)] + [[] for _ in range(n_beam - 1)]
    score, done, off, clear = np.array([0.0] + [-np.inf] * (n_beam - 1)), np.zeros(n_beam, int), np.zeros(n_beam), True
    for _ in range(n_new):
        logits, new = np.zeros((n_beam, tm.V)), off.copy()
        for i, (r, d) in enumerate(zip(rows, done)):
            if r and not d:
                x, tol = model64.forward(tm, np.array(r), rope, stored)
                logits[i] = x[-1]
                new[i] += 2 * tol[-1].max() + S.LSE + S.U * (abs(score[i]) + 50)
        wide = [np.concatenate([a, np.full((n_beam,) + a.shape[1:], f)]) for a, f in ((logits, 0.0), (score, -np.inf), (done, 0))]
        more = B.select(*wide, None, 2 * n_beam, eos, 0)
        for i in range(n_beam):
            if more["parent"][i + 1] >= 0:
                clear &= more["rank"][i] - more["rank"][i + 1] > new[more["parent"][i]] + new[more["parent"][i + 1]]
        keep = more["parent"][:n_beam]
        rows = [rows[p] + ([int(t)] if not done[p] else []) if p >= 0 else [] for p, t in zip(keep, more["token"])]
        score, done, off = more["score"][:n_beam], more["done"][:n_beam], np.where(keep >= 0, new[keep], 0)
    return [r[len(prompt):] for r in rows], score, off, clear


@pytest.mark.parametrize("kind,experts,nq", [("f32", False, 4), ("f16", False, 4), ("f32", False, 16), ("f32", True, 4)])
def test_search(moehip, kind, experts, nq):
    """Model.beam_search against the search on the 64-bit model, wherever its choices are clear."""
    M, dtype = moehip, C.TYPES[kind]
    tm = model64.plain_model(O, 40 + nq, 1, experts, nq=nq, nkv=2)
    m = M.model_from_tiny(tm, 256)
    rng = np.random.default_rng(31)
    rope = O.rope_tables(tm.hd, tm.theta, 256)
    stored = (0.0, 0.0) if dtype == C.F32 else (C.HALF[dtype], C.TINY[dtype])
    prompts = [rng.integers(0, tm.V, n) for n in (1, 17, 33)]
    compared = 0
    for n_beam, n_new, eos in ((1, 6, -1), (3, 7, -1), (4, 6, 11)):
        ids, score = m.beam_search(prompts, n_beam, n_new, eos, page_size=8, dtype=dtype)
        assert (np.diff(score) <= 0).all()
        for g, p in enumerate(prompts):
            want, ws, off, clear = _host_search(tm, rope, stored, p, n_beam, n_new, eos)
            if clear:
                compared += 1
                assert ids[g] == want, (n_beam, g)
                assert (np.abs(score[g] - ws) <= off + S.U * np.abs(ws)).all()
    assert compared >= (0 if experts else 1)   # (of nine, as many as the plain form finds clear)
    one, _ = m.beam_search(prompts[:1], 1, 6)   # one beam is the greedy choice, where it is as clear
    if _host_search(tm, rope, (0.0, 0.0), prompts[0], 1, 6, -1)[3]:
        assert one[0][0] == m.generate(prompts[0], 6)[0].tolist()
    m.close()


@pytest.mark.parametrize("n_prompt,n_beam,n_new,ps", [(5, 4, 10, 16), (1, 8, 15, 16), (3, 6, 20, 4), (2, 3, 1, 1)])
def test_search_with_no_page_to_spare(moehip, n_prompt, n_beam, n_new, ps):
    """Beams that fill their last pages at once: what a search takes by itself is enough, and what it finds does not depend on it;
    too few pages raise."""
    M = moehip
    tm = model64.plain_model(O, 50, 1, False, nq=4, nkv=2)
    m = M.model_from_tiny(tm, 256)
    prompt = [np.random.default_rng(n_new).integers(0, tm.V, n_prompt)]
    ids, score = m.beam_search(prompt, n_beam, n_new, page_size=ps)
    assert [len(x) for x in ids[0]] == [n_new] * n_beam
    more, other = m.beam_search(prompt, n_beam, n_new, page_size=ps, n_pages=300)
    assert ids == more
    np.testing.assert_array_equal(score, other)
    if n_new > 1:
        with pytest.raises(M.MoeError):
            m.beam_search(prompt, n_beam, n_new, page_size=ps, n_pages=-(-n_prompt // ps))
    m.close()


def test_search_of_fewer_tokens_than_beams(moehip):
    """One step of more beams than tokens: a beam a token, the others without one."""
    M = moehip
    tm = O.TinyModel(D=64, L=1, hd=16, nq=4, nkv=2, dff=32, E=8, top_k=8, V=7, seed=6, std=0.3, theta=1e4)
    m = M.model_from_tiny(tm, 64)
    ids, score = m.beam_search([[1, 2]], 10, 1)
    assert sorted(x[0] for x in ids[0][:7]) == list(range(7)) and ids[0][7:] == [[]] * 3
    assert np.isfinite(score[0, :7]).all() and (score[0, 7:] == -np.inf).all()
    ids, score = m.beam_search([[1, 2]], 10, 3)
    assert [len(x) for x in ids[0]] == [3] * 10 and np.isfinite(score).all()
    m.close()


def test_fork_of_a_cache(moehip):
    """PagedCache.fork between steps of any kind: answers that part ways after a common prompt are those of separate requests."""
    M = moehip
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=32, E=8, top_k=8, V=90, seed=4, std=0.3, theta=1e4)
    m = M.model_from_tiny(tm, 128)
    rng = np.random.default_rng(32)
    prompt, tails = rng.integers(0, tm.V, 21), rng.integers(0, tm.V, (4, 9))
    c = M.PagedCache(2, 2, 16, 40, 8, 4, 10, 30)
    m.step_paged(c, [21, 0, 0, 0], prompt)
    assert c.status == 0
    c.fork([0, 0, 0, 0])
    for i in range(9):
        lg, _ = m.step_paged(c, [1, 1, 1, 1], tails[:, i])
        assert c.status == 0
    for r in range(4):
        want = m.forward_full(np.concatenate([prompt, tails[r]]))
        np.testing.assert_allclose(lg[r], want, atol=2e-4 * np.abs(want).max())
    before = int(c.array("ring_at", 2)[1])
    c.fork([-1, 1, -1, 1])   # 0 and 2 end, 3 is given up for a copy of 1
    tables, held = c.array("tables", 4, 10), c.array("held", 4)
    assert held.tolist() == [0, 30, 0, 30] and tables[1, :3].tolist() == tables[3, :3].tolist() and tables[1, 3] != tables[3, 3]
    assert int(c.array("ring_at", 2)[1]) == 40 - 5 and before < 35
    with pytest.raises(M.MoeError):
        c.fork([0, 1, 2])
    with pytest.raises(M.MoeError):
        c.fork([0, 1, 2, 4])
    m.close()


class Step:
    """The operators of a search's step over a cache of two layers, without a model."""

    def __init__(self, M, G, K, V, ps, kind, n_prompt):
        self.M, self.G, self.K, self.V, self.R = M, G, K, V, G * K
        rng, R, nq, nkv, hd = np.random.default_rng(G * K), G * K, 8, 2, 64
        width = -(-(n_prompt + 40) // ps)
        self.c = c = M.PagedCache(2, nkv, hd, R * (width + 1), ps, R, width, max(R, G * n_prompt), C.TYPES[kind])
        for pool in c._pools:
            x = rng.standard_normal(pool.nbytes // 2).astype(np.float16)
            pool.upload(x if kind == "f16" else x.view(np.float32) if kind == "f32" else x)
        fresh = np.zeros(R, np.int32)
        fresh[::K] = n_prompt
        c.set_step(fresh, np.zeros(G * n_prompt, np.int32))
        M.check(M.lib().moe_paged_plan_dev(ctypes.byref(c.plan)))
        assert c.status == 0
        c.plan.max_tokens = R
        buf, zero = M.DeviceBuffer.from_array, np.zeros(R, np.int32)
        L = M.lib()
        sizes = (R, G, nq, nkv, hd)
        need = [L.moe_beam_select_work_bytes(G, K, V), L.moe_paged_share_plan_bytes(*sizes), L.moe_paged_attn_shared_work_bytes(*sizes)]
        self.b = b = {"logits": M.DeviceBuffer(4 * R * V), "score": buf(np.where(np.arange(R) % K == 0, 0, -np.inf).astype(np.float32)), "done": buf(zero), "parent": buf(zero),
                      "token": buf(zero), "q": M.DeviceBuffer(4 * R * nq * hd), "out": buf(np.zeros(R * nq * hd, np.float32)), "first": buf(np.arange(0, R + 1, K).astype(np.int32)),
                      "prefix": buf(np.zeros(G, np.int32)), "work": M.DeviceBuffer(need[0]), "plan": M.DeviceBuffer(need[1]), "attn": M.DeviceBuffer(need[2])}
        p, d = {n: x.ptr for n, x in b.items()}, {n: x.ptr for n, x in c._b.items()}
        self.select = M.BeamSelect(G, K, V, p["logits"], V, p["score"], p["done"], None, -1, 0, p["parent"], p["token"], p["score"], p["done"], d["fresh"], p["work"], need[0])
        self.fork = c.fork_args(p["parent"])
        self.share = M.PagedShare(R, R, width, ps, nq, nkv, hd, d["req"], d["pos"], d["tables"], G, p["first"], p["prefix"], p["plan"], need[1])
        self.attn = M.PagedAttn(p["q"], nq * hd, R, nq, d["req"], d["pos"], d["tables"], R, width, 0.125, p["out"], nq * hd, p["attn"], need[2])

    def calls(self):
        M, L, c, ref = self.M, self.M.lib(), self.c, ctypes.byref
        M.check(L.moe_beam_select_dev(ref(self.select)))
        M.check(L.moe_paged_fork_dev(ref(self.fork)))
        M.check(L.moe_paged_copy_dev(self.fork.copies, self.fork.max_copies, c.layers, 2))
        M.check(L.moe_paged_plan_dev(ref(c.plan)))
        M.check(L.moe_paged_share_dev(ref(self.share)))
        for l in range(2):
            M.check(L.moe_paged_attn_shared_dev(ref(self.attn), ref(c.layers[l]), ref(self.share)))

    def state(self):
        R, p = self.R, self.c.plan
        got = {n: self.c.array(n, *s) for n, s in (("held", (R,)), ("tables", (R, p.max_pages)), ("ring", (p.n_pages,)), ("ring_at", (2,)), ("req", (R,)), ("pos", (R,)))}
        got.update({n: self.b[n].download((R,), np.int32) for n in ("parent", "token")}, prefix=self.b["prefix"].download((self.G,), np.int32),
                   score=self.b["score"].download((R,), np.float32), out=self.b["out"].download((R * 512,), np.float32),
                   **{f"pool {i}": x.download((x.nbytes,), np.uint8) for i, x in enumerate(self.c._pools)})
        return got


@pytest.mark.parametrize("G,K,kind,n_prompt", [(2, 4, "f16", 45), (1, 20, "f32", 200), (3, 16, "bf16", 170)])
def test_operators_in_a_graph(moehip, G, K, kind, n_prompt):
    """The operators of a step, captured together and replayed over a state that moves on, between eager steps of another cache:
    every replay leaves what the eager step leaves."""
    import test_gpu_paged_serving as S2
    hip, V, ps = S2.Hip(moehip), 600, 16
    a, e = (Step(moehip, G, K, V, ps, kind, n_prompt) for _ in "ab")
    rng = np.random.default_rng(7)
    graph = hip.capture(a.calls)
    shared = 0
    for step in range(20):
        logits, q = (3 * rng.standard_normal((G * K, V))).astype(np.float32), rng.standard_normal((G * K, 512)).astype(np.float32)
        for x in (a, e):
            x.b["logits"].upload(logits)
            x.b["q"].upload(q)
        hip.launch(graph)
        moehip.synchronize()
        e.calls()
        assert a.c.status == e.c.status == a.c.fork_status == e.c.fork_status == 0
        got, want = a.state(), e.state()
        for n in want:
            np.testing.assert_array_equal(got[n], want[n], err_msg=f"step {step}, {n}")
        shared += int((want["prefix"] > 0).all())
        assert (want["held"] == n_prompt + step + 1).all()
    assert shared == 20
    hip.destroy(graph)


def test_step_beams_refused(moehip):
    """What the three descriptions hand on to each other has to be the same; a capture is refused."""
    import test_gpu_paged_serving as G
    M = moehip
    tm = O.TinyModel(D=64, L=1, hd=16, nq=4, nkv=2, dff=32, E=8, top_k=8, V=90, seed=5, std=0.3, theta=1e4)
    m = M.model_from_tiny(tm, 64)
    s = Search(M, m, [[1, 2, 3]], 4, 8, "f32", 8, -1)
    L, c = M.lib(), s.c

    def refused(**kw):
        args = {"select": s.select, "fork": s.fork, "plan": c.plan}
        kept = []
        for name, change in kw.items():
            for field, value in change.items():
                kept.append((args[name], field, getattr(args[name], field)))
                setattr(args[name], field, value)
        st = L.moe_model_step_beams(m.h, ctypes.byref(s.select), ctypes.byref(s.fork), ctypes.byref(c.plan), c.layers, s.logits.ptr)
        for obj, field, value in kept:
            setattr(obj, field, value)
        return st

    other = M.DeviceBuffer(1 << 16)
    for bad in (dict(select=dict(vocab=80)), dict(select=dict(n_beam=2)), dict(fork=dict(n_req=3)), dict(fork=dict(parent=other.ptr)), dict(plan=dict(fresh=other.ptr)),
                dict(plan=dict(held=other.ptr)), dict(plan=dict(tables=other.ptr)), dict(fork=dict(ring=other.ptr)), dict(fork=dict(ring_at_out=other.ptr)),
                dict(select=dict(work_bytes=0)), dict(fork=dict(copies=None)), dict(plan=dict(max_tokens=0)), dict(plan=dict(max_tokens=1 << 15))):
        assert refused(**bad) == 2, bad
    assert L.moe_model_step_beams(m.h, None, ctypes.byref(s.fork), ctypes.byref(c.plan), c.layers, s.logits.ptr) == 2
    hip = G.Hip(M)
    out = []
    hip.destroy(hip.capture(lambda: out.append(refused())))
    assert out == [2]
    s.step()
    m.close()
