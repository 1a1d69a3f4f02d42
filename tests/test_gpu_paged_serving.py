"""The paged-cache operators as a server runs them: plan, heads and attention, step after step over requests that
start, decode, end and give their pages to others; called one by one, and captured once and replayed with the step's
numbers in device memory.  Each step's plan is checked against a simulation, every new key and value and every row of
the attention against 64-bit evaluations on what the pages hold.

The model path (moe_model_step_paged) gives bit for bit what the public entry points give one after another, and, for
requests of one token, whose attention is their own value, what moe_model_forward gives."""
import ctypes

import numpy as np
import pytest

import oracle as O
import paged_cases as C
import test_gpu_paged_plan as P

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Hip:
    """Capture of the library's stream, through the HIP runtime that the library has loaded."""

    def __init__(self, M):
        path = next(l.split()[-1] for l in open("/proc/self/maps") if "libamdhip64" in l)
        self.L, self.stream = ctypes.CDLL(path), ctypes.c_void_p(M.lib().moe_get_stream())

    def ok(self, st):
        assert st == 0, f"hip error {st}"

    def capture(self, work):
        graph, run = ctypes.c_void_p(), ctypes.c_void_p()
        self.ok(self.L.hipStreamBeginCapture(self.stream, 1))
        try:
            work()
        finally:
            st = self.L.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        self.ok(st)
        self.ok(self.L.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
        self.ok(self.L.hipGraphDestroy(graph))
        return run

    def launch(self, run):
        self.ok(self.L.hipGraphLaunch(run, self.stream))

    def destroy(self, run):
        self.ok(self.L.hipGraphExecDestroy(run))


class Server:
    def __init__(self, M, kind, n_req, nq, nkv, hd, ps, width, n_pages, tokens, order, seed):
        self.M, self.nq, self.nkv, self.hd, self.tokens = M, nq, nkv, hd, tokens
        self.rng = np.random.default_rng(seed)
        dtype = C.TYPES[kind]
        scales = [0.01 + 0.01 * self.rng.random(nkv) for _ in "kv"] if kind == "e4m3" else [None, None]
        self.pool = C.Pool(M, dtype, n_pages, ps, nkv, hd, order, *scales)
        self.state = P.State(n_req, width, n_pages, ps, tokens, seed=seed, head=n_pages - 2)
        self.dev = P.Device(M, self.state)
        self.H = nq + 2 * nkv
        self.qn, self.kn = (self.rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in "qk")
        self.cos, self.sin = C.rope_tables(width * ps, hd)
        buf = M.DeviceBuffer.from_array
        self.const = [buf(x) for x in (self.qn, self.kn, self.cos, self.sin)]
        self.qkv, self.q, self.out = (M.DeviceBuffer(tokens * n * hd * 4) for n in (self.H, nq, nq))
        need = M.lib().moe_paged_attn_work_bytes(tokens, nq, nkv, hd)
        self.work = buf(np.full(need, 0xA5, np.uint8))
        b = self.dev.b
        self.heads = M.PagedHeads(self.qkv.ptr, self.H * hd, tokens, nq, b["pos"].ptr, b["slot"].ptr, *[x.ptr for x in self.const[:2]], EPS,
                                  *[x.ptr for x in self.const[2:]], width * ps, hd, self.q.ptr, nq * hd)
        self.scale = float(np.float32(1 / np.sqrt(hd)))
        self.attn = M.PagedAttn(self.q.ptr, nq * hd, tokens, nq, b["req"].ptr, b["pos"].ptr, b["tables"].ptr, n_req, width, self.scale, self.out.ptr,
                                nq * hd, self.work.ptr, need)

    def calls(self):
        M, L = self.M, self.M.lib()
        M.check(L.moe_paged_plan_dev(C.ref(self.dev.args)))
        M.check(L.moe_paged_heads_dev(C.ref(self.heads), C.ref(self.pool.pages)))
        M.check(L.moe_paged_attn_dev(C.ref(self.attn), C.ref(self.pool.pages)))

    def step(self, fresh, run):
        """One step by `run`, checked; returns whether the plan could be done."""
        s, d, hd, nq, nkv, T = self.state, self.dev, self.hd, self.nq, self.nkv, self.tokens
        qkv = self.rng.standard_normal((T, self.H, hd)).astype(np.float32)
        old_q, old_out = (self.rng.standard_normal((T, nq * hd)).astype(np.float32) for _ in "qo")
        self.qkv.upload(qkv)
        self.q.upload(old_q)
        self.out.upload(old_out)
        d.b["fresh"].upload(np.asarray(fresh, np.int32))
        run()
        starts, req, pos, slot, status = s.step(fresh)
        for n, w in (("starts", starts), ("req", req), ("pos", pos), ("slot", slot), ("status", np.array([status]))):
            np.testing.assert_array_equal(d.get(n, w.size), w, err_msg=n)
        np.testing.assert_array_equal(d.get("tables", s.n_req, s.width), s.tables)
        np.testing.assert_array_equal(d.get("held2", s.n_req), s.held)
        self.pool.download()
        q, out = self.q.download((T, nq * hd), np.float32), self.out.download((T, nq * hd), np.float32)
        at = np.maximum(pos, 0)
        cs = [a[at][:, None].astype(np.float64) for a in (self.cos, self.sin)]
        x = qkv.astype(np.float64)
        qd, qt = C.turn_head(x[:, :nq], self.qn.astype(np.float64), EPS, *cs, hd)
        kd, kt = C.turn_head(x[:, nq:nq + nkv], self.kn.astype(np.float64), EPS, *cs, hd)
        for t in range(T):
            if req[t] < 0:   # a row behind the last token
                np.testing.assert_array_equal(q[t], old_q[t])
                np.testing.assert_array_equal(out[t], old_out[t])
                continue
            assert (np.abs(q[t].reshape(nq, hd) - qd[t]) <= qt[t]).all()
            k, v = self.pool.rows(s.tables[req[t]], int(pos[t]) + 1)
            dt = self.pool.dtype
            for got, want, tol, side in ((k[-1], kd[t], kt[t], 0), (v[-1], x[t, nq + nkv:], 0.0, 1)):
                f = self.pool.factor(side)
                lim = tol * (1 + C.HALF[dt]) + np.maximum(np.abs(want) * (C.HALF[dt] + 4 * C.U), C.TINY[dt] * f)
                assert (np.abs(got - want) <= lim).all(), f"row {t}, {'kv'[side]}"
            want, tol = C.attend(q[t].reshape(nq, hd).astype(np.float64), k, v, self.scale)
            got = out[t].reshape(nq, hd)
            assert (np.abs(got - want) <= tol).all(), f"row {t}: {np.max(np.abs(got - want) / tol):.2f} times the bound"
        return status == P.OK

    def life(self, steps):
        """fresh tokens of each step: prompts first, then decode; requests end and their places are taken again"""
        n = self.state.n_req
        for i in range(steps):
            fresh = np.ones(n, np.int64)
            idle = self.state.held == 0
            room = max(1, (self.tokens - n) // max(1, int(idle.sum())))
            fresh[idle] = self.rng.integers(0, room + 1, int(idle.sum()))
            long = self.state.held + fresh > self.state.width * self.state.ps
            fresh[long] = -1
            if i % 3 == 2:
                fresh[self.rng.integers(0, n)] = -1
            yield fresh


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("n_req,nq,nkv,hd,ps,width,n_pages,tokens,order", [
    (5, 8, 2, 64, 16, 12, 40, 48, "slot"), (3, 32, 4, 128, 7, 30, 60, 70, "head"), (20, 6, 1, 48, 32, 3, 50, 90, "shared")])
def test_server(moehip, kind, n_req, nq, nkv, hd, ps, width, n_pages, tokens, order):
    print("paged server", kind, n_req, ps, flush=True)
    sv = Server(moehip, kind, n_req, nq, nkv, hd, ps, width, n_pages, tokens, order, seed=n_req)
    done = sum(sv.step(fresh, sv.calls) for fresh in sv.life(12))
    assert done >= 8


@pytest.mark.parametrize("kind", ["f32", "e4m3"])
def test_server_captured(moehip, kind):
    """One capture of the three calls, replayed with other numbers in device memory, eager steps between; a second
    capture with a work buffer of its own beside it."""
    M, hip = moehip, Hip(moehip)
    sv = Server(M, kind, 6, 16, 4, 64, 16, 20, 90, 40, "slot", seed=77)
    other = Server(M, kind, 2, 4, 1, 128, 8, 40, 100, 30, "slot", seed=78)
    run, run2 = hip.capture(sv.calls), hip.capture(other.calls)
    steps = [sv.life(9), other.life(9)]
    for i in range(9):
        sv.step(next(steps[0]), sv.calls if i % 4 == 3 else (lambda: hip.launch(run)))
        other.step(next(steps[1]), lambda: hip.launch(run2))
        M.synchronize()
    hip.destroy(run)
    hip.destroy(run2)


# ---- the model


def _caches(M, tm, dtype, n_req, tokens, ps=8, width=6):
    scale = np.full(tm.nkv, 0.02, np.float32) if dtype == C.E4M3 else None
    return M.PagedCache(tm.L, tm.nkv, tm.hd, n_req * width, ps, n_req, width, tokens, dtype, scale, scale)


@pytest.mark.parametrize("n_req", [1, 3, 20, 40])
def test_model_single_tokens(moehip, n_req):
    """Requests of one token: the attention is the token's own value, so the logits are moe_model_forward's, bit for bit."""
    M = moehip
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=32, E=16, V=97, seed=5, bias=True, random_norms=True)
    m = M.model_from_tiny(tm)
    ids = np.arange(n_req) * 7 % 97
    lg, nx = m.step_paged(_caches(M, tm, C.F32, n_req, n_req + 2), np.ones(n_req), ids)
    for r in range(n_req):
        m.reset()
        want, choice = m.forward([ids[r]])
        np.testing.assert_array_equal(lg[r].view(np.uint32), want.view(np.uint32), err_msg=f"request {r}")
        assert nx[r] == choice
    m.close()


def _chain(M, tm, layers, cache, ids, T):
    """A step by the public entry points, one after another -> logits [n_req, V]"""
    L, n = M.lib(), cache.n_req
    buf = M.DeviceBuffer.from_array
    f = np.float32
    x = tm.tok_emb[np.clip(ids, 0, tm.V - 1)].astype(f)
    nqkv, Dq = (tm.nq + 2 * tm.nkv) * tm.hd, tm.nq * tm.hd
    cos, sin = (M.DeviceBuffer.from_array(a) for a in _rope(tm))
    M.check(L.moe_paged_plan_dev(C.ref(cache.plan)))
    p = cache.plan
    need = L.moe_paged_attn_work_bytes(T, tm.nq, tm.nkv, tm.hd)
    work, H = M.DeviceBuffer(need), buf(np.zeros((T, Dq), f))
    for l, lw in enumerate(tm.layers):
        dx, dn, w1 = buf(x), M.DeviceBuffer(x.nbytes), buf(lw["rms1_w"])
        M.check(L.moe_rmsnorm_dev(dx.ptr, w1.ptr, dn.ptr, T, tm.D, tm.eps))
        W = buf(np.concatenate([lw["Wq"], lw["Wk"], lw["Wv"]]))
        dq = M.DeviceBuffer(T * nqkv * 4)
        M.check(L.moe_matmul_f32_dev(dn.ptr, W.ptr, dq.ptr, T, nqkv, tm.D))
        qn, kn = buf(lw["q_norm"]), buf(lw["k_norm"])
        h = M.PagedHeads(dq.ptr, nqkv, T, tm.nq, p.pos, p.slot, qn.ptr, kn.ptr, tm.eps, cos.ptr, sin.ptr, 64, tm.hd, dq.ptr, nqkv)
        M.check(L.moe_paged_heads_dev(C.ref(h), C.ref(cache.layers[l])))
        a = M.PagedAttn(dq.ptr, nqkv, T, tm.nq, p.req, p.pos, p.tables, n, p.max_pages, float(f(1) / np.sqrt(f(tm.hd))), H.ptr, Dq, work.ptr, need)
        M.check(L.moe_paged_attn_dev(C.ref(a), C.ref(cache.layers[l])))
        wo, do = buf(lw["Wo"]), M.DeviceBuffer(x.nbytes)
        M.check(L.moe_matmul_f32_dev(H.ptr, wo.ptr, do.ptr, T, tm.D, Dq))
        x = layers[l].block_forward(x + do.download(x.shape, f), tm.eps)
    starts = cache.array("starts", n + 1)
    last = np.stack([x[b - 1] if b > a else np.zeros(tm.D, f) for a, b in zip(starts[:-1], starts[1:])])
    dl, df, fn = buf(last), M.DeviceBuffer(last.nbytes), buf(tm.final_norm_w)
    M.check(L.moe_rmsnorm_dev(dl.ptr, fn.ptr, df.ptr, n, tm.D, tm.eps))
    head, lg = buf(tm.tok_emb if tm.lm_head is None else tm.lm_head), M.DeviceBuffer(n * tm.V * 4)
    M.check(L.moe_matmul_f32_dev(df.ptr, head.ptr, lg.ptr, n, tm.V, tm.D))
    return lg.download((n, tm.V), f)


def _rope(tm):
    """the reference's tables (test_model_trace.c:310-336) as the host C library gives them"""
    libm = ctypes.CDLL("libm.so.6")
    for n, k in (("powf", 2), ("cosf", 1), ("sinf", 1)):
        getattr(libm, n).restype, getattr(libm, n).argtypes = ctypes.c_float, [ctypes.c_float] * k
    f = np.float32
    inv = [f(libm.powf(f(tm.theta), f(f(-2.0) * f(i)) / f(tm.hd))) for i in range(tm.hd // 2)]
    ang = [[f(f(p) * v) for v in inv] for p in range(64)]
    return [np.array([[fn(a) for a in row] for row in ang], f) for fn in (libm.cosf, libm.sinf)]


@pytest.mark.parametrize("kind", list(C.TYPES))
def test_model_steps(moehip, kind):
    """Prompts, decode steps and an ended request: the model's step equals the entry points' chain bit for bit, and the
    choice is moe_greedy_dev's."""
    print("paged model", kind, flush=True)
    M, dtype = moehip, C.TYPES[kind]
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=32, E=16, V=97, seed=9, random_norms=True)
    m = M.model_from_tiny(tm)
    layers = [M.MoeLayer.from_arrays(lw["experts"].dtype, lw["router_w"], lw["router_b"], lw["experts"].gq, lw["experts"].gs, lw["experts"].uq,
                                     lw["experts"].us, lw["experts"].dq, lw["experts"].ds, lw["rms2_w"], tm.top_k) for lw in tm.layers]
    n, T = 4, 24
    mine, theirs = _caches(M, tm, dtype, n, T), _caches(M, tm, dtype, n, T)
    rng = np.random.default_rng(3)
    for fresh in ([5, 1, 9, 0], [1, 1, 1, 6], [1, -1, 1, 1], [1, 12, 1, 1], [0, 1, 3, 1]):
        ids = rng.integers(0, tm.V, T).astype(np.int32)
        lg, nx = m.step_paged(mine, fresh, ids)
        theirs.set_step(fresh, ids)
        want = _chain(M, tm, layers, theirs, ids, T)
        assert mine.status == theirs.status == 0
        for r, k in enumerate(fresh):
            if k <= 0:
                assert nx[r] == -1 and not lg[r].any()
                continue
            np.testing.assert_array_equal(lg[r].view(np.uint32), want[r].view(np.uint32), err_msg=f"request {r}")
            assert nx[r] == O.greedy(want[r])
    # a step that cannot be done: no request has tokens in it
    lg, nx = m.step_paged(mine, [T, 1, 1, 1], np.zeros(T, np.int32))
    assert mine.status == P.TOKENS and (nx == -1).all()
    held = mine.array("held", n)
    np.testing.assert_array_equal(held, theirs.array("held", n))
    for l in layers:
        l.close()
    m.close()


def test_model_refusals(moehip):
    M = moehip
    tm = O.TinyModel(seed=4)
    m = M.model_from_tiny(tm)
    ok = _caches(M, tm, C.F32, 2, 4)
    lg, nx = M.DeviceBuffer(2 * tm.V * 4), M.DeviceBuffer(8)
    f = M.lib().moe_model_step_paged
    args = [m.h, C.ref(ok.plan), ok.layers, ok._b["ids"].ptr, lg.ptr, nx.ptr]
    for i in range(4):
        assert f(*[None if j == i else a for j, a in enumerate(args)]) == 2
    assert f(*args[:4], None, None) == 2
    wrong = M.PagedCache(tm.L, tm.nkv, 32, 12, 8, 2, 6, 4)
    assert f(m.h, C.ref(ok.plan), wrong.layers, *args[3:]) == 2 and M.lib().moe_last_error()
    small = _caches(M, tm, C.F32, 2, 4, width=5)
    assert f(m.h, C.ref(ok.plan), small.layers, *args[3:]) == 2
    m.close()


def test_model_refuses_before_any_work(moehip):
    """Pages of the last layer that no call takes, a plan that none takes, a capture: refused with the state as it was."""
    M, hip = moehip, Hip(moehip)
    tm = O.TinyModel(seed=4)
    m = M.model_from_tiny(tm)
    c = _caches(M, tm, C.F32, 2, 4)
    lg, nx = M.DeviceBuffer(2 * tm.V * 4), M.DeviceBuffer(8)
    c.set_step([2, 1], [1, 2, 3])
    names = (("held", 2), ("ring_at", 2), ("tables", 12), ("status", 1))
    before = [c.array(*n) for n in names]

    def step():
        return M.lib().moe_model_step_paged(m.h, C.ref(c.plan), c.layers, c._b["ids"].ptr, lg.ptr, nx.ptr)

    last = c.layers[tm.L - 1]
    for name, bad in (("slot_stride", tm.hd - 1), ("head_stride", tm.hd + 1), ("dtype", 2), ("k", last.k + 4), ("v", None), ("k_scale", lg.ptr)):
        good = getattr(last, name)
        setattr(last, name, bad)
        assert step() == 2, name
        setattr(last, name, good)
    good, c.plan.ring = c.plan.ring, None
    assert step() == 2
    c.plan.ring = good
    hip.ok(hip.L.hipStreamBeginCapture(hip.stream, 1))
    refused, graph = step(), ctypes.c_void_p()
    hip.ok(hip.L.hipStreamEndCapture(hip.stream, ctypes.byref(graph)))
    hip.ok(hip.L.hipGraphDestroy(graph))
    assert refused == 2 and b"capture" in M.lib().moe_last_error()
    for n, want in zip(names, before):
        np.testing.assert_array_equal(c.array(*n), want, err_msg=n[0])
    assert step() == 0 and c.status == 0
    np.testing.assert_array_equal(c.array("held", 2), [2, 1])
    with pytest.raises(M.MoeError):
        c.set_step([2, 1], [1, 2])
    with pytest.raises(M.MoeError):
        c.set_step([1], [1])
    m.close()


def test_model_past_its_positions(moehip):
    """A request that outgrows the model's rotation tables has NaN logits; the other request's stay numbers."""
    M = moehip
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=32, E=16, V=97, seed=9, random_norms=True)
    m = M.model_from_tiny(tm)
    c = _caches(M, tm, C.F32, 2, 72, width=12)
    ids = np.arange(72) % tm.V
    lg, _ = m.step_paged(c, [64, 3], ids)
    assert c.status == 0 and np.isfinite(lg).all()
    lg, _ = m.step_paged(c, [1, 1], ids)
    assert c.status == 0 and np.isnan(lg[0]).all() and np.isfinite(lg[1]).all()
    lg, _ = m.step_paged(c, [-1, 1], ids)
    assert c.status == 0 and not lg[0].any() and np.isfinite(lg[1]).all()
    m.close()
