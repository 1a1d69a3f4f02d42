"""The whole model (test_model_trace.c:433-571) in 64 bits with a running bound on what an fp32 evaluation in any order of
its sums may be off by: every value is a pair (x, d) with |fp32 - x| <= d.

Rules, U = 2^-24 half a step of fp32; first-order terms times 1.01, and no bound at all (infinite) where a relative error
passes 5e-3, so that 1.01 holds what they leave out:
  sum of products      sum |w| d, and U sum |w x| for each of the sum's n - 1 adds and for the products; n counts the
                       weights that are not zero, and products by 1 and -1 are exact
  rmsnorm              x inv w: the squares' sum loses (n + 2) U, half of it in inv, 6 U more; d through both factors
  rotation             3 U of the two products' sizes
  attention            scores: (hd + 3) U of the sum of products' sizes and d of both sides; a weight's relative error is
                       twice the largest score error, 8 U and 4 U of the scores' range, the sums' (n + 32) U
  expert products      activations are cut to whole sevenths (kernels.c:96-128): exact where [x - d, x + d] holds no
                       border, else off by whole steps; the dot of whole numbers is exact, 4 U behind it
  silu                 slope at most 1.1, 8 U
A random model's bound is useless after one layer (|w| d adds up where errors do not), so `plain_model` has products that
take and sign values: the layer's norms, rotation, attention, experts and residuals are all there.  top_k is the number of
experts: no choice of experts can flip."""
import numpy as np

U = 2.0 ** -24
MORE = 1.01


def plain_model(O, seed, L, experts, hd=16, nq=4, nkv=2, bias=False):
    """A TinyModel whose products but the experts' and the router's take and sign values.  experts false: theirs add zero."""
    D = nq * hd
    tm = O.TinyModel(D=D, L=L, hd=hd, nq=nq, nkv=nkv, dff=32, E=8, top_k=8, V=D, seed=seed, std=0.1, theta=1e4, random_norms=True, bias=bias, expert_std=0.3)
    rng = np.random.default_rng(seed)

    def take(rows):
        W = np.zeros((rows, D), np.float32)
        W[np.arange(rows), rng.permutation(D)[:rows]] = rng.choice([-1, 1], rows)
        return W

    tm.tok_emb = rng.standard_normal((D, D)).astype(np.float32)
    tm.lm_head = take(D)
    for lw in tm.layers:
        lw["Wq"], lw["Wk"], lw["Wv"], lw["Wo"] = take(D), take(nkv * hd), take(nkv * hd), take(D)
        if not experts:
            lw["experts"].ds[...] = 0
    tm._build_structs()
    return tm


def product(x, d, W):
    W = W.astype(np.float64)
    n = (W != 0).sum(-1)
    rounded = n - 1 + ~np.isin(W, (-1, 0, 1)).all(-1)
    return x @ W.T, MORE * (d @ np.abs(W).T + rounded * U * (np.abs(x) @ np.abs(W).T))


def add(x, d, y, e):
    z = x + y
    return z, d + e + U * np.abs(z)


def norm(x, d, w, eps):
    n = x.shape[-1]
    w = np.ones(n) if w is None else w.astype(np.float64)
    ms = (x * x).mean(-1, keepdims=True) + eps
    inv = ms ** -0.5
    y = x * inv * w
    dinv = (np.abs(x) * d).sum(-1, keepdims=True) / n / ms     # relative
    dinv = np.where(dinv > 5e-3, np.inf, dinv)
    return y, MORE * (d * inv * np.abs(w) + np.abs(y) * (dinv + (n / 2 + 8) * U))


def turn(x, d, cos, sin):
    h = x.shape[-1] // 2
    (a, b), (da, db) = (x[..., :h], x[..., h:]), (d[..., :h], d[..., h:])
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    y = np.concatenate([a * c - b * s, b * c + a * s], -1)
    e = np.concatenate([np.abs(c) * da + np.abs(s) * db + 3 * U * (np.abs(a * c) + np.abs(b * s)),
                        np.abs(c) * db + np.abs(s) * da + 3 * U * (np.abs(b * c) + np.abs(a * s))], -1)
    return y, MORE * e


def attend(q, dq, k, dk, v, dv, scale):
    """rows [T, heads, hd], causal -> [T, heads * hd]"""
    T, nq, hd = q.shape
    g = nq // k.shape[1]
    out, tol = np.zeros((T, nq, hd)), np.zeros((T, nq, hd))
    for t in range(T):
        for h in range(nq):
            kh, dkh, vh, dvh = (z[:t + 1, h // g] for z in (k, dk, v, dv))
            s = scale * (kh @ q[t, h])
            ds = scale * (np.abs(kh) @ dq[t, h] + dkh @ np.abs(q[t, h]) + dkh @ dq[t, h] + (hd + 3) * U * (np.abs(kh) @ np.abs(q[t, h])))
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vh
            ds = np.inf if ds.max() > 2.5e-3 else ds.max()
            tol[t, h] = MORE * ((2 * ds + 4 * U * (s.max() - s.min()) + (t + 41) * U) * (p @ np.abs(vh)) + p @ dvh)
    return out.reshape(T, -1), tol.reshape(T, -1)


def q4_values(q):
    """[rows, K / 2] bytes -> [rows, K] whole numbers (kernels.c:110-112)"""
    q = q.astype(np.int64)
    w = np.empty((q.shape[0], 2 * q.shape[1]))
    w[:, 0::2], w[:, 1::2] = (q & 15) - 8, (q >> 4) - 8
    return w


def expert_product(x, d, q, s):
    w, s = q4_values(q), s.astype(np.float64)
    t = np.trunc(7 * x)
    far = np.minimum(7 * d + 8 * U * np.abs(x), 1e9)   # (the product by 7 is rounded too)
    dt = np.maximum(np.abs(np.trunc(7 * x + far) - t), np.abs(np.trunc(7 * x - far) - t))
    y = (t @ w.T) / 7 * s
    return y, MORE * ((dt @ np.abs(w).T) / 7 * s + 4 * U * np.abs(y))


def experts(x, d, lw, E):
    ex = lw["experts"]
    lg, dl = product(x, d, lw["router_w"])
    if lw["router_b"] is not None:
        lg, dl = add(lg, dl, lw["router_b"].astype(np.float64), 0.0)
    p = np.exp(lg - lg.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    dp = MORE * p * (2 * dl.max(-1, keepdims=True) + (E + 16) * U + 4 * U * (lg.max(-1, keepdims=True) - lg))
    out, tol, size = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    for e in range(E):
        a, da = expert_product(x, d, ex.gq[e], ex.gs[e])
        u, du = expert_product(x, d, ex.uq[e], ex.us[e])
        act = a / (1 + np.exp(-a))
        dact = 1.1 * da + 8 * U * np.abs(act)
        h = act * u
        y, dy = expert_product(h, MORE * (dact * np.abs(u) + np.abs(act) * du + dact * du + U * np.abs(h)), ex.dq[e], ex.ds[e])
        pe, dpe = p[:, e:e + 1], dp[:, e:e + 1]
        out += pe * y
        tol += MORE * (pe * dy + dpe * (np.abs(y) + dy))
        size += np.abs(pe * y)
    return out, tol + (E + 2) * U * size


@np.errstate(invalid="ignore")   # (an infinite bound times a zero weight)
def forward(tm, ids, tables, stored=(0.0, 0.0)):
    """ids of one request, from position 0 -> (logits [T, V], bound).  tables: the rotation's cos and sin [positions,
    hd / 2]; stored: half a step of the cache's type, relative, and half its smallest step."""
    assert tm.top_k == tm.E and tm.expert_dtype == 3
    T = len(ids)
    cos, sin = (a[:T] for a in tables)
    x = tm.tok_emb[np.asarray(ids)].astype(np.float64)
    d = np.zeros_like(x)
    for lw in tm.layers:
        xn, dn = norm(x, d, lw["rms1_w"], tm.eps)
        heads = []
        for n, W, b, w in ((tm.nq, "Wq", "bq", "q_norm"), (tm.nkv, "Wk", "bk", "k_norm"), (tm.nkv, "Wv", "bv", None)):
            y, e = product(xn, dn, lw[W])
            if lw[b] is not None:
                y, e = add(y, e, lw[b].astype(np.float64), 0.0)
            y, e = (z.reshape(T, n, tm.hd) for z in (y, e))
            if w:
                y, e = turn(*(norm(y, e, lw[w], tm.eps) if lw[w] is not None else (y, e)), cos, sin)
            if W != "Wq":
                e = e * (1 + stored[0]) + np.maximum(stored[0] * np.abs(y), stored[1])
            heads += [y, e]
        a, da = attend(*heads, 1 / np.sqrt(tm.hd))
        o, do = product(a, da, lw["Wo"])
        if lw["bo"] is not None:
            o, do = add(o, do, lw["bo"].astype(np.float64), 0.0)
        xa, dxa = add(x, d, o, do)
        m, dm = experts(*norm(xa, dxa, lw["rms2_w"], tm.eps), lw, tm.E)
        x, d = add(xa, dxa, m, dm)
    f, df = norm(x, d, tm.final_norm_w, tm.eps)
    return product(f, df, tm.tok_emb if tm.lm_head is None else tm.lm_head)
