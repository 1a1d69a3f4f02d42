"""The operators that serve many requests from a paged key-value cache, as calls whose speed is watched.

Three operators, in the order a serving step runs them:

  plan   moe_paged_plan_dev: pages taken from and given back to the ring of free pages, block tables extended,
         and the request, position and slot of every new token, all from the requests' lengths
  heads  moe_paged_heads_dev: RMS norm of each query and key head, position rotation, keys and values into their pages
  attn   moe_paged_attn_dev: attention of the new tokens over their requests' pages

Head geometries are the repository's model (32 query heads, 4 key-value heads of 128) and generic ones around it.
Queries and keys are as a per-head norm leaves them, values N(0, 1); an 8-bit cache has one scale a head.
With `own` false the operators run in their plain form, torch operations in 32 bits; with it true, in the library.
"""
import ctypes
import math
import os
import sys

import torch

own = False

HEADS = {"nq": 32, "nkv": 4, "hd": 128}  # the 48-layer model's attention
KINDS = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (4, torch.bfloat16), "e4m3": (5, torch.float8_e4m3fn)}
EPS = 1e-6


def listed():
    return [
        # the first answers of one request, in the model's own cache type: latency alone
        {"name": "attn_one_short", "kind": "attn", "type": "f32", "T": 1, "lo": 30, "hi": 60, "page": 16, "order": "slot", "pad": 0, **HEADS},
        # a chat server's decode step
        {"name": "attn_chat", "kind": "attn", "type": "bf16", "T": 24, "lo": 64, "hi": 2048, "page": 16, "order": "slot", "pad": 0, **HEADS},
        # one request over a very long document: the length is all there is to split
        {"name": "attn_one_long", "kind": "attn", "type": "bf16", "T": 1, "lo": 131000, "hi": 131072, "page": 64, "order": "head", "pad": 0, **HEADS},
        # a batch of middle-sized requests over an 8-bit cache
        {"name": "attn_e4m3_batch", "kind": "attn", "type": "e4m3", "T": 64, "lo": 512, "hi": 8192, "page": 32, "order": "slot", "pad": 0, **HEADS},
        # the model's own precision for a few requests, a captured batch that is not full
        {"name": "attn_f32_batch", "kind": "attn", "type": "f32", "T": 16, "lo": 100, "hi": 2048, "page": 128, "order": "head", "pad": 3, **HEADS},
        # no power of two anywhere, one request with nothing in its cache
        {"name": "attn_odd", "kind": "attn", "type": "f16", "T": 37, "lo": 0, "hi": 900, "page": 24, "order": "slot", "pad": 2, "nq": 15, "nkv": 3, "hd": 80},
        # a full card: many requests of very different lengths
        {"name": "attn_wide", "kind": "attn", "type": "bf16", "T": 256, "lo": 1, "hi": 8192, "page": 16, "order": "slot", "pad": 0, **HEADS},
        # one request's new row, in the model's own cache type
        {"name": "heads_one", "kind": "heads", "type": "f32", "T": 1, "page": 16, "order": "slot", "pad": 0, **HEADS},
        # one decode step's new rows into an 8-bit cache
        {"name": "heads_decode", "kind": "heads", "type": "e4m3", "T": 48, "page": 16, "order": "slot", "pad": 0, **HEADS},
        # a prompt's rows into a 16-bit cache
        {"name": "heads_prompt", "kind": "heads", "type": "bf16", "T": 4096, "page": 64, "order": "head", "pad": 0, **HEADS},
        # the plan of a decode step
        {"name": "plan_decode", "kind": "plan", "n_req": 64, "tokens": 64, "page": 16, "width": 512, "prompts": 0},
        # a large server's step: decode, some prompts, some requests that ended
        {"name": "plan_mixed", "kind": "plan", "n_req": 1024, "tokens": 16384, "page": 16, "width": 512, "prompts": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "heads", "plan"])
    page = rng.choice([8, 16, 16, 20, 32, 64, 100, 128, 256])
    if kind == "plan":
        n = _log(rng, 1, 1024)
        return {"kind": kind, "n_req": n, "tokens": n + _log(rng, 1, 15000), "page": page, "width": rng.randint(40, 512), "prompts": rng.randint(0, 12)}
    nkv = rng.choice([1, 2, 3, 4, 8])
    case = {"kind": kind, "type": rng.choice(list(KINDS)), "page": page, "order": rng.choice(["slot", "head"]),
            "nq": nkv * rng.choice([1, 2, 3, 4, 6, 8, 16]), "nkv": nkv, "hd": 16 * rng.randint(2, 16) if rng.random() < 0.4 else rng.choice([64, 128, 128, 256])}
    if kind == "heads":
        T = _log(rng, 1, min(4096, int(20e6 / ((case["nq"] + 2 * case["nkv"]) * case["hd"]))))
        return {**case, "T": T, "pad": min(T - 1, rng.randint(0, 5))}
    T = _log(rng, 1, 256)
    row = case["nkv"] * case["hd"] * (4 if case["type"] == "f32" else 2)
    hi = _log(rng, 1, max(2, min(131072, int(500e6 / (T * row)))))
    return {**case, "T": T, "lo": rng.randint(0, hi), "hi": hi, "pad": min(T - 1, rng.randint(0, 3))}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _ints(gen, lo, hi, *shape):
    """whole numbers lo .. hi"""
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda")


def _normed(x):
    return x * x.square().mean(-1, keepdim=True).add(EPS).rsqrt()


def _pool(gen, case, n_pages, normed):
    """One side's pages as [page, slot, head, dim], whatever their order in memory, and the scale of each head."""
    _, dtype = KINDS[case["type"]]
    dims = (n_pages, case["page"], case["nkv"], case["hd"])
    if case["order"] == "head":
        dims = (dims[0], dims[2], dims[1], dims[3])
    pool = torch.empty(dims, device="cuda", dtype=dtype)
    scale = 0.01 + 0.01 * torch.rand(case["nkv"], generator=gen, device="cuda") if case["type"] == "e4m3" else None
    view = pool if case["order"] == "slot" else pool.transpose(1, 2)
    for p in range(0, n_pages, 4096):
        x = _normal(gen, *view[p:p + 4096].shape)
        x = _normed(x) if normed else x
        if scale is not None:
            x = (x / scale[:, None]).clamp(-448, 448)
        view[p:p + 4096].copy_(x)
    return view, scale


def _tables(gen, lens, page, width, n_pages):
    """Block tables of requests that hold `lens` positions, on pages in no order; -1 behind the last."""
    used = (lens + page - 1) // page
    order = torch.randperm(n_pages, generator=gen, device="cuda")
    at = (torch.cumsum(used, 0) - used)[:, None] + torch.arange(width, device="cuda")
    live = torch.arange(width, device="cuda") < used[:, None]
    return torch.where(live, order[at.clamp(max=n_pages - 1)], -1).int()


def _prepare_attn(gen, case):
    T, page = case["T"], case["page"]
    lens = _ints(gen, case["lo"], case["hi"], T)
    if case["lo"] == 0:
        lens[T // 2] = 0
    width = max(1, -(-case["hi"] // page)) + 2
    n_pages = int(((lens + page - 1) // page).sum()) + 3
    req = torch.arange(T, device="cuda", dtype=torch.int32)
    if case["pad"]:
        req[T - case["pad"]:] = -1  # rows of a fixed batch that no request fills
    (k, ks), (v, vs) = _pool(gen, case, n_pages, True), _pool(gen, case, n_pages, False)
    return {"q": _normed(_normal(gen, T, case["nq"], case["hd"])).reshape(T, -1), "k": k, "v": v, "ks": ks, "vs": vs, "req": req,
            "pos": (lens - 1).int(), "tables": _tables(gen, lens, page, width, n_pages), "out": _normal(gen, T, case["nq"] * case["hd"]),
            "work": torch.empty(96 << 20, device="cuda", dtype=torch.uint8)}


def _prepare_heads(gen, case):
    T, page, hd = case["T"], case["page"], case["hd"]
    n_pages = 2 * -(-T // page) + 4
    (k, ks), (v, vs) = _pool(gen, case, n_pages, True), _pool(gen, case, n_pages, False)
    pos = _ints(gen, 0, 40000, T)
    angle = torch.arange(40001, device="cuda", dtype=torch.float64)[:, None] * 1e7 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    slot = torch.randperm(n_pages * page, generator=gen, device="cuda")[:T].int()
    if case["pad"]:
        slot[T - case["pad"]:] = -1
    return {"qkv": _normal(gen, T, (case["nq"] + 2 * case["nkv"]) * hd), "k": k, "v": v, "ks": ks, "vs": vs, "pos": pos.int(), "slot": slot,
            "cos": angle.cos().float(), "sin": angle.sin().float(), "qn": 1 + 0.1 * _normal(gen, hd), "kn": 1 + 0.1 * _normal(gen, hd),
            "out": _normal(gen, T, case["nq"] * hd)}


def _prepare_plan(gen, case):
    n, page, width = case["n_req"], case["page"], case["width"]
    held = _ints(gen, 0, (width - 1) * page // 2, n)
    fresh = torch.ones(n, device="cuda", dtype=torch.int64)
    room = (case["tokens"] - n) // max(1, case["prompts"])
    for i in _ints(gen, 0, n - 1, case["prompts"]).tolist():
        fresh[i] = min(room, width * page // 2 - 1)
        held[i] = held[i] // 3
    ended = torch.rand(n, generator=gen, device="cuda") < (0.03 if n > 1 else 0.0)
    fresh[ended] = -1
    used = (held + page - 1) // page
    n_pages = n * width
    ring = torch.randperm(n_pages, generator=gen, device="cuda").int()
    at = int(_ints(gen, 0, n_pages - 1, 1))
    tables = _tables(gen, held, page, width, n_pages)
    # the free pages are those that no table holds, from ring[at] on
    free = torch.ones(n_pages, device="cuda", dtype=torch.bool)
    free[tables[tables >= 0].long()] = False
    left = free.nonzero()[:, 0]
    ring[(at + torch.arange(left.numel(), device="cuda")) % n_pages] = left[torch.randperm(left.numel(), generator=gen, device="cuda")].int()
    assert left.numel() == n_pages - int(used.sum())
    new = lambda m: torch.zeros(m, device="cuda", dtype=torch.int32)  # noqa: E731
    return {"fresh": fresh.int(), "held": held.int(), "ring": ring, "ring_at": torch.tensor([at, left.numel()], device="cuda", dtype=torch.int32), "tables": tables,
            "held_out": new(n), "ring_at_out": new(2), "starts": new(n + 1), "req": new(case["tokens"]), "pos": new(case["tokens"]), "slot": new(case["tokens"]),
            "status": new(1)}


def prepare(case, seed):
    state = {"attn": _prepare_attn, "heads": _prepare_heads, "plan": _prepare_plan}[case["kind"]](_gen(seed), case)
    state["case"] = case
    torch.cuda.synchronize()  # the library works on a stream of its own
    return state


# ---- the plain forms


def _values(pool, scale):
    """the numbers that a part of a pool stands for, [..., head, dim]"""
    x = pool.float()
    return x if scale is None else x * scale[:, None]


def _gather(pool, pages):
    """pool[pages], by bytes where the type has eight bits"""
    if pool.dtype == torch.float8_e4m3fn:
        return pool.view(torch.uint8)[pages].view(pool.dtype)
    return pool[pages]


def _plain_attn(s):
    case = s["case"]
    T, nkv, hd = case["T"], case["nkv"], case["hd"]
    used = max(1, -(-case["hi"] // case["page"]))
    pages = s["tables"][s["req"].clamp(min=0).long(), :used].clamp(min=0).long()
    seen = torch.arange(used * case["page"], device="cuda") <= s["pos"][:, None]  # [T, position]
    k = _values(_gather(s["k"], pages), s["ks"]).reshape(T, -1, nkv, hd)
    v = _values(_gather(s["v"], pages), s["vs"]).reshape(T, -1, nkv, hd)
    q = s["q"].reshape(T, nkv, -1, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1 / math.sqrt(hd))
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, :, None, None], v, 0.0).transpose(1, 2).contiguous()
    o = torch.matmul(p / torch.where(total == 0, 1.0, total), v).reshape(T, -1)
    return torch.where(s["req"][:, None] < 0, s["out"], o)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_heads(s):
    case = s["case"]
    T, nq, nkv, hd = case["T"], case["nq"], case["nkv"], case["hd"]
    x = s["qkv"].reshape(T, -1, hd)
    at = s["pos"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]

    def norm(h, w):
        return h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w

    q = _rotate(norm(x[:, :nq], s["qn"]), cos, sin).reshape(T, -1)
    live = s["slot"] >= 0
    slot = s["slot"][live].long()
    page, off = slot // case["page"], slot % case["page"]
    for pool, scale, h in ((s["k"], s["ks"], _rotate(norm(x[:, nq:nq + nkv], s["kn"]), cos, sin)), (s["v"], s["vs"], x[:, nq + nkv:])):
        h = h[live]
        if scale is not None:
            h = (h / scale[:, None]).clamp(-448, 448)
        h = h.to(pool.dtype)
        if pool.dtype == torch.float8_e4m3fn:
            pool, h = pool.view(torch.uint8), h.view(torch.uint8)
        pool[page, off] = h
    s["out"].copy_(torch.where(live[:, None], q, s["out"]))
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _plain_plan(s):
    case = s["case"]
    n, page, width, most = case["n_req"], case["page"], case["width"], case["tokens"]
    fresh, held, n_pages = s["fresh"].long(), s["held"].long(), s["ring"].numel()
    head, count = s["ring_at"].long()
    ended, new = fresh < 0, fresh.clamp(min=0)
    old = (held + page - 1) // page
    need = (held + new + page - 1) // page - old
    back = torch.where(ended, old, 0)
    take0, back0 = torch.cumsum(need, 0) - need, torch.cumsum(back, 0) - back
    status = torch.where((held < 0).any() | (fresh < -1).any() | (count + back.sum() > n_pages), 4, torch.where(
        (held + new > width * page).any(), 3, torch.where(new.sum() > most, 2, torch.where(need.sum() > count, 1, 0))))
    ok = status == 0
    col = torch.arange(width, device="cuda")
    j = col - old[:, None]
    give = s["ring"][(head + take0[:, None] + j) % n_pages]
    to = torch.where((col < back[:, None]) & ok, (head + count + back0[:, None] + col) % n_pages, n_pages)
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring[to] = s["tables"]
    s["tables"].copy_(torch.where((j >= 0) & (j < need[:, None]) & ok, give, s["tables"]))
    s["ring"].copy_(ring[:n_pages])
    starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)]) * ok
    t = torch.arange(most, device="cuda")
    live = t < starts[-1]
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=n - 1)
    pos = held[r] + t - starts[r]
    slot = s["tables"][r, (pos // page).clamp(max=width - 1)] * page + pos % page
    return {"tables": s["tables"], "ring": s["ring"], "held": torch.where(ended & ok, 0, held + new * ok).int(),
            "ring_at": torch.stack([(head + need.sum() * ok) % n_pages, count + (back.sum() - need.sum()) * ok]).int(), "starts": starts.int(),
            "req": torch.where(live, r, -1).int(), "pos": torch.where(live, pos, -1).int(), "slot": torch.where(live, slot, -1).int(),
            "status": status.int().reshape(1)}


# ---- the library's calls


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe.cc_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import moehip
    return moehip


def _pages(M, s):
    case, k, v = s["case"], s["k"], s["v"]
    assert k.stride() == v.stride()
    return M.Pages(k.data_ptr(), v.data_ptr(), KINDS[case["type"]][0], k.shape[0], case["page"], case["nkv"], case["hd"], k.stride(0), k.stride(2), k.stride(1),
                   s["ks"].data_ptr() if s["ks"] is not None else None, s["vs"].data_ptr() if s["vs"] is not None else None)


def _call(s):
    """The descriptors that a program fills once for its buffers: (entry point, arguments)."""
    M, case = _library(), s["case"]
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    if case["kind"] == "plan":
        a = M.PagedPlan(case["n_req"], case["width"], s["ring"].numel(), case["page"], case["tokens"], p["fresh"], p["held"], p["ring_at"], p["ring"], p["tables"],
                        p["held_out"], p["ring_at_out"], p["starts"], p["req"], p["pos"], p["slot"], p["status"])
        return M.check, M.lib().moe_paged_plan_dev, [ctypes.byref(a)]
    pages = _pages(M, s)
    if case["kind"] == "heads":
        a = M.PagedHeads(p["qkv"], s["qkv"].stride(0), case["T"], case["nq"], p["pos"], p["slot"], p["qn"], p["kn"], EPS, p["cos"], p["sin"], s["cos"].shape[0], case["hd"],
                         p["out"], s["out"].stride(0))
        return M.check, M.lib().moe_paged_heads_dev, [ctypes.byref(a), ctypes.byref(pages)]
    a = M.PagedAttn(p["q"], s["q"].stride(0), case["T"], case["nq"], p["req"], p["pos"], p["tables"], case["T"], s["tables"].shape[1], 1 / math.sqrt(case["hd"]),
                    p["out"], s["out"].stride(0), p["work"], s["work"].numel())
    return M.check, M.lib().moe_paged_attn_dev, [ctypes.byref(a), ctypes.byref(pages)]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"attn": _plain_attn, "heads": _plain_heads, "plan": _plain_plan}[kind](state)
    if "call" not in state:
        state["call"] = _call(state)
    check, entry, args = state["call"]
    check(entry(*args), kind)
    if kind == "attn":
        return state["out"]
    if kind == "heads":
        return {"q": state["out"], "k": state["k"], "v": state["v"]}
    return {"tables": state["tables"], "ring": state["ring"], "held": state["held_out"], "ring_at": state["ring_at_out"], "starts": state["starts"],
            "req": state["req"], "pos": state["pos"], "slot": state["slot"], "status": state["status"]}


def work(case):
    if case["kind"] == "plan":
        # lengths, starts and places of the tokens; a page moved is read and written once
        return {"bytes": 4 * (4 * case["n_req"] + 3 * case["tokens"] + 2 * (case["tokens"] // case["page"] + 1)), "flops": 4 * case["tokens"]}
    T, nq, nkv, hd = case["T"] - case["pad"], case["nq"], case["nkv"], case["hd"]
    size = 4 if case["type"] == "f32" else 1 if case["type"] == "e4m3" else 2
    if case["kind"] == "heads":
        return {"bytes": T * hd * (4 * (nq + 2 * nkv) + 4 * nq + 2 * nkv * size + 4) + 8 * T, "flops": T * hd * (nq + nkv) * 7}
    seen = T * (case["lo"] + case["hi"]) / 2
    return {"bytes": seen * nkv * hd * 2 * size + 8 * T * nq * hd + 4 * seen / case["page"], "flops": 4 * seen * nq * hd}


# ---- the definitions in 64 bits


def _exact_attn(s):
    case = s["case"]
    out = s["out"].double()
    for t in range(case["T"]):
        n = int(s["pos"][t]) + 1
        if int(s["req"][t]) < 0:
            continue
        out[t] = 0
        if n == 0:
            continue
        pages = s["tables"][t, :-(-n // case["page"])].long()
        k, v = (_gather(s[m], pages).flatten(0, 1)[:n].double() * (1.0 if s[m + "s"] is None else s[m + "s"].double()[:, None]) for m in "kv")
        for h in range(case["nkv"]):
            g = case["nq"] // case["nkv"]
            q = s["q"][t].double().reshape(-1, case["hd"])[h * g:(h + 1) * g]
            p = torch.softmax(q @ k[:, h].T / math.sqrt(case["hd"]), -1)
            out[t, h * g * case["hd"]:(h + 1) * g * case["hd"]] = (p @ v[:, h]).reshape(-1)
    return out


def _exact_heads(s):
    case = s["case"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    k, v, q = s["k"].double(), s["v"].double(), s["out"].double()
    x = s["qkv"].double().reshape(case["T"], -1, hd)
    keys = x[:, :nq + nkv]
    w = torch.cat([s["qn"].double().expand(nq, hd), s["kn"].double().expand(nkv, hd)])
    keys = keys * (keys.pow(2).sum(-1, keepdim=True) / hd + EPS).pow(-0.5) * w
    z = torch.complex(keys[..., :hd // 2], keys[..., hd // 2:]) * torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    keys = torch.cat([z.real, z.imag], -1)
    live = (s["slot"] >= 0).nonzero()[:, 0]
    at = s["slot"][live].long()
    one = torch.ones(nkv, device="cuda", dtype=torch.float64)
    for pool, scale, rows in ((k, s["ks"], keys[live, nq:]), (v, s["vs"], x[live, nq + nkv:])):
        rows = rows / (one if scale is None else scale.double())[:, None]
        pool[at // case["page"], at % case["page"]] = rows.clamp(-448, 448) if case["type"] == "e4m3" else rows
    q[live] = keys[live, :nq].reshape(live.numel(), -1)
    return {"q": q, "k": k, "v": v}


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    state = prepare(case, seed)
    return (_exact_attn if case["kind"] == "attn" else _exact_heads)(state)
