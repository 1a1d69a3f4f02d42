"""The operators of a beam search over the paged key-value cache, as calls whose speed is watched.

Five operators, in the order a step runs them:

  select  moe_beam_select_dev: of the log probabilities of every beam's next tokens the best of each group, with the beam
          that each continues
  fork    moe_paged_fork_dev: the requests' block tables after it: beams that go on share their full pages, a page that is
          not full is copied for all but one, pages that no beam holds go back to the ring of free ones
  copy    moe_paged_copy_dev: those pages' keys and values, in every layer
  share   moe_paged_share_dev: how many leading positions the rows of each group hold in the same pages
  attn    moe_paged_attn_shared_dev: attention of the new tokens, what a group shares read once for all its rows

The first fits any step, beams or not, whose requests came from one (several answers to one prompt), and the last two any
batch whose requests begin alike.  Sizes are the repository's model (vocabulary 151936, 48 layers, 32 query heads and 4
key-value heads of 128) and generic ones around it.  With `own` false the operators run in their plain form, torch
operations in 32 bits (the selection's in 64, as candidates of different beams may lie that near); with it true, in the
library.
"""
import ctypes
import math
import os
import sys

import torch

own = False

VOCAB = 151936  # the 48-layer model's head
HEADS = {"nq": 32, "nkv": 4, "hd": 128}  # its attention
LAYERS = 48
KINDS = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (4, torch.bfloat16), "e4m3": (5, torch.float8_e4m3fn)}


def listed():
    return [
        # one user's search: latency
        {"name": "select_one", "kind": "select", "groups": 1, "beams": 4, "vocab": VOCAB, "ended": 0.0, "masked": 0.0, "weighted": False},
        # a server's searches, some beams ended, banned tokens, a length penalty
        {"name": "select_batch", "kind": "select", "groups": 24, "beams": 8, "vocab": VOCAB, "ended": 0.1, "masked": 0.05, "weighted": True},
        # the tables of eight searches between two steps
        {"name": "fork_step", "kind": "fork", "groups": 8, "beams": 8, "page": 16, "width": 160, "shared": 64, "most": 64, "ended": 0.0},
        # a large server: searches and single requests, some of which ended
        {"name": "fork_server", "kind": "fork", "groups": 128, "beams": 8, "page": 16, "width": 512, "shared": 256, "most": 256, "ended": 0.03},
        # one page of every layer, in the model's own cache type: latency
        {"name": "copy_one", "kind": "copy", "type": "f32", "layers": LAYERS, "copies": 1, "page": 16, "order": "head", **HEADS},
        # the pages that eight searches of eight beams copy in a step
        {"name": "copy_step", "kind": "copy", "type": "bf16", "layers": LAYERS, "copies": 40, "page": 16, "order": "head", **HEADS},
        # the rows of a few searches
        {"name": "share_beams", "kind": "share", "groups": 8, "rows": 8, "ragged": 0, "plo": 256, "phi": 2048, "slo": 1, "shi": 256, "page": 16, "pad": 0, "empty": False, **HEADS},
        # a large batch of answers, sixteen to a prompt
        {"name": "share_wide", "kind": "share", "groups": 48, "rows": 16, "ragged": 5, "plo": 500, "phi": 8000, "slo": 0, "shi": 1500, "page": 16, "pad": 3, "empty": True, **HEADS},
        # one search over a short prompt, in the model's own cache type: latency
        {"name": "attn_beams_one", "kind": "attn", "type": "f32", "groups": 1, "rows": 4, "ragged": 0, "plo": 500, "phi": 600, "slo": 1, "shi": 64, "page": 16, "order": "head", "pad": 0, "empty": False, **HEADS},
        # eight searches of eight beams
        {"name": "attn_beams", "kind": "attn", "type": "bf16", "groups": 8, "rows": 8, "ragged": 0, "plo": 256, "phi": 2048, "slo": 1, "shi": 256, "page": 16, "order": "head", "pad": 0, "empty": False, **HEADS},
        # a batch of answers over one long document, 8-bit cache
        {"name": "attn_document", "kind": "attn", "type": "e4m3", "groups": 1, "rows": 64, "ragged": 0, "plo": 16000, "phi": 16384, "slo": 32, "shi": 1024, "page": 64, "order": "head", "pad": 0, "empty": False, **HEADS},
        # no power of two anywhere, groups of several sizes, rows of no request and one with nothing in its cache
        {"name": "attn_odd", "kind": "attn", "type": "f16", "groups": 5, "rows": 11, "ragged": 9, "plo": 0, "phi": 3500, "slo": 0, "shi": 700, "page": 24, "order": "slot", "pad": 2, "empty": True, "nq": 15, "nkv": 3, "hd": 80},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        most = [work(c) for c in listed() if c["kind"] == case["kind"]]
        if all(work(case)[m] <= max(w[m] for w in most) for m in ("bytes", "flops")):
            return case


def _draw(rng):
    kind = rng.choice(["select", "select", "fork", "copy", "share", "attn", "attn", "attn"])
    page = rng.choice([8, 16, 16, 20, 32, 64, 100, 128, 256])
    if kind == "select":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32, 64]), _log(rng, 50, 200000)
        groups = _log(rng, 1, max(1, min(300, int(24 * 8 * VOCAB / (beams * vocab)))))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "ended": rng.choice([0.0, 0.2]), "masked": rng.choice([0.0, 0.1, 0.9]), "weighted": rng.random() < 0.5}
    if kind == "fork":
        beams = rng.choice([1, 2, 4, 5, 8, 16])
        width = rng.randint(20, 512)
        return {"kind": kind, "groups": _log(rng, 1, 1024 // beams), "beams": beams, "page": page, "width": width, "shared": rng.randint(0, width // 2), "most": rng.randint(1, width // 2),
                "ended": rng.choice([0.0, 0.05])}
    nkv = rng.choice([1, 2, 3, 4, 8])
    heads = {"nq": nkv * rng.choice([1, 2, 3, 4, 6, 8, 16]), "nkv": nkv, "hd": 16 * rng.randint(2, 16) if rng.random() < 0.4 else rng.choice([64, 128, 128, 256])}
    form = {"type": rng.choice(list(KINDS)), "page": page, "order": rng.choice(["slot", "head"]), **heads}
    if kind == "copy":
        row = page * nkv * heads["hd"] * 2 * (4 if form["type"] == "f32" else 2)
        layers = rng.randint(1, LAYERS)
        return {"kind": kind, **form, "layers": layers, "copies": _log(rng, 1, max(1, min(64, int(64e6 / (row * layers)))))}
    groups, rows = _log(rng, 1, 64), _log(rng, 1, 64)
    batch = {"groups": groups, "rows": rows, "ragged": rng.randint(0, rows - 1), "page": page, "pad": rng.randint(0, 2) if groups * rows > 8 and rows > 2 else 0, "empty": rng.random() < 0.3}
    if kind == "share":
        room = min(8000, int(48 * 16 * 8000 / (groups * rows)))
        batch["page"] = rng.choice([8, 16, 20, 32])
        phi, shi = _log(rng, 40 * batch["page"], room), _log(rng, 1, max(1, room // 4))
        return {"kind": kind, **batch, **heads, "plo": rng.randint(0, phi // 2), "phi": phi, "slo": rng.randint(0, shi), "shi": shi}
    # positions of all rows, by what a gathered copy of them takes, and the products on them
    room = min(16384, int(1.1e9 / (groups * rows * nkv * heads["hd"] * 4)), int(3e11 / (groups * rows * heads["nq"] * heads["hd"] * 4)))
    phi = _log(rng, 1, max(2, room))
    shi = _log(rng, 1, max(2, min(1024, room // 4)))
    return {"kind": kind, **batch, **form, "plo": rng.randint(0, phi), "phi": phi, "slo": rng.randint(0, shi), "shi": shi}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _ints(gen, lo, hi, *shape):
    """whole numbers lo .. hi"""
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda")


def _new(*shape):
    return torch.zeros(shape, device="cuda", dtype=torch.int32)


def _normed(x):
    return x * x.square().mean(-1, keepdim=True).add(1e-6).rsqrt()


# ---- inputs


def _prepare_select(gen, case):
    g, b, v = case["groups"], case["beams"], case["vocab"]
    n = g * b
    logits = 2.5 * _normal(gen, n, v)
    if case["masked"]:
        logits[_uniform(gen, n, v) < case["masked"]] = -math.inf  # tokens that a grammar or a list of banned words forbids
    score = -20 - 3 * _normal(gen, n).abs()
    if b > 1:
        score[b // 2::b] = torch.where(_uniform(gen, g) < 0.2, -math.inf, score[b // 2::b])  # beams that no candidate took
    done = (_uniform(gen, n) < case["ended"]).int()
    weight = 1 / _ints(gen, 5, 60, n).float().pow(0.6) if case["weighted"] else None
    s = {"logits": logits, "score": score, "done": done, "weight": weight, "parent": _new(n), "token": _new(n), "score_out": torch.zeros(n, device="cuda"),
         "done_out": _new(n), "fresh": _new(n), "eos": 2, "pad": 0}
    if own:
        s["work"] = torch.empty(_library().lib().moe_beam_select_work_bytes(g, b, v), device="cuda", dtype=torch.uint8)
    return s


def _prepare_fork(gen, case):
    b, page, width = case["beams"], case["page"], case["width"]
    n = case["groups"] * b
    group = torch.arange(n, device="cuda") // b
    shared = _ints(gen, 0, case["shared"], case["groups"])
    mine = _ints(gen, 0, case["most"], n)
    used = shared[group] + mine
    held = torch.where(mine > 0, used * page - _ints(gen, 0, page - 1, n), used * page)  # a page that beams share is full
    pages = case["groups"] * case["shared"] + n * (case["most"] + 1) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    col = torch.arange(width, device="cuda")
    s0, m0 = torch.cumsum(shared, 0) - shared, torch.cumsum(mine, 0) - mine + shared.sum()
    at = torch.where(col < shared[group][:, None], s0[group][:, None] + col, m0[:, None] + col - shared[group][:, None])
    tables = torch.where(col < used[:, None], order[at.clamp(0, pages - 1)], -1)
    left = order[int(shared.sum() + mine.sum()):]
    at0 = int(_ints(gen, 0, pages - 1, 1))
    ring = torch.randint(0, pages, (pages,), generator=gen, device="cuda", dtype=torch.int32)
    ring[(at0 + torch.arange(left.numel(), device="cuda")) % pages] = left
    # the better half of a group goes on more often
    parent = group * b + torch.minimum(_ints(gen, 0, b - 1, n), _ints(gen, 0, b - 1, n))
    parent = torch.where(_uniform(gen, n) < case["ended"], -1, parent)
    s = {"parent": parent.int(), "held": held.int(), "tables": tables.int(), "ring": ring, "ring_at": torch.tensor([at0, left.numel()], device="cuda", dtype=torch.int32),
         "held_out": _new(n), "tables_out": tables.int().clone(), "ring_at_out": _new(2), "copies": _new(n, 3), "status": _new(1)}
    if own:
        s["work"] = torch.empty(_library().lib().moe_paged_fork_work_bytes(n, width, pages), device="cuda", dtype=torch.uint8)
    return s


def _pool(gen, case, sides, n_pages):
    """`sides` pools of pages as [side, page, slot, head, dim], whatever their order in memory."""
    _, dtype = KINDS[case["type"]]
    dims = (sides, n_pages, case["page"], case["nkv"], case["hd"])
    if case["order"] == "head":
        dims = (sides, n_pages, dims[3], dims[2], dims[4])
    pool = torch.empty(dims, device="cuda", dtype=dtype)
    view = pool if case["order"] == "slot" else pool.transpose(2, 3)
    for i in range(sides):
        for p in range(0, n_pages, 4096):
            view[i, p:p + 4096].copy_(_normal(gen, *view[i, p:p + 4096].shape) * (60 if case["type"] == "e4m3" else 1))
    return view


def _prepare_copy(gen, case):
    n, page = case["copies"], case["page"]
    pool = _pool(gen, case, 2 * case["layers"], 3 * n + 4)
    to = 2 * n + 4 + torch.randperm(n, generator=gen, device="cuda")
    copies = torch.stack([_ints(gen, 0, 2 * n + 3, n), to, _ints(gen, 1, page, n)], 1)
    copies = torch.cat([copies, torch.full((2, 3), -1, device="cuda")]).int()  # a list of fixed length, not full
    return {"pool": pool, "copies": copies}


def _batch(gen, case):
    """Rows in groups whose requests begin in the same pages."""
    page = case["page"]
    sizes = [max(1, case["rows"] - i * 5 % (case["ragged"] + 1)) for i in range(case["groups"])]
    first = torch.tensor([0] + sizes, device="cuda").cumsum(0)
    T = int(first[-1])
    group = torch.repeat_interleave(torch.arange(case["groups"], device="cuda"), torch.tensor(sizes, device="cuda"))
    shared = _ints(gen, case["plo"], case["phi"], case["groups"]) // page
    mine = _ints(gen, case["slo"], case["shi"], T)
    pos = shared[group] * page + mine - 1
    if case["empty"]:
        pos[T // 2] = -1  # a request with nothing in its cache yet
    own_pages = (mine + page - 1) // page
    width = case["phi"] // page + -(-case["shi"] // page) + 2
    total = int(shared.sum() + own_pages.sum())
    n_pages = total + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda")
    col = torch.arange(width, device="cuda")
    s0, m0 = torch.cumsum(shared, 0) - shared, torch.cumsum(own_pages, 0) - own_pages + shared.sum()
    sh = shared[group][:, None]
    at = torch.where(col < sh, s0[group][:, None] + col, m0[:, None] + col - sh)
    tables = torch.where(col < sh + own_pages[:, None], order[at.clamp(0, n_pages - 1)], -1).int()
    req = torch.arange(T, device="cuda", dtype=torch.int32)
    if case["pad"]:
        req[T - case["pad"]:] = -1  # rows of a fixed batch that no request fills
    return T, n_pages, {"first": first.int(), "req": req, "pos": pos.int(), "tables": tables, "prefix": _new(case["groups"])}


def _share_args(M, s, T):
    case, p = s["case"], {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    return M.PagedShare(T, T, s["tables"].shape[1], case["page"], case["nq"], case["nkv"], case["hd"], p["req"], p["pos"], p["tables"], case["groups"], p["first"], p["prefix"],
                        p["plan"], s["plan"].numel())


def _prepare_share(gen, case):
    T, _, s = _batch(gen, case)
    s["T"] = T
    if own:
        s["plan"] = torch.empty(_library().lib().moe_paged_share_plan_bytes(T, case["groups"], case["nq"], case["nkv"], case["hd"]), device="cuda", dtype=torch.uint8)
    return s


def _prepare_attn(gen, case):
    T, n_pages, s = _batch(gen, case)
    pool = _pool(gen, case, 2, n_pages)
    scale = 0.01 + 0.01 * _uniform(gen, 2, case["nkv"]) if case["type"] == "e4m3" else None
    s.update({"T": T, "case": case, "k": pool[0], "v": pool[1], "scale": scale, "q": _normed(_normal(gen, T, case["nq"], case["hd"])).reshape(T, -1),
              "out": _normal(gen, T, case["nq"] * case["hd"])})
    if own:
        # one plan a step, which all layers' calls read
        M = _library()
        sizes = (T, case["groups"], case["nq"], case["nkv"], case["hd"])
        s["plan"] = torch.empty(M.lib().moe_paged_share_plan_bytes(*sizes), device="cuda", dtype=torch.uint8)
        s["work"] = torch.empty(M.lib().moe_paged_attn_shared_work_bytes(*sizes), device="cuda", dtype=torch.uint8)
        torch.cuda.synchronize()
        M.check(M.lib().moe_paged_share_dev(ctypes.byref(_share_args(M, s, T))), "share")
        M.synchronize()
    return s


def prepare(case, seed):
    make = {"select": _prepare_select, "fork": _prepare_fork, "copy": _prepare_copy, "share": _prepare_share, "attn": _prepare_attn}
    state = make[case["kind"]](_gen(seed), case)
    state["case"] = case
    torch.cuda.synchronize()  # the library works on a stream of its own
    return state


# ---- the plain forms


def _plain_select(s):
    case = s["case"]
    g, b, v = case["groups"], case["beams"], case["vocab"]
    x = s["logits"].double()
    score, weight = s["score"].double(), torch.ones_like(s["score"]).double() if s["weight"] is None else s["weight"].double()
    top = x.amax(-1, keepdim=True)
    lse = top[:, 0] + (x - top).exp().sum(-1).log()
    lives = score.isfinite() & weight.isfinite() & (weight > 0)
    ended = lives & (s["done"] != 0)
    lives &= (s["done"] == 0) & lse.isfinite()
    # a beam's own order: by logit, then by token, as one whole number
    bits = (s["logits"] + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    take = min(b, v)
    token = (order * (1 << 32) + (v - 1 - torch.arange(v, device="cuda"))).topk(take, -1).indices
    at = x.gather(-1, token)
    value = torch.where(lives[:, None] & (at > -math.inf), (score - lse)[:, None] + at, -math.inf)
    value[:, 0] = torch.where(ended, score, value[:, 0])
    token = torch.where(ended[:, None], s["pad"], token)
    value = value.reshape(g, -1)
    rank = torch.where(value > -math.inf, value * weight.repeat_interleave(take).reshape(g, -1), -math.inf)
    if take < b:
        value, rank = (torch.nn.functional.pad(t, (0, b), value=-math.inf) for t in (value, rank))
    best = rank.sort(dim=-1, descending=True, stable=True).indices[:, :b]
    value = value.gather(-1, best)
    none = value == -math.inf
    best = torch.where(none, 0, best)
    parent = torch.where(none, -1, best // take + torch.arange(g, device="cuda")[:, None] * b).reshape(-1)
    token = torch.where(none, -1, token.reshape(g, -1).gather(-1, best)).reshape(-1)
    was = (s["done"] != 0)[parent.clamp(min=0)] & (parent >= 0)
    done = (was | ((token == s["eos"]) & (parent >= 0))).int()
    return {"parent": parent.int(), "token": token.int(), "score": value.reshape(-1).float(), "done": done, "fresh": ((parent >= 0) & (done == 0)).int()}


def _plain_fork(s):
    case = s["case"]
    page, width = case["page"], case["width"]
    parent, held, n_pages = s["parent"].long(), s["held"].long(), s["ring"].numel()
    n = parent.numel()
    head, count = s["ring_at"].long()
    r = torch.arange(n, device="cuda")
    live, src = parent >= 0, parent.clamp(min=0)
    used = (held + page - 1) // page
    keeps = torch.where(parent == r, r, torch.full_like(r, n).scatter_reduce(0, src, torch.where(live, r, n), "amin"))
    copied = live & (held % page != 0)[src] & (keeps[src] != r)
    taken = torch.cumsum(copied.long(), 0) - copied.long()
    need = copied.sum()
    # how each request goes on, page by page
    col = torch.arange(width, device="cuda")
    fills = live[:, None] & (col < used[src][:, None])
    last = copied[:, None] & (col == used[src][:, None] - 1)
    fresh = s["ring"][(head + taken) % n_pages].long()
    old = s["tables"].long()
    new = torch.where(last, fresh[:, None], old[src])
    # pages that no request holds any more, each once, column by column
    held_page = (col < used[:, None]) & (old >= 0) & (old < n_pages)
    stays = torch.zeros(n_pages + 1, device="cuda", dtype=torch.bool)
    stays[torch.where(fills & ~last & (new >= 0) & (new < n_pages), new, n_pages)] = True
    place = (col * n + r[:, None]).expand(n, width)
    firsts = torch.full((n_pages + 1,), n * width, device="cuda").scatter_reduce(0, torch.where(held_page, old, n_pages).reshape(-1), place.reshape(-1), "amin")
    out = (held_page & ~stays[old.clamp(0, n_pages)] & (firsts[old.clamp(0, n_pages)] == place)).T
    back = out.sum()
    status = torch.where((parent < -1).any() | (parent >= n).any() | (held < 0).any() | (held > width * page).any() | (count + back - need > n_pages), 4, torch.where(
        need > s["copies"].shape[0], 2, torch.where(need > count, 1, 0)))
    ok = status == 0
    to = torch.where(out.reshape(-1) & ok, (head + count + torch.cumsum(out.reshape(-1).long(), 0) - 1) % n_pages, n_pages)
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring[to] = s["tables"].T.reshape(-1)
    s["ring"].copy_(ring[:n_pages])
    copies = torch.full((n + 1, 3), -1, device="cuda", dtype=torch.int64)
    tail = (used[src] - 1).clamp(min=0)
    copies[torch.where(copied & ok, taken, n)] = torch.stack([old[src, tail], fresh, held[src] - tail * page], 1)
    return {"tables": torch.where(fills & ok, new, old).int(), "held": torch.where(ok, torch.where(live, held[src], 0), held).int(), "ring": s["ring"],
            "ring_at": torch.stack([(head + need * ok) % n_pages, count + (back - need) * ok]).int(), "copies": copies[:n].int(), "status": status.int().reshape(1)}


def _bytes(pool):
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def _plain_copy(s):
    pool, copies = _bytes(s["pool"]), s["copies"].long()
    live = copies[:, 0] >= 0
    copies = copies[live]
    part = (torch.arange(pool.shape[2], device="cuda") < copies[:, 2:])[:, :, None, None]
    pool[:, copies[:, 1]] = torch.where(part, pool[:, copies[:, 0]], pool[:, copies[:, 1]])
    return s["pool"]


def _plain_share(s):
    page, T = s["case"]["page"], s["T"]
    tables, first = s["tables"], s["first"].long()
    r = torch.arange(T, device="cuda")
    group = torch.searchsorted(first[1:].contiguous(), r, right=True)
    full = torch.where(s["req"] >= 0, (s["pos"].long() + 1).clamp(min=0) // page, 0)
    live = (s["req"] >= 0) & (s["pos"] >= 0)
    lead = torch.full((s["case"]["groups"],), T, device="cuda").scatter_reduce(0, group, torch.where(live, r, T), "amin").clamp(max=T - 1)
    mine = tables[s["req"].clamp(min=0).long()]
    other = mine[lead][group]
    same = torch.cumprod((mine == other).long(), 1).sum(1)
    both = torch.where(live, torch.minimum(same, full), 1 << 30)
    least = torch.full((s["case"]["groups"],), 1 << 30, device="cuda").scatter_reduce(0, group, both, "amin")
    return torch.where(least == 1 << 30, 0, least * page).int()


def _values(pool, pages, scale):
    """the numbers that pages of a pool stand for, [..., slot, head, dim]"""
    x = _bytes(pool)[pages].view(pool.dtype).float()
    return x if scale is None else x * scale[:, None]


def _plain_attn(s):
    case = s["case"]
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    out, scale = s["out"].clone(), s["scale"]
    ks, vs = (None, None) if scale is None else scale
    ends = [0]
    for i in range(case["groups"]):
        ends.append(ends[-1] + max(1, case["rows"] - i * 5 % (case["ragged"] + 1)))
        a, b = ends[-2:]
        rows = slice(a, b)
        pages = s["tables"][s["req"][rows].clamp(min=0).long()].clamp(min=0).long()
        seen = torch.arange(pages.shape[1] * page, device="cuda") <= s["pos"][rows, None]
        k = _values(s["k"], pages, ks).reshape(b - a, -1, nkv, hd)
        q = s["q"][rows].reshape(b - a, nkv, -1, hd)
        x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1 / math.sqrt(hd))
        del k
        x = x.masked_fill(~seen[:, None, None], -math.inf)
        top = x.amax(-1, keepdim=True)
        p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
        total = p.sum(-1, keepdim=True)
        v = _values(s["v"], pages, vs).reshape(b - a, -1, nkv, hd)
        v = torch.where(seen[:, :, None, None], v, 0.0).transpose(1, 2).contiguous()
        o = torch.matmul(p / torch.where(total == 0, 1.0, total), v).reshape(b - a, -1)
        out[rows] = torch.where(s["req"][rows, None] < 0, s["out"][rows], o)
    return out


# ---- the library's calls


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe.cc_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import moehip
    return moehip


def _pages(M, case, k, v, scale):
    return M.Pages(k.data_ptr(), v.data_ptr(), KINDS[case["type"]][0], k.shape[0], case["page"], case["nkv"], case["hd"], k.stride(0), k.stride(2), k.stride(1),
                   *([None, None] if scale is None else [scale[0].data_ptr(), scale[1].data_ptr()]))


def _call(s):
    """The descriptors that a program fills once for its buffers: (check, entry point, arguments)."""
    M, case = _library(), s["case"]
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    L, kind = M.lib(), case["kind"]
    if kind == "select":
        a = M.BeamSelect(case["groups"], case["beams"], case["vocab"], p["logits"], s["logits"].stride(0), p["score"], p["done"], p.get("weight"), s["eos"], s["pad"],
                         p["parent"], p["token"], p["score_out"], p["done_out"], p["fresh"], p["work"], s["work"].numel())
        return M.check, L.moe_beam_select_dev, [ctypes.byref(a)]
    if kind == "fork":
        n = s["parent"].numel()
        a = M.PagedFork(n, case["width"], s["ring"].numel(), case["page"], n, p["parent"], p["held"], p["ring_at"], p["ring"], p["tables"], p["held_out"], p["ring_at_out"],
                        p["tables_out"], p["copies"], p["status"], p["work"], s["work"].numel())
        return M.check, L.moe_paged_fork_dev, [ctypes.byref(a)]
    if kind == "copy":
        layers = (M.Pages * case["layers"])(*[_pages(M, case, s["pool"][2 * i], s["pool"][2 * i + 1], None) for i in range(case["layers"])])
        return M.check, L.moe_paged_copy_dev, [p["copies"], s["copies"].shape[0], layers, case["layers"]]
    share = _share_args(M, s, s["T"])
    if kind == "share":
        return M.check, L.moe_paged_share_dev, [ctypes.byref(share)]
    a = M.PagedAttn(p["q"], s["q"].stride(0), s["T"], case["nq"], p["req"], p["pos"], p["tables"], s["T"], s["tables"].shape[1], 1 / math.sqrt(case["hd"]),
                    p["out"], s["out"].stride(0), p["work"], s["work"].numel())
    return M.check, L.moe_paged_attn_shared_dev, [ctypes.byref(a), ctypes.byref(_pages(M, case, s["k"], s["v"], s["scale"])), ctypes.byref(share)]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"select": _plain_select, "fork": _plain_fork, "copy": _plain_copy, "share": _plain_share, "attn": _plain_attn}[kind](state)
    if "call" not in state:
        state["call"] = _call(state)
    check, entry, args = state["call"]
    check(entry(*args), kind)
    if kind == "select":
        return {"parent": state["parent"], "token": state["token"], "score": state["score_out"], "done": state["done_out"], "fresh": state["fresh"]}
    if kind == "fork":
        return {"tables": state["tables_out"], "held": state["held_out"], "ring": state["ring"], "ring_at": state["ring_at_out"], "copies": state["copies"], "status": state["status"]}
    return state[{"copy": "pool", "share": "prefix", "attn": "out"}[kind]]


def _sizes(case):
    return [max(1, case["rows"] - i * 5 % (case["ragged"] + 1)) for i in range(case["groups"])]


def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["groups"] * case["beams"] * (1 - case["ended"])
        return {"bytes": 4 * rows * case["vocab"] + 36 * case["groups"] * case["beams"], "flops": 6 * rows * case["vocab"]}
    if kind == "fork":
        # every entry read, as any may be a page's last holder; about two thirds of the rows written anew
        n = case["groups"] * case["beams"]
        entries = n * (case["shared"] + case["most"]) / 2
        return {"bytes": 4 * (entries * (2 if case["beams"] > 1 else 1) + 6 * n), "flops": entries}
    size = 4 if case.get("type") == "f32" else 1 if case.get("type") == "e4m3" else 2
    if kind == "copy":
        moved = case["copies"] * (case["page"] + 1) / 2 * case["nkv"] * case["hd"] * size * 2 * case["layers"]
        return {"bytes": 2 * moved + 12 * (case["copies"] + 2), "flops": 0}
    T = sum(_sizes(case))
    shared, mine = (case["plo"] + case["phi"]) / 2, (case["slo"] + case["shi"]) / 2
    if kind == "share":
        return {"bytes": 4 * (T * shared / case["page"] + 2 * T + 2 * case["groups"]), "flops": T * shared / case["page"]}
    T -= case["pad"]
    kept = case["groups"] * shared + T * mine
    return {"bytes": kept * case["nkv"] * case["hd"] * 2 * size + 8 * T * case["nq"] * case["hd"] + 4 * kept / case["page"], "flops": 4 * T * (shared + mine) * case["nq"] * case["hd"]}


# ---- the definitions in 64 bits


def _exact_select(s):
    case = s["case"]
    g, b = case["groups"], case["beams"]
    logp = torch.log_softmax(s["logits"].double(), -1)
    out = torch.full((g, b), -math.inf, device="cuda", dtype=torch.float64)
    weight = torch.ones(g * b, device="cuda") if s["weight"] is None else s["weight"]
    for i in range(g):
        found = []
        for r in range(i * b, i * b + b):
            if not math.isfinite(float(s["score"][r])):
                continue
            v = s["score"][r].double() + (torch.sort(logp[r], descending=True).values[:b] if s["done"][r] == 0 else torch.zeros(1, device="cuda", dtype=torch.float64))
            found.append(torch.stack([v * weight[r].double(), v]))
        if found:
            found = torch.cat(found, 1)
            found = found[:, found[0].sort(dim=-1, descending=True, stable=True).indices[:b]]
            out[i, :found.shape[1]] = found[1]
    return {"parent": None, "token": None, "score": out.reshape(-1), "done": None, "fresh": None}


def _exact_copy(s):
    pool = _bytes(s["pool"]).clone()
    for src, dst, n in s["copies"].tolist():
        if src >= 0:
            pool[:, dst, :n] = pool[:, src, :n]
    return pool.view(s["pool"].dtype).double()


def _exact_attn(s):
    case = s["case"]
    out, g = s["out"].double(), case["nq"] // case["nkv"]
    for t in range(s["T"]):
        if int(s["req"][t]) < 0:
            continue
        n = int(s["pos"][t]) + 1
        out[t] = 0
        if n == 0:
            continue
        pages = s["tables"][int(s["req"][t]), :-(-n // case["page"])].long()
        k, v = (_bytes(s[m])[pages].view(s[m].dtype).flatten(0, 1)[:n].double() for m in "kv")
        if s["scale"] is not None:
            k, v = k * s["scale"][0].double()[:, None], v * s["scale"][1].double()[:, None]
        q = s["q"][t].double().reshape(case["nkv"], g, case["hd"])
        for h in range(case["nkv"]):
            p = torch.softmax(q[h] @ k[:, h].T / math.sqrt(case["hd"]), -1)
            out[t, h * g * case["hd"]:(h + 1) * g * case["hd"]] = (p @ v[:, h]).reshape(-1)
    return out


def exact(case, seed):
    if case["kind"] in ("fork", "share"):
        return None  # whole numbers
    state = prepare(case, seed)
    return {"select": _exact_select, "copy": _exact_copy, "attn": _exact_attn}[case["kind"]](state)
