"""Plain forms of the beam-search operators over the paged cache, for the tests
of moe_beam_select_dev, moe_paged_fork_dev, moe_paged_copy_dev and
moe_paged_share_dev."""
import numpy as np

OK, NO_PAGES, TOO_MANY, BAD = 0, 1, 2, 4


def fork(parent, held, tables, ring, ring_at, page_size, max_copies):
    """One call on host arrays -> dict of what it leaves (tables, held, ring, ring_at, copies, status)."""
    parent, held = np.asarray(parent), np.asarray(held)
    n, width = tables.shape
    n_pages = ring.size
    head, count = (int(x) for x in ring_at)
    same = dict(tables=tables.copy(), held=held.copy(), ring=ring.copy(), ring_at=np.array([head, count], np.int32),
                copies=np.full((max_copies, 3), -1, np.int32))
    if ((parent < -1) | (parent >= n) | (held < 0) | (held > width * page_size)).any() or not 0 <= head < n_pages or not 0 <= count <= n_pages:
        return dict(same, status=BAD)
    used = -(-held // page_size)
    keeper = {}
    for r in range(n):
        s = int(parent[r])
        if s >= 0 and (s not in keeper or r == s):
            keeper[s] = r
    copies, new = [], tables.copy()
    for r in range(n):
        s = int(parent[r])
        if s < 0:
            continue
        new[r, :used[s]] = tables[s, :used[s]]
        if held[s] % page_size and keeper[s] != r:
            dst = int(ring[(head + len(copies)) % n_pages])
            copies.append((int(tables[s, used[s] - 1]), dst, int(held[s] - (used[s] - 1) * page_size)))
            new[r, used[s] - 1] = dst
    good = lambda p: 0 <= p < n_pages  # noqa: E731
    stays = set()
    for r in range(n):
        s = int(parent[r])
        if s >= 0:
            copied = held[s] % page_size and keeper[s] != r
            stays.update(int(p) for p in tables[s, :used[s] - (1 if copied else 0)])
    back = []
    for c in range(width):
        for r in range(n):
            p = int(tables[r, c])
            if c < used[r] and good(p) and p not in stays and p not in back:
                back.append(p)
    if count + len(back) > n_pages:
        return dict(same, status=BAD)
    if len(copies) > max_copies:
        return dict(same, status=TOO_MANY)
    if len(copies) > count:
        return dict(same, status=NO_PAGES)
    out = dict(same, tables=new, status=OK)
    for i, p in enumerate(back):
        out["ring"][(head + count + i) % n_pages] = p
    out["held"] = np.array([held[s] if s >= 0 else 0 for s in parent], np.int32)
    out["ring_at"] = np.array([(head + len(copies)) % n_pages, count + len(back) - len(copies)], np.int32)
    if copies:
        out["copies"][:len(copies)] = copies
    return out


def select(logits, score, done, weight, n_beam, eos, pad):
    """-> dict(parent, token, score, done, fresh, rank, values): new rows, and every row's log probabilities, in 64 bits"""
    rows, vocab = logits.shape
    weight = np.ones(rows) if weight is None else np.asarray(weight, np.float64)
    x = logits.astype(np.float64)
    values = np.full((rows, vocab), -np.inf)
    out = {n: np.full(rows, -1, np.int32) for n in ("parent", "token")}
    out.update(score=np.full(rows, -np.inf), rank=np.full(rows, -np.inf), done=np.zeros(rows, np.int32), fresh=np.zeros(rows, np.int32))
    for g0 in range(0, rows, n_beam):
        found = []   # (-rank, row, order in the row, token, value)
        for r in range(g0, g0 + n_beam):
            if not np.isfinite(score[r]) or not (0 < weight[r] < np.inf):
                continue
            if done[r]:
                found.append((-(float(score[r]) * weight[r]), r, 0, pad, float(score[r])))
                continue
            if np.isnan(x[r]).any() or (x[r] == np.inf).any() or (x[r] == -np.inf).all():
                continue
            top = x[r].max()
            values[r] = float(score[r]) - (top + np.log(np.exp(x[r] - top).sum())) + x[r]
            best = np.argsort(-x[r], kind="stable")[:n_beam]
            found += [(-(values[r, v] * weight[r]), r, i, int(v), values[r, v]) for i, v in enumerate(best) if x[r, v] > -np.inf]
        for i, (rank, r, _, token, value) in enumerate(sorted(found)[:n_beam]):
            out["parent"][g0 + i], out["token"][g0 + i], out["score"][g0 + i], out["rank"][g0 + i] = r, token, value, -rank
            out["done"][g0 + i] = int(bool(done[r]) or token == eos)
            out["fresh"][g0 + i] = 1 - out["done"][g0 + i]
    return dict(out, values=values)


def share(req, pos, tables, first, page_size):
    """-> prefix of each group"""
    n_req, width = tables.shape
    T = len(pos)
    req = np.arange(T) if req is None else np.asarray(req)
    first = [int(f) for f in first]
    prefix = np.zeros(len(first) - 1, np.int32)
    if any(a > b for a, b in zip(first, first[1:])) or first[0] < 0 or first[-1] > T:
        return prefix
    for g, (a, b) in enumerate(zip(first, first[1:])):
        live = [t for t in range(a, b) if 0 <= req[t] < n_req and 0 <= pos[t] < width * page_size]
        if live:
            lead = tables[req[live[0]]]
            least = width
            for t in live:
                full = (int(pos[t]) + 1) // page_size
                differ = np.nonzero(tables[req[t], :full] != lead[:full])[0]
                least = min(least, int(differ[0]) if differ.size else full)
            prefix[g] = least * page_size
    return prefix
