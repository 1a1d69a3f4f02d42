"""moe_paged_attn_dev against a 64-bit evaluation on the values that the pages hold; the bound on an fp32 evaluation
is derived in paged_cases.attend.  Every slot that no position fills holds a NaN or an infinity."""
import numpy as np
import pytest

import paged_cases as C

pytestmark = pytest.mark.gpu

ARG = 2


class Batch:
    """Requests of given lengths on pages in no order, queries, and the call."""

    def __init__(self, M, dtype, lens, nq, nkv, hd, ps, order="slot", seed=0, ld_extra=0, spare=2, gain=1.0):
        self.M, self.lens, self.nq, self.hd, self.ps = M, lens, nq, hd, ps
        rng = np.random.default_rng(1000 + seed)
        scales = [0.01 + 0.02 * rng.random(nkv) for _ in "kv"] if dtype == C.E4M3 else [None, None]
        used = [-(-n // ps) for n in lens]
        self.width = max(max(used), 1) + 1
        n_pages = sum(used) + spare
        self.pool = C.Pool(M, dtype, n_pages, ps, nkv, hd, order, *scales)
        order_of = rng.permutation(n_pages)
        self.tables = np.full((len(lens), self.width), -7, np.int32)
        at = 0
        for r, n in enumerate(lens):
            self.tables[r, :used[r]] = order_of[at:at + used[r]]
            at += used[r]
            if n:
                p = np.arange(n)
                k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) * g for g in (gain, 1.0))
                slot = (self.tables[r][p // ps], p % ps)
                for side, (pool, x) in enumerate(((self.pool.k, k), (self.pool.v, v))):
                    pool[slot] = C.encode((x / self.pool.factor(side)).astype(np.float32), dtype)
        self.pool.upload()
        self.scale = float(np.float32(1 / np.sqrt(hd)))
        self.rng, self.ld = rng, nq * hd + ld_extra

    def run(self, req=None, pos=None, T=None, q=None, work_from=0xA5):
        """-> (out [T, ld], q [T, nq, hd]); out starts as 7s"""
        M = self.M
        T = T or len(self.lens)
        pos = np.asarray(self.lens, np.int32) - 1 if pos is None else np.asarray(pos, np.int32)
        if q is None:
            q = self.rng.standard_normal((T, self.ld)).astype(np.float32)
        out = np.full((T, self.ld), 7.0, np.float32)
        need = M.lib().moe_paged_attn_work_bytes(T, self.nq, self.pool.n_kv, self.hd)
        bufs = [M.DeviceBuffer.from_array(x) for x in (q, pos, self.tables, out)]
        rq = None if req is None else M.DeviceBuffer.from_array(np.asarray(req, np.int32))
        work = M.DeviceBuffer.from_array(np.full(need, work_from, np.uint8))
        a = M.PagedAttn(bufs[0].ptr, self.ld, T, self.nq, None if rq is None else rq.ptr, bufs[1].ptr, bufs[2].ptr, len(self.lens), self.width,
                        self.scale, bufs[3].ptr, self.ld, work.ptr, need)
        M.check(M.lib().moe_paged_attn_dev(C.ref(a), C.ref(self.pool.pages)), "paged_attn")
        return bufs[3].download(out.shape, np.float32), q[:, :self.nq * self.hd].reshape(T, self.nq, self.hd)

    def check(self, out, q, t, r, n):
        k, v = self.pool.rows(self.tables[r], n)
        want, tol = C.attend(q[t].astype(np.float64), k, v, self.scale)
        got = out[t, :self.nq * self.hd].reshape(self.nq, self.hd)
        assert np.isfinite(got).all(), f"row {t} of {n} positions: not finite"
        off = np.abs(got - want) / np.maximum(tol, 1e-30)
        if n == 0:
            assert not got.any()
        else:
            assert off.max() <= 1, f"row {t} of {n} positions: {off.max():.2f} times the bound at {np.unravel_index(off.argmax(), off.shape)}"
        assert (out[t, self.nq * self.hd:] == 7).all()


def _all(b, out, q):
    for t, n in enumerate(b.lens):
        b.check(out, q, t, t, n)


LENS = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("nq,nkv,hd,ps,order", [
    (32, 4, 128, 16, "slot"), (8, 8, 64, 32, "head"), (6, 2, 80, 24, "slot"), (16, 1, 256, 64, "shared"), (40, 2, 128, 7, "head"),
    (3, 3, 16, 1, "slot"), (5, 1, 48, 128, "shared"), (34, 2, 96, 16, "head"), (4, 4, 208, 100, "slot")])
def test_shapes(moehip, kind, nq, nkv, hd, ps, order):
    print("paged attention", kind, nq, nkv, hd, ps, order, flush=True)
    b = Batch(moehip, C.TYPES[kind], LENS, nq, nkv, hd, ps, order, seed=hd + ps, ld_extra=3 if hd == 80 else 0)
    out, q = b.run()
    _all(b, out, q)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("lens", [[5000], [70000], [1] * 300, [3, 40000, 1, 9, 2000, 0, 12], list(range(0, 1100, 4))],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_lengths(moehip, kind, lens):
    print("paged attention lengths", kind, len(lens), max(lens), flush=True)
    b = Batch(moehip, C.TYPES[kind], lens, 8, 2, 64, 32, seed=len(lens))
    out, q = b.run()
    for t in range(0, len(lens), max(1, len(lens) // 40)):
        b.check(out, q, t, t, lens[t])


def test_same_bits_every_time(moehip):
    """The split and its join are fixed by the lengths: the same call gives the same bits."""
    b = Batch(moehip, C.BF16, [9000, 1, 300, 2500], 32, 4, 128, 16, seed=3)
    out, q = b.run()
    for fill in (0, 0xFF):
        again, _ = b.run(q=q.reshape(4, -1), work_from=fill)
        np.testing.assert_array_equal(out.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_of_one_request_and_padding(moehip, kind):
    """A prompt's rows (each sees one position more), rows of other requests between them, rows that no request fills."""
    b = Batch(moehip, C.TYPES[kind], [90, 33], 8, 4, 64, 16, seed=5)
    rows = [(0, p) for p in range(60, 90)] + [(-1, 5), (1, 32), (1, 0), (-1, -1), (0, 0), (0, -1), (-3, 1 << 30)]
    req, pos = zip(*rows)
    out, q = b.run(req=req, pos=pos, T=len(rows))
    for t, (r, p) in enumerate(rows):
        if r < 0:
            assert (out[t] == 7).all(), f"row {t} of no request was written"
        else:
            b.check(out, q, t, r, p + 1)


@pytest.mark.parametrize("kind", ["f32", "e4m3"])
@pytest.mark.parametrize("bad_page", [-1, 10 ** 9, -2 ** 31])
def test_bad_pages_and_places(moehip, kind, bad_page):
    """A table entry that is no page, a request or a position past the tables: that row is NaN, the others are right."""
    lens = [100, 700, 40, 3000, 64]
    b = Batch(moehip, C.TYPES[kind], lens, 8, 2, 64, 16, seed=9)
    b.tables[1, 20] = bad_page
    b.tables[3, 0] = b.pool.n_pages
    b.tables[4, 4:] = bad_page           # behind the last position: never read
    wide = b.width * 16
    req = [0, 1, 2, 3, 4, 5, 2 ** 31 - 1, 0, 0]
    pos = [99, 699, 39, 2999, 63, 3, 3, wide, 2 ** 31 - 1]
    out, q = b.run(req=req, pos=pos, T=9)
    for t in (0, 2, 4):
        b.check(out, q, t, t, lens[t])
    for t in (1, 3, 5, 6, 7, 8):
        assert np.isnan(out[t]).all(), f"row {t}"


@pytest.mark.parametrize("kind", list(C.TYPES))
def test_far_scores(moehip, kind):
    """Scores hundreds apart: the running maximum carries every earlier weight to zero and none overflows."""
    b = Batch(moehip, C.TYPES[kind], [1, 50, 3000, 700], 8, 2, 64, 16, seed=11, gain=40.0 if kind != "e4m3" else 4.0)
    out, q = b.run()
    _all(b, out, q)


@pytest.mark.parametrize("kind", list(C.TYPES))
def test_nan_stays_in_its_heads(moehip, kind):
    """NaN in an attended key or value makes its heads NaN and no others."""
    b = Batch(moehip, C.TYPES[kind], [40, 2000, 40], 4, 2, 64, 16, seed=13)
    k = b.pool.k
    k[b.tables[1, 7], 3, 1, 5] = C.NAN_BITS[C.TYPES[kind]] if kind != "f32" else np.nan
    b.pool.v[b.tables[2, 1], 2, 0, 9] = C.NAN_BITS[C.TYPES[kind]] if kind != "f32" else np.nan
    b.pool.upload()
    out, q = b.run()
    o = out.reshape(3, 4, 64)
    b.check(out, q, 0, 0, 40)
    assert np.isnan(o[1, 2:]).all() and np.isfinite(o[1, :2]).all()
    assert np.isnan(o[2, :2, 9]).all() and np.isfinite(o[2, 2:]).all()


def test_offsets_past_32_bits(moehip):
    """Pages 2^28 elements apart: the last lie past 2^32 bytes and elements."""
    M = moehip
    n_pages, ps, hd, nkv = 18, 16, 64, 2
    stride = 1 << 28
    pool = M.DeviceBuffer(n_pages * stride)
    rng = np.random.default_rng(17)
    table = np.array([[17, 0, 16, 9]], np.int32)
    k, v = (rng.standard_normal((64, nkv, hd)).astype(np.float32) for _ in "kv")
    gap = ps * nkv * hd   # V's rows behind K's in each page
    for i, page in enumerate(table[0]):
        for side, x in enumerate((k, v)):
            pool.upload(C.encode(x[i * ps:(i + 1) * ps], C.E4M3), offset=int(page) * stride + side * gap)
    pages = M.Pages(pool.ptr, pool.ptr + gap, C.E4M3, n_pages, ps, nkv, hd, stride, hd, nkv * hd, None, None)
    q = rng.standard_normal((1, 4 * hd)).astype(np.float32)
    bufs = [M.DeviceBuffer.from_array(x) for x in (q, np.array([59], np.int32), table, np.zeros_like(q))]
    need = M.lib().moe_paged_attn_work_bytes(1, 4, nkv, hd)
    work = M.DeviceBuffer(need)
    a = M.PagedAttn(bufs[0].ptr, 4 * hd, 1, 4, None, bufs[1].ptr, bufs[2].ptr, 1, 4, 0.125, bufs[3].ptr, 4 * hd, work.ptr, need)
    M.check(M.lib().moe_paged_attn_dev(C.ref(a), C.ref(pages)))
    got = bufs[3].download((4, hd), np.float32)
    kd, vd = (C.decode(C.encode(x[:60], C.E4M3), C.E4M3) for x in (k, v))
    want, tol = C.attend(q.reshape(4, hd).astype(np.float64), kd, vd, 0.125)
    assert (np.abs(got - want) <= tol).all()
    pool.free()


@pytest.mark.parametrize("kind,T,nq,nkv,hd,long", [
    ("bf16", 100, 16, 8, 128, 3000), ("f16", 200, 8, 8, 64, 1500), ("e4m3", 256, 4, 4, 128, 2000), ("bf16", 700, 8, 8, 64, 900), ("f32", 300, 4, 2, 256, 600),
    ("bf16", 2048, 4, 4, 64, 400), ("f16", 2049, 4, 2, 64, 300), ("f32", 65, 32, 16, 128, 5000)])
def test_many_rows(moehip, kind, T, nq, nkv, hd, long):
    """More rows than a wave, a block's threads, the pieces, the rows that are cut; few of them long, some empty, some of
    no request, several of one request."""
    print("paged attention rows", kind, T, nq, nkv, hd, flush=True)
    rng = np.random.default_rng(T)
    lens = [int(n) for n in rng.integers(0, 200, 24)] + [long, 0, long // 2, 1]
    b = Batch(moehip, C.TYPES[kind], lens, nq, nkv, hd, 16, "head", seed=T)
    req = rng.integers(0, len(lens), T)
    pos = np.array([rng.integers(-1, lens[r]) if lens[r] else -1 for r in req])
    full = rng.random(T) < 0.2
    pos[full] = np.array(lens)[req[full]] - 1
    req[rng.random(T) < 0.15] = -1
    req[[0, T - 1]] = -1, len(lens) - 4
    pos[T - 1] = long - 1
    out, q = b.run(req=req, pos=pos, T=T)
    again, _ = b.run(req=req, pos=pos, T=T, q=q.reshape(T, -1), work_from=0x3C)
    np.testing.assert_array_equal(out.view(np.uint32), again.view(np.uint32))
    for t in list(range(0, T, max(1, T // 60))) + [T - 1]:
        if req[t] < 0:
            assert (out[t] == 7).all()
        else:
            b.check(out, q, t, int(req[t]), int(pos[t]) + 1)


def test_no_row_of_any_request(moehip):
    b = Batch(moehip, C.BF16, [300, 20], 8, 2, 64, 16, seed=21)
    for T in (1, 40, 100, 400):
        out, _ = b.run(req=[-1] * T, pos=[299] * T, T=T)
        assert (out == 7).all()


def test_two_calls_with_work_of_their_own_and_one_shared_in_turn(moehip):
    """Calls one after another on the library's stream may share their work buffer, of any content, whatever their sizes."""
    M = moehip
    a, b = Batch(M, C.BF16, [5000, 1, 700], 8, 2, 64, 16, seed=31), Batch(M, C.F32, [900, 3000], 16, 4, 128, 32, seed=32)
    need = max(M.lib().moe_paged_attn_work_bytes(len(x.lens), x.nq, x.pool.n_kv, x.hd) for x in (a, b))
    work = M.DeviceBuffer.from_array(np.full(need, 0x7F, np.uint8))
    calls, keep = [], []
    for x in (a, b):
        T = len(x.lens)
        q, out = x.rng.standard_normal((T, x.ld)).astype(np.float32), np.zeros((T, x.ld), np.float32)
        bufs = [M.DeviceBuffer.from_array(v) for v in (q, np.array(x.lens, np.int32) - 1, x.tables, out)]
        keep.append(bufs)
        calls.append((x, q, bufs, M.PagedAttn(bufs[0].ptr, x.ld, T, x.nq, None, bufs[1].ptr, bufs[2].ptr, T, x.width, x.scale, bufs[3].ptr, x.ld,
                                              work.ptr, need)))
    for _ in range(3):
        for x, q, bufs, args in calls:
            M.check(M.lib().moe_paged_attn_dev(C.ref(args), C.ref(x.pool.pages)))
    for x, q, bufs, args in calls:
        out = bufs[3].download((len(x.lens), x.ld), np.float32)
        for t, n in enumerate(x.lens):
            k, v = x.pool.rows(x.tables[t], n)
            want, tol = C.attend(q[t].reshape(x.nq, x.hd).astype(np.float64), k, v, x.scale)
            assert (np.abs(out[t].reshape(x.nq, x.hd) - want) <= tol).all()


# ---- rows of one request that share a tile's columns (more rows than requests)


def _prompts(rng, lens, T):
    """T rows: stretches of one request, mostly upwards, some down, repeated or empty, with rows of no request between"""
    rows = []
    while len(rows) < T:
        r = int(rng.integers(0, len(lens)))
        n, at = int(rng.integers(1, 40)), int(rng.integers(-1, max(lens[r], 1)))
        step = int(rng.choice([1, 1, 1, 0, -1, 50]))
        rows += [(r, min(max(at + i * step, -1), lens[r] - 1)) for i in range(n)]
        if rng.random() < 0.3:
            rows += [(-1, 3)] * int(rng.integers(1, 20))
    return rows[:T]


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("T,nq,nkv,hd,ps", [
    (40, 4, 4, 64, 16), (70, 8, 4, 128, 7), (130, 6, 2, 80, 32), (300, 10, 2, 48, 16), (600, 8, 1, 256, 16), (2048, 4, 4, 32, 16), (2050, 9, 3, 64, 5)])
def test_prompts_share_tiles(moehip, kind, T, nq, nkv, hd, ps):
    """1, 2, 3, 5 and 8 query heads a key-value head: 16, 8, 5, 3 and 2 rows a tile; runs that cross a tile's rows, that
    are cut into pieces, of one length and of many."""
    print("paged attention prompts", kind, T, nq, nkv, hd, ps, flush=True)
    rng = np.random.default_rng(T + hd)
    lens = [700, 1, 90, 0, 3000 if T < 1000 else 400, 33, 250]
    b = Batch(moehip, C.TYPES[kind], lens, nq, nkv, hd, ps, seed=T)
    rows = _prompts(rng, lens, T)
    req, pos = zip(*rows)
    out, q = b.run(req=req, pos=pos, T=T)
    again, _ = b.run(req=req, pos=pos, T=T, q=q.reshape(T, -1), work_from=0x3C)
    np.testing.assert_array_equal(out.view(np.uint32), again.view(np.uint32))
    for t in range(0, T, 1 + T // 150):
        if req[t] < 0:
            assert (out[t] == 7).all(), f"row {t} of no request was written"
        else:
            b.check(out, q, t, req[t], pos[t] + 1)


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("ps,nq,hd", [(16, 4, 64), (7, 2, 128), (32, 16, 256)])
def test_what_lies_behind_a_row_is_not_its_own(moehip, kind, side, ps, nq, hd):
    """A NaN or an infinity at a position that only some rows of a run attend: those before it are right."""
    b = Batch(moehip, C.TYPES[kind], [600, 40], nq, 2, hd, ps, seed=41)
    for at, bits in ((300, C.NAN_BITS), (20, C.INF_BITS)):
        pool = getattr(b.pool, side)
        raw = np.array([bits[b.pool.dtype]], np.uint32).view(np.float32)[0] if kind == "f32" else bits[b.pool.dtype]
        pool[b.tables[0 if at == 300 else 1, at // ps], at % ps, 0, 11] = raw
    b.pool.upload()
    rows = [(0, p) for p in range(290, 310)] + [(1, p) for p in (40 - 1, 19, 20, 5, 21, 0)] + [(0, 599), (0, 299), (0, 300)]
    req, pos = zip(*rows)
    out, q = b.run(req=req, pos=pos, T=len(rows))
    half = nq // 2
    for t, (r, p) in enumerate(rows):
        hit = p >= (300 if r == 0 else 20)
        o = out[t].reshape(nq, hd)
        k, v = b.pool.rows(b.tables[r], p + 1)
        first = half if hit else 0   # the heads of the other key-value head stay right
        with np.errstate(invalid="ignore", over="ignore"):
            want, tol = C.attend(q[t].astype(np.float64), k, v, b.scale)
        assert (np.abs(o[first:] - want[first:]) <= tol[first:]).all(), f"row {t}"
        if hit and (side == "v" or r == 0):
            assert not np.isfinite(o[:half]).all(), f"row {t}"


@pytest.mark.parametrize("kind,ps", [("f32", 16), ("bf16", 7), ("e4m3", 32)])
def test_bad_pages_in_a_run(moehip, kind, ps):
    """A table entry that is no page: the run's rows behind it are NaN, those before it right; a request or a position
    outside the tables ends the run."""
    b = Batch(moehip, C.TYPES[kind], [500, 200], 8, 2, 64, ps, seed=43)
    page = 300 // ps
    b.tables[0, page] = -5
    rows = [(0, p) for p in range(page * ps - 9, page * ps + 9)] + [(1, 5), (1, b.width * ps), (1, 6), (7, 6), (1, 199), (0, 499), (0, 3)]
    req, pos = zip(*rows)
    out, q = b.run(req=req, pos=pos, T=len(rows))
    for t, (r, p) in enumerate(rows):
        if r == 7 or p >= b.width * ps or (r == 0 and p >= page * ps):
            assert np.isnan(out[t]).all(), f"row {t}"
        else:
            b.check(out, q, t, r, p + 1)
