"""moe_beam_select_dev against a selection in 64 bits.

Bound of a value: a term of a row's sum is off by three half steps of fp32 (the hardware's exp2 by two, its correction one),
sums of four add two, so the logarithm of the sum by 5 U at most, taken as 8 U; then value is rounded to fp32 once.
Whole numbers are equal wherever the plain form's candidates lie further apart than that."""
import ctypes

import numpy as np
import pytest

import beam_cases as B
from paged_cases import U

pytestmark = pytest.mark.gpu

LSE = 8 * U


class Select:
    def __init__(self, M, logits, score, done, weight, n_beam, eos, pad, ld=None, in_place=False):
        rows, vocab = logits.shape
        self.M, self.rows = M, rows
        wide = np.full((rows, ld or vocab), np.nan, np.float32)   # what lies behind a row is not read
        wide[:, :vocab] = logits
        buf = M.DeviceBuffer.from_array
        self.b = {"logits": buf(wide), "score": buf(score.astype(np.float32))}
        self.b["done"] = None if done is None else buf(np.asarray(done, np.int32))
        self.b["weight"] = None if weight is None else buf(np.asarray(weight, np.float32))
        for n in ("parent", "token", "fresh"):
            self.b[n] = buf(np.full(rows, -7, np.int32))
        self.b["score_out"] = self.b["score"] if in_place else buf(np.full(rows, 7, np.float32))
        self.b["done_out"] = self.b["done"] if in_place else buf(np.full(rows, -7, np.int32))
        need = M.lib().moe_beam_select_work_bytes(rows // n_beam, n_beam, vocab)
        assert need > 0
        self.work = buf(np.full(need, 0xA5, np.uint8))
        p = {n: None if b is None else b.ptr for n, b in self.b.items()}
        self.args = M.BeamSelect(rows // n_beam, n_beam, vocab, p["logits"], wide.shape[1], p["score"], p["done"], p["weight"], eos, pad, p["parent"], p["token"],
                                 p["score_out"], p["done_out"], p["fresh"], self.work.ptr, need)

    def run(self):
        self.M.check(self.M.lib().moe_beam_select_dev(ctypes.byref(self.args)), "select")
        out = {n: self.b[n].download((self.rows,), np.int32) for n in ("parent", "token", "fresh")}
        return dict(out, done=self.b["done_out"].download((self.rows,), np.int32), score=self.b["score_out"].download((self.rows,), np.float32))


def check(got, logits, score, done, weight, n_beam, eos, pad):
    rows = len(score)
    done = np.zeros(rows, int) if done is None else done
    want = B.select(logits, score, done, weight, n_beam, eos, pad)
    w = np.ones(rows) if weight is None else np.asarray(weight, np.float64)
    for r in range(rows):
        p, t = int(got["parent"][r]), int(got["token"][r])
        msg = f"row {r}: parent {p}, token {t}, score {got['score'][r]}; {[(n, want[n][r]) for n in ('parent', 'token', 'score')]}"
        if want["parent"][r] < 0:
            assert (p, t, got["done"][r], got["fresh"][r]) == (-1, -1, 0, 0) and got["score"][r] == -np.inf, msg
            continue
        assert r // n_beam * n_beam <= p < (r // n_beam + 1) * n_beam, msg
        value = float(score[p]) if done[p] else want["values"][p, t]
        # the candidate at this place is the plain form's, or as good within what the sums may be off by
        near = LSE * (w[p] + w[want["parent"][r]]) if p != want["parent"][r] else 0.0
        assert abs(value * w[p] - want["rank"][r]) <= near, msg
        if near == 0.0:
            assert t == want["token"][r], msg
        assert abs(float(got["score"][r]) - value) <= (0 if done[p] else LSE) + U * abs(value) * 1.01, msg
        ended = int(bool(done[p]) or t == eos)
        assert got["done"][r] == ended and got["fresh"][r] == 1 - ended, msg
        if done[p]:
            assert t == pad, msg
    for g in range(0, rows, n_beam):   # no candidate twice
        taken = [(p, t) for p, t in zip(got["parent"][g:g + n_beam], got["token"][g:g + n_beam]) if p >= 0]
        assert len(set(taken)) == len(taken)


@pytest.mark.parametrize("n_groups,n_beam,vocab", [(1, 1, 1), (1, 4, 3), (2, 3, 7), (3, 2, 1023), (1, 5, 1024), (2, 8, 1025), (1, 64, 64), (2, 64, 5000), (7, 5, 50257),
                                                   (1, 4, 151936), (70, 2, 4097), (5, 33, 9000), (300, 1, 300), (1, 64, 151936), (3, 31, 50257), (2, 32, 50257), (3, 20, 1000), (2, 64, 257), (5, 7, 256), (2, 17, 40)])
@pytest.mark.parametrize("style", ["plain", "masked", "ended"])
def test_select(moehip, n_groups, n_beam, vocab, style):
    print("beam select", n_groups, n_beam, vocab, style, flush=True)
    rng = np.random.default_rng(n_groups * 1000003 + n_beam * 1009 + vocab)
    rows = n_groups * n_beam
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    score = -20 * rng.random(rows)
    done = weight = None
    eos, pad = -1, 0
    if style != "plain":
        logits[rng.random((rows, vocab)) < 0.5] = -np.inf
        score[rng.random(rows) < 0.2] = -np.inf
        weight = rng.uniform(0.05, 1, rows)
    if style == "ended":
        done = rng.random(rows) < 0.4
        eos, pad = int(np.argmax(logits[0])), -3
    score = score.astype(np.float32)
    weight = None if weight is None else weight.astype(np.float32)
    s = Select(moehip, logits, score, done, weight, n_beam, eos, pad, ld=vocab + 3 if style == "masked" else None)
    got = s.run()
    check(got, logits, score, done, weight, n_beam, eos, pad)
    again = s.run()
    for n in got:
        np.testing.assert_array_equal(got[n], again[n], err_msg=n)


@pytest.mark.parametrize("n_beam", [6, 16, 18, 64])
def test_ties(moehip, n_beam):
    """Equal logits: the lower token; equal rows: the lower row; -0 is 0."""
    vocab = 3000
    rng = np.random.default_rng(5)
    logits = np.repeat(rng.integers(-3, 4, (2, vocab)), n_beam, 0).astype(np.float32)
    logits[logits == 0] = np.where(rng.random((logits == 0).sum()) < 0.5, 0.0, -0.0)
    logits[:n_beam] = logits[0]
    logits[n_beam:] = 1.0
    score = np.array([-1.0] * n_beam + [-3.0, -1.0, -1.0, -3.0, -1.0, -2.0] + [-4.0] * (n_beam - 6), np.float32)
    check(Select(moehip, logits, score, None, None, n_beam, -1, 0).run(), logits, score, None, None, n_beam, -1, 0)
    got = Select(moehip, logits, score, None, None, n_beam, -1, 0).run()
    top = np.nonzero(logits[0] == 3)[0]
    assert got["parent"][:n_beam].tolist() == [0] * n_beam and got["token"][:n_beam].tolist() == top[:n_beam].tolist()
    assert got["parent"][n_beam:].tolist() == [n_beam + 1] * n_beam and got["token"][n_beam:].tolist() == list(range(n_beam))


@pytest.mark.parametrize("n_beam", [16, 17, 64])
def test_all_zero_large(moehip, n_beam):
    """Every logit the same, over many blocks."""
    logits = np.zeros((n_beam, 70000), np.float32)
    score = np.linspace(-2, -1, n_beam).astype(np.float32)
    got = Select(moehip, logits, score, None, None, n_beam, 3, 0).run()
    assert got["parent"].tolist() == [n_beam - 1] * n_beam and got["token"].tolist() == list(range(n_beam))
    assert got["done"].tolist() == [int(t == 3) for t in range(n_beam)]
    np.testing.assert_allclose(got["score"], score[-1] - np.log(70000.0), rtol=2 * U, atol=LSE)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("n_beam", [9, 25])
def test_rows_without_candidates(moehip, bad, n_beam):
    """A NaN or an infinity in a row, all of it masked, scores and weights that cannot be."""
    rng = np.random.default_rng(8)
    vocab = 5001
    logits = rng.standard_normal((n_beam, vocab)).astype(np.float32)
    score = -rng.random(n_beam).astype(np.float32)
    weight = np.ones(n_beam, np.float32)
    logits[0, 4999] = bad
    logits[1] = -np.inf
    logits[2, :] = -np.inf
    logits[2, [17, 4000]] = [-50, -49.5]      # two candidates, far below the others
    score[3], score[4] = bad, -np.inf
    weight[5], weight[6], weight[7] = 0.0, bad, -1.0
    logits[8, 2:] = -np.inf
    logits[9:] = -np.inf
    args = (logits, score, None, weight, n_beam, -1, 0)
    got = Select(moehip, *args).run()
    check(got, *args)
    assert sorted(got["parent"].tolist()) == [-1] * (n_beam - 4) + [2, 2, 8, 8]


@pytest.mark.parametrize("n_beam", [6, 40])
def test_large_and_small_logits(moehip, n_beam):
    """Rows whose logits lie far from zero, rise step by step, or span all of fp32."""
    rng = np.random.default_rng(9)
    vocab = 20000
    x = rng.standard_normal((n_beam, vocab))
    x[0] += 3000
    x[1] -= 3000
    x[2] = np.sort(x[2]) * 30
    x[3] = -np.sort(-x[3]) * 30
    x[4] *= 1e30
    x[5] *= 1e-30
    logits = x.astype(np.float32)
    score = np.zeros(n_beam, np.float32)
    args = (logits, score, None, None, n_beam, -1, 0)
    check(Select(moehip, *args).run(), *args)


@pytest.mark.parametrize("n_beam", [4, 24])
def test_in_place_and_graph(moehip, n_beam):
    """A search's steps with score and done updated in place, by a captured graph; the same calls made eagerly between."""
    import test_gpu_paged_serving as G
    rng = np.random.default_rng(11)
    vocab, groups = 2500, 3
    rows = n_beam * groups
    hip = G.Hip(moehip)
    score = np.where(np.arange(rows) % n_beam == 0, 0.0, -np.inf).astype(np.float32)
    done = np.zeros(rows, np.int32)
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    s, e = (Select(moehip, logits, score, done, None, n_beam, 1, 0, in_place=True) for _ in "ab")
    graph = hip.capture(lambda: moehip.check(moehip.lib().moe_beam_select_dev(ctypes.byref(s.args))))
    for step in range(5):
        logits = (4 * rng.standard_normal((rows, vocab))).astype(np.float32)
        logits[:, 1] += 6
        for x in (s, e):
            x.b["logits"].upload(logits)
        hip.launch(graph)
        moehip.synchronize()
        got = {n: s.b[n].download((rows,), np.int32) for n in ("parent", "token", "fresh")}
        got.update(done=s.b["done_out"].download((rows,), np.int32), score=s.b["score_out"].download((rows,), np.float32))
        eager = e.run()
        for n in got:
            np.testing.assert_array_equal(got[n], eager[n], err_msg=f"step {step}, {n}")
        check(got, logits, score, done, None, n_beam, 1, 0)
        score, done = got["score"], got["done"]
    assert done.any()
    hip.destroy(graph)
