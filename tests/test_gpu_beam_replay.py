"""Model.beam_search followed step by step, whatever its logits: each choice against the selection in 64 bits, the lists and
scores that it returns against those that its own choices make; and steps over 16-bit and 8-bit pages against the 64-bit
model on what such pages hold."""
import numpy as np
import pytest

import model64
import oracle as O
import paged_cases as C
import test_gpu_beam_search as G
import test_gpu_beam_select as S

pytestmark = pytest.mark.gpu


class Watch:
    """The library, which notes what each choice of a search had and left."""

    def __init__(self, M):
        self.M, self.real, self.steps = M, M.lib(), []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def read(self, ptr, shape, dtype):
        out = np.empty(shape, dtype)
        self.M.check(self.real.moe_memcpy_d2h(out.ctypes.data, ptr, out.nbytes))
        return out

    def _note(self, ref, call):
        s = ref._obj
        rows = (s.n_groups * s.n_beam,)
        had = (self.read(s.logits, rows + (s.vocab,), np.float32), self.read(s.score, rows, np.float32), self.read(s.done, rows, np.int32))
        st = call()
        got = {n: self.read(getattr(s, p), rows, np.int32) for n, p in (("parent", "parent"), ("token", "token"), ("done", "done_out"), ("fresh", "fresh"))}
        got["score"] = self.read(s.score_out, rows, np.float32)
        self.steps.append((had, got, s.n_beam, s.eos, s.pad))
        return st

    def moe_model_step_beams(self, m, select, *rest):
        return self._note(select, lambda: self.real.moe_model_step_beams(m, select, *rest))

    def moe_beam_select_dev(self, select):
        return self._note(select, lambda: self.real.moe_beam_select_dev(select))


def _followed(steps, rows):
    seq = [[] for _ in range(rows)]
    for (logits, score, done), got, n_beam, eos, pad in steps:
        S.check(got, logits, score, done, None, n_beam, eos, pad)
        seq = [seq[p] + ([] if done[p] else [int(t)]) if p >= 0 else [] for p, t in zip(got["parent"], got["token"])]
    return seq, steps[-1][1]["score"]


@pytest.mark.parametrize("kind", list(C.TYPES))
@pytest.mark.parametrize("experts,n_beam,n_new,ps", [(False, 3, 9, 8), (True, 4, 8, 16), (True, 20, 7, 4), (False, 1, 6, 8)])
def test_replay(moehip, kind, experts, n_beam, n_new, ps, monkeypatch):
    M = moehip
    tm = model64.plain_model(O, 70 + n_beam, 1, experts, nq=4, nkv=2)
    m = M.model_from_tiny(tm, 256)
    rng = np.random.default_rng(71)
    prompts = [rng.integers(0, tm.V, n) for n in (1, 18, 150)]
    eos, ended = -1, 0
    for _ in range(3):   # without an end, then with tokens that it chose first and in its middle
        w = Watch(M)
        monkeypatch.setattr(M, "lib", lambda: w)
        ids, score = m.beam_search(prompts, n_beam, n_new, eos, page_size=ps, dtype=C.TYPES[kind])
        monkeypatch.undo()
        assert len(w.steps) == n_new
        want, last = _followed(w.steps, 3 * n_beam)
        assert [x for g in ids for x in g] == want
        np.testing.assert_array_equal(score.reshape(-1), last)
        ended += sum(bool(x) and x[-1] == eos for x in want)
        assert all(len(x) == n_new or x[-1] == eos for x in want)
        eos = want[0][0] if eos < 0 else want[-1][len(want[-1]) // 2]
    assert ended
    m.close()


def _stored(k, dk, dtype):
    """What a page holds of values k, each off by dk at most -> (value, bound): exact unless a border of the type lies between."""
    dec = lambda x: C.decode(C.encode(x.astype(np.float32), dtype), dtype)  # noqa: E731
    y = dec(k)
    return y, np.maximum(np.abs(dec(k - dk) - y), np.abs(dec(k + dk) - y))


def _attend(q, dq, k, dk, v, dv, scale):
    """model64.attend with a bound for each position's score d_i instead of one for all, since a border between a few of many
    values leaves those few uncertain by a whole step: weights p_i e^(+-d_i) move sum p v by at most (sum w |v| + sum w |out|)
    / (1 - sum w), w = p (e^d - 1)."""
    U, (T, nq, hd) = model64.U, q.shape
    g = nq // k.shape[1]
    out, tol = np.zeros((T, nq, hd)), np.full((T, nq, hd), np.inf)
    for t in range(T):
        for h in range(nq):
            kh, dkh, vh, dvh = (z[:t + 1, h // g] for z in (k, dk, v, dv))
            s = scale * (kh @ q[t, h])
            ds = scale * (np.abs(kh) @ dq[t, h] + dkh @ np.abs(q[t, h]) + dkh @ dq[t, h] + (hd + 3) * U * (np.abs(kh) @ np.abs(q[t, h])))
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vh
            w = p * np.expm1(np.minimum(ds, 1.0))
            if ds.max() < 1 and w.sum() < 0.2:
                moved = w @ np.abs(vh) + w.sum() * np.abs(out[t, h]) + (p + w) @ dvh
                tol[t, h] = model64.MORE * (moved + (4 * U * (s.max() - s.min()) + (t + 41) * U) * ((p + w) @ np.abs(vh))) / (1 - w.sum())
    return out.reshape(T, -1), tol.reshape(T, -1)


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("n_groups,n_beam,ps,lo,hi", [(2, 4, 16, 20, 60), (1, 16, 8, 140, 180)])
def test_steps_over_small_types(moehip, kind, n_groups, n_beam, ps, lo, hi, monkeypatch):
    print("beam steps", kind, n_groups, n_beam, flush=True)
    dtype = C.TYPES[kind]
    tm = model64.plain_model(O, 80 + n_beam, 1, False, nq=8, nkv=2)
    m = moehip.model_from_tiny(tm, 256)
    rng = np.random.default_rng(81)
    prompts = [rng.integers(0, tm.V, int(rng.integers(lo, hi))) for _ in range(n_groups)]
    rope = O.rope_tables(tm.hd, tm.theta, 256)
    monkeypatch.setattr(model64, "attend", lambda q, dq, k, dk, v, dv, scale: _attend(q, dq, *_stored(k, dk, dtype), *_stored(v, dv, dtype), scale))
    s = G.Search(moehip, m, prompts, n_beam, 8, kind, ps, eos=-1)
    told = seen = 0
    for _ in range(6):
        s.step()
        logits = s.logits.download((s.R, s.V), np.float32)
        for r in range(s.R):
            want, tol = model64.forward(tm, np.array(s.seq[r]), rope)
            seen += 1
            if np.isfinite(tol[-1]).all():
                told += 1
                assert (np.abs(logits[r] - want[-1]) <= tol[-1]).all(), f"row {r}: {np.max(np.abs(logits[r] - want[-1]) / tol[-1]):.2f} times the bound"
    assert told > seen // 2
    m.close()
