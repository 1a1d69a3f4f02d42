"""Searches at the ends of what a model and its cache hold."""
import numpy as np
import pytest

import model64
import oracle as O

pytestmark = pytest.mark.gpu


def test_to_the_last_position(moehip):
    """A search that feeds the model's last position finds what a longer model finds; a token more is refused, whichever prompt
    it is for."""
    M = moehip
    tm = model64.plain_model(O, 61, 1, False, nq=4, nkv=2)
    short, long = M.model_from_tiny(tm, 24), M.model_from_tiny(tm, 200)
    assert (short.max_seq, long.max_seq) == (24, 200) and M.lib().moe_model_max_seq(None) == -1
    rng = np.random.default_rng(61)
    for lengths, n_new in (((17,), 8), ((3, 15, 1), 10), ((24,), 1)):
        prompts = [rng.integers(0, tm.V, n) for n in lengths]
        ids, score = short.beam_search(prompts, 3, n_new, page_size=8)
        want, ws = long.beam_search(prompts, 3, n_new, page_size=8)
        assert ids == want and [[len(x) for x in g] for g in ids] == [[n_new] * 3] * len(lengths)
        np.testing.assert_array_equal(score, ws)
        with pytest.raises(M.MoeError, match="max_seq 24"):
            short.beam_search(prompts, 3, n_new + 1, page_size=8)
    short.close()
    long.close()


def test_ended_requests_of_a_forked_cache(moehip):
    """Samples of one prompt that end one after another, by set_step: the pages of those that go on are not given back, so a
    new request, which takes what is free, changes nothing for them."""
    M = moehip
    tm = O.TinyModel(D=64, L=2, hd=16, nq=4, nkv=2, dff=32, E=8, top_k=8, V=90, seed=7, std=0.3, theta=1e4)
    m = M.model_from_tiny(tm, 128)
    rng = np.random.default_rng(62)
    prompt, tails, other = rng.integers(0, tm.V, 29), rng.integers(0, tm.V, (4, 12)), rng.integers(0, tm.V, 20)
    # the prompt: 8 pages of 4, the last one copied by three; 5 free ones beside
    c = M.PagedCache(2, 2, 16, 16, 4, 4, 12, 32)
    m.step_paged(c, [29, 0, 0, 0], prompt)
    c.fork([0, 0, 0, 0])
    seq = [np.concatenate([prompt, t[:2]]) for t in tails]
    for i in range(2):
        m.step_paged(c, [1] * 4, tails[:, i])
        assert c.status == 0
    assert c.array("ring_at", 2)[1] == 16 - 11

    def same(lg, rows):
        for r in rows:
            want = m.forward_full(seq[r])
            np.testing.assert_allclose(lg[r], want, atol=2e-4 * np.abs(want).max())

    def step(fresh, ids):
        at = 0
        for r, n in enumerate(fresh):
            if n > 0:
                seq[r] = np.concatenate([seq[r], ids[at:at + n]])
                at += n
            elif n < 0:
                seq[r] = np.zeros(0, np.int64)
        lg, _ = m.step_paged(c, fresh, ids)
        assert c.status == 0 and c.fork_status == 0
        held, tables = c.array("held", 4), c.array("tables", 4, 12)
        assert held.tolist() == [len(s) for s in seq]
        # what is held and what is free are the whole pool, and neither is both
        head, count = c.array("ring_at", 2)
        free = c.array("ring", 16)[(head + np.arange(count)) % 16]
        used = {int(p) for r in range(4) for p in tables[r, :-(-int(held[r]) // 4)]}
        assert len(set(free.tolist())) == count and used.isdisjoint(free.tolist()) and len(used) + count == 16
        return lg

    same(step([-1, 1, -1, 1], tails[[1, 3], 2]), (1, 3))     # two of four end
    same(step([20, 1, 0, 1], np.concatenate([other, tails[[1, 3], 3]])), (0, 1, 3))   # the free pages go to a new request
    same(step([1, 1, 0, -1], [3, tails[1, 4]]), (0, 1))      # the last but one of the samples
    same(step([-1, 1, 0, 0], [tails[1, 5]]), (1,))
    lg = step([0, -1, 0, 0], np.zeros(0, np.int32))
    assert not lg.any() and c.array("ring_at", 2)[1] == 16
    m.close()
