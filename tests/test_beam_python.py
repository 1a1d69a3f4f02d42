"""What the Python wrappers of the beam search refuse before any device memory is made, and what they keep of a cache's
state on the host.  CPU only."""
import numpy as np
import pytest

import moehip as M


def _model(max_seq, vocab=90):
    m = M.Model.__new__(M.Model)
    m.h, m.V, m.max_seq = None, vocab, max_seq
    m.cfg = M.qwen_config(64, 1, 16, 4, 2, 32, 8, 8, vocab)
    return m


class Made(Exception):
    pass


@pytest.fixture
def no_memory(monkeypatch):
    def made(*a):
        raise Made

    monkeypatch.setattr(M.DeviceBuffer, "__init__", made)


@pytest.mark.parametrize("lengths,n_new,fits", [((5,), 16, True), ((5,), 17, False), ((20,), 1, True), ((21,), 1, False), ((1, 18, 3), 3, True), ((1, 18, 3), 4, False)])
def test_search_past_the_model(lengths, n_new, fits, no_memory):
    """A model of 20 positions: what the steps feed is the prompt and every new token but the last."""
    with pytest.raises(Made if fits else M.MoeError, match=None if fits else "max_seq 20"):
        _model(20).beam_search([np.zeros(n, np.int32) for n in lengths], 3, n_new)


@pytest.mark.parametrize("bad", [-1, 90, 1 << 30])
def test_search_of_no_token(bad, no_memory):
    """An id that is none is refused, as moe_model_generate does, not clamped."""
    with pytest.raises(M.MoeError, match="id outside 0 .. 89"):
        _model(20).beam_search([[1, 2], [0, 89, bad, 3]], 2, 3)
    with pytest.raises(Made):
        _model(20).beam_search([[1, 2], [0, 89, 3]], 2, 3)


class Buffer:
    def __init__(self):
        self.ptr, self.nbytes, self.got = 1, 1 << 20, []

    def upload(self, a):
        self.got.append(np.array(a))


def _cache(n_req=4):
    c = M.PagedCache.__new__(M.PagedCache)
    c.n_req, c.max_tokens, c.layers = n_req, 8, ()
    c.plan = M.PagedPlan(n_req, 3, 20, 4, 8)
    c._b = {n: Buffer() for n in ("fresh", "ids", "held", "ring_at", "ring", "tables", "copies", "fork_status", "fork_work")}
    c.forks = []
    c.fork = lambda parent: c.forks.append(np.asarray(parent).tolist())
    return c


def test_ended_requests_of_a_forked_cache():
    """The plan gives an ended request's pages back whoever else holds them, so that one of a forked cache is ended by a fork
    before; one of a cache that was never forked by the plan alone."""
    c = _cache()
    c.set_step([-1, 1, 0, -1], [5])
    assert c.forks == []
    c.fork_args(1)
    c.set_step([1, 1, 0, 2], [5, 6, 7, 8])
    assert c.forks == []
    c.set_step([-1, 1, 0, -1], [5])
    assert c.forks == [[-1, 1, 2, -1]]
    assert [x.tolist() for x in c._b["fresh"].got] == [[-1, 1, 0, -1], [1, 1, 0, 2], [-1, 1, 0, -1]]
    for fresh, ids in (([-1, 1, 0], [5]), ([-1, 2, 0, 0], [5]), ([-1, 1, 0, 0], np.zeros(9))):   # a refused step ends none
        with pytest.raises(M.MoeError):
            c.set_step(fresh, ids)
    assert len(c.forks) == 1
