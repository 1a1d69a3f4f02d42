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
