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
