"""Beams whose values lie close together: how far apart they have to be for the order to be the formula's.

A row's log sum exp is off by at most 2^-21 (test_gpu_beam_select.py), which does not average out where one token, or some equal
ones, hold nearly all of it; so rows keep their order from 2^-20 on, and a candidate's log probability, at most its row's, is
above it by no more than 2^-21 and a rounding."""
import numpy as np
import pytest

import test_gpu_beam_select as S
from paged_cases import U

pytestmark = pytest.mark.gpu


def _logits(style, rows, vocab, rng):
    x = np.full((rows, vocab), -30.0, np.float32) + rng.standard_normal((rows, vocab)).astype(np.float32)
    base = rng.uniform(-9, 9, rows).astype(np.float32)
    if style == "one":      # one token holds all but 1e-9 or so
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 0
    elif style == "two":    # two equal ones
        x[:, rng.permutation(vocab)[:2]] = 0
    else:                   # all alike
        x[:] = 0
    return x + base[:, None]


@pytest.mark.parametrize("style", ["one", "two", "all"])
@pytest.mark.parametrize("n_beam,vocab", [(4, 5000), (4, 700), (16, 40000), (20, 5000), (64, 3000)])
def test_close_beams(moehip, style, n_beam, vocab):
    """Scores from -1 on in steps of 2^-18, in any order of the rows."""
    rng = np.random.default_rng(n_beam + vocab)
    logits = _logits(style, n_beam, vocab, rng)
    score = (-1 - rng.permutation(n_beam) * 2.0 ** -18).astype(np.float32)
    got = S.Select(moehip, logits, score, None, None, n_beam, -1, 0).run()
    S.check(got, logits, score, None, None, n_beam, -1, 0)
    order = np.argsort(-score)
    each = {"one": 1, "two": 2, "all": vocab}[style]   # candidates that a row has before those of the next come
    want = np.repeat(order, min(each, n_beam))[:n_beam]
    np.testing.assert_array_equal(got["parent"], want)
    assert (got["score"].astype(np.float64) <= score[want].astype(np.float64) + S.LSE + 1.01 * U * np.abs(score[want])).all()
