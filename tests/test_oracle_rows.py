"""Pins of oracle/paged.py's log probabilities and norms between blocks."""
import math

import numpy as np
import pytest
from scipy.special import log_softmax
from scipy.stats import entropy as scipy_entropy

from oracle import paged as ref


def test_logprobs_are_those_of_a_softmax():
    x = np.random.default_rng(1).standard_normal(500) * 4
    lp, h, top, best = ref.logprobs(x, 17, 7)
    want = log_softmax(x)
    assert lp == pytest.approx(want[17], abs=1e-13) and h == pytest.approx(scipy_entropy(np.exp(want)), abs=1e-12)
    assert top == list(np.argsort(-x)[:7]) and best == pytest.approx(list(want[top]), abs=1e-13)


def test_logprobs_edges():
    inf, nan = math.inf, math.nan
    assert ref.logprobs([0.0, 0.0, nan, 0.0, -inf], 3, 4) == (pytest.approx(-math.log(3)), pytest.approx(math.log(3)),
                                                             [0, 1, 3, -1], [pytest.approx(-math.log(3))] * 3 + [-inf])
    assert ref.logprobs([nan, -inf], 1, 2) == (-inf, 0.0, [-1, -1], [-inf, -inf])
    assert ref.logprobs([inf, 5.0, inf], 1, 3) == (-inf, pytest.approx(math.log(2)), [0, 2, 1],
                                                   [pytest.approx(-math.log(2))] * 2 + [-inf])
    for token in (-1, 2):
        assert ref.logprobs([1.0, 2.0], token)[0] == -inf


def test_block_norm_by_hand():
    u, out = ref.block_norm([[1.0, 3.0]], [[3.0, 4.0]], post=[2.0, 1.0], gate=[0.5, -1.0], scale=5.0, pre=[1.0, 10.0])
    r = math.sqrt(12.5)
    want = [1.0 + 5 * 0.5 * 3 / r * 2, 3.0 - 5 * 4 / r]
    assert u[0] == pytest.approx(want)
    m = math.sqrt((want[0] ** 2 + want[1] ** 2) / 2)
    assert out[0] == pytest.approx([want[0] / m, 10 * want[1] / m])
    assert ref.block_norm([[1.0, 2.0]])[0].tolist() == [[1.0, 2.0]] and ref.block_norm([[1.0, 2.0]])[1] is None
