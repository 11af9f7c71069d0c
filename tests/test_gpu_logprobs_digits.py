"""rqmv_logprobs of rows with one very likely token: log probabilities next to 0 and small entropies keep their digits.

Bars, relative to the values themselves. With d = x - m and r = sum e^d over all logits but one largest, the row's
log probabilities are d - log(1 + r) and its entropy log(1 + r) - sum d e^d / (1 + r), whose two parts are both positive.
A term e^d is off by 9 * 2^-24 |d| + 3 * 2^-22, and sums of terms of one sign by 90 * 2^-24 more (counted in test_gpu_logprobs.py: the
additions of 1 where parts that do not hold the row's largest logit join are within the 90), so r is off by Er =
(sum (9 * 2^-24 |d| + 3 * 2^-22) e^d) / r + 90 * 2^-24, relative; log(1 + r), of at most the relative error of r, by Er, and by 2^-22 for the
logarithm. A log probability adds the roundings of d, 2^-24 |d|, and of the difference, 2^-24 of itself. sum d e^d is off by
(10 * 2^-24 |d| + 3 * 2^-22) of each term and 120 * 2^-24, its quotient with 1 + r by Er and 2^-23 more, the entropy by
2^-24 of itself.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_logprobs import run

pytestmark = pytest.mark.gpu


def check(gpu, x, tokens, top):
    x = np.asarray(x, np.float32)
    got = run(gpu, x, tokens, top)
    for i, row in enumerate(x.astype(np.float64)):
        largest = int(row.argmax())
        d = row - row[largest]
        e = np.exp(d)
        rest, size = np.delete(e, largest), np.delete(np.abs(d), largest)
        r = math.fsum(rest)
        log_s, td = math.log1p(r), math.fsum(rest * size)
        er = math.fsum((9 * 2.0 ** -24 * size + 3 * 2.0 ** -22) * rest) / r + 90 * 2.0 ** -24 if r else 0.0
        off_log = (er + 2.0 ** -22) * log_s
        order = np.argsort(-row, kind="stable")[:top]
        assert top == 0 or got["top_tokens"].reshape(-1, top)[i].tolist() == order.tolist()
        pairs = [(int(tokens[i]), got["logprob"][i])]
        pairs += [(int(t), got["top_logprobs"].reshape(-1, top)[i, k]) for k, t in enumerate(order)]
        for token, value in pairs:
            want = d[token] - log_s
            bar = off_log + 2.0 ** -24 * (abs(d[token]) + abs(want))
            assert abs(value - want) <= bar, (i, token, value, want, bar)
        want = log_s + td / (1 + r)
        off_t = math.fsum((10 * 2.0 ** -24 * size + 3 * 2.0 ** -22) * rest * size) + (120 * 2.0 ** -24 + er + 2.0 ** -23) * td
        bar = off_log + off_t / (1 + r) + 2.0 ** -24 * want
        assert abs(got["entropy"][i] - want) <= bar, (i, got["entropy"][i], want, bar)


@pytest.mark.parametrize("n", [2, 5, 63, 1000, 4096, 4097, 8192, 8193, 40000, 128256])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_a_token_of_almost_all(gpu, n, top):
    """The likeliest token stands 3 to 60 above the rest, at the row's start, its end, or between."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((7, n)).astype(np.float32)
    at = [0, n - 1, n // 2, n // 3, 1, n // 5, n - 2]
    x[np.arange(7), at] = [3, 10, 20, 25, 30, 40, 60]
    check(gpu, x, at, min(top, n))
    check(gpu, x, [(a + 1) % n for a in at], min(top, n))


@pytest.mark.parametrize("n", [300, 5000, 40000])
def test_two_and_more_largest(gpu, n):
    """Equal largest logits in one lane, one wave, or far apart, alone and beside others."""
    x = np.full((6, n), -25.0, np.float32)
    for row, at in enumerate([[0, 1], [0, 4], [0, n - 1], [7, n // 2, n - 3], range(0, n, 97), range(n)]):
        x[row, list(at)] = 4.0
    check(gpu, x, [0, 4, n - 1, 8, 97, n - 1], 4)
    check(gpu, np.where(x == 4.0, x, -np.float32(80.0)), [1, 0, 0, 7, 0, 1], 0)


@pytest.mark.parametrize("n", [1, 500, 20000])
def test_nothing_beside_the_token(gpu, n):
    """One candidate: log probability and entropy are 0."""
    x = np.full((1, n), -np.inf, np.float32)
    x[0, n // 2] = 3.5
    got = run(gpu, x, [n // 2], 1)
    assert got["logprob"][0] == 0 and got["entropy"][0] == 0 and got["top_logprobs"][0] == 0
