"""GPU parity of rqmv_sample against the definition in oracle/paged.py.

Tokens are whole numbers and equal: the reference sums f64 exponentials
exactly, the library their roundings to 2^-42, and the draws here lie further
than n * 2^-42 of the largest from every border (checked on the host; rows
whose border is exact, equal logits, agree by construction). The probability is one
f64 quotient of such sums rounded to fp32: 2^-24 of it, and 2^-42 n of the sums.
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu


def buf(gpu, a, dt):
    return None if a is None else gpu.DeviceBuffer.from_array(np.ascontiguousarray(a, dtype=dt))


def run(gpu, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, ld=None, offset=0, ws=None):
    m, n = logits.shape
    ld = ld or n
    wide = np.full(m * ld + offset, 1e30, np.float32)  # (larger than any logit: reading past a row would show)
    for r in range(m):
        wide[offset + r * ld:offset + r * ld + n] = logits[r]
    L = gpu.DeviceBuffer.from_array(wide)
    T, P = buf(gpu, np.full(m, -9), np.int32), buf(gpu, np.full(m, -9), np.float32)
    gpu.sample(L.view(4 * offset, 4 * m * ld), m, n, ld, buf(gpu, u, np.float32), T, ws or gpu.sample_workspace(m, n),
               buf(gpu, temperature, np.float32), buf(gpu, top_k, np.int32), buf(gpu, top_p, np.float32),
               buf(gpu, min_p, np.float32), P)
    gpu.synchronize()
    return T.download(np.int32), P.download(np.float32)


def check(gpu, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    m, n = logits.shape
    tok, prob = run(gpu, logits, u, temperature, top_k, top_p, min_p, **kw)
    at = lambda a, r, d: d if a is None else a[r]  # noqa: E731
    for r in range(m):
        t, p = ref.sample(logits[r], np.float32(u[r]), np.float32(at(temperature, r, 1.0)), int(at(top_k, r, 0)),
                          np.float32(at(top_p, r, 1.0)), np.float32(at(min_p, r, 0.0)))
        assert tok[r] == t, (r, tok[r], t)
        assert abs(prob[r] - p) <= 2.0 ** -24 * p + 2.0 ** -42 * n, r


def settings(rng, m):
    return {"temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5, 5.0], m), "top_k": rng.choice([0, 1, 2, 7, 50, 400], m),
            "top_p": rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0], m), "min_p": rng.choice([0.0, 0.0, 0.02, 0.3, 1.0], m)}


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 4099, 32000])
@pytest.mark.parametrize("m,spread", [(1, 3.0), (24, 3.0), (24, 0.3), (5, 30.0)])
def test_sample(gpu, n, m, spread):
    rng = np.random.default_rng(n + m)
    logits = (rng.standard_normal((m, n)) * spread).astype(np.float32)
    check(gpu, logits, rng.random(m), **settings(rng, m))
    check(gpu, logits, rng.random(m), ld=n + 3, offset=1)  # all settings off, rows at odd places


@pytest.mark.parametrize("spread", [0.01, 2.0, 8.0])
def test_large_vocabulary(gpu, spread):
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((9, 128256)) * spread).astype(np.float32)
    check(gpu, logits, rng.random(9), temperature=[0, 1, 1, 1, 0.5, 2, 1, 1, 1], top_k=[0, 0, 50, 0, 5000, 0, 0, 100000, 1],
          top_p=[1, 1, 1, 0.9, 0.5, 0.999, 1, 0.7, 1], min_p=[0, 0, 0, 0, 0, 0, 0.001, 0, 0])


def test_largest_rows(gpu):
    """2^20 logits of one value: every candidate the same, the sums at their largest; and one more row count."""
    n = 1 << 20
    logits = np.full((2, n), 3.25, np.float32)
    tok, prob = run(gpu, logits, [0.75, 0.5 ** 20], top_p=[0.5, 1.0])
    assert list(tok) == [int(0.75 * (n // 2)), 1]
    assert prob[0] == 2.0 / n and prob[1] == 1.0 / n


@pytest.mark.parametrize("step", [0.25, 4.0])
def test_ties(gpu, step):
    """Few distinct values, so that every border falls among equals."""
    rng = np.random.default_rng(7)
    logits = (np.round(rng.standard_normal((40, 999)) / step) * step).astype(np.float32)
    check(gpu, logits, rng.random(40), **settings(rng, 40))


def test_exact_borders(gpu):
    """Equal logits: u and top_p at whole fractions, where the running sum meets the target exactly."""
    logits = np.zeros((8, 8), np.float32)
    logits[:, ::2] = -0.0  # the same value as +0
    tok, prob = run(gpu, logits, [0.0, 0.125, 0.5, 0.875, 0.0, 0.5, 0.75, 0.5], top_p=[1, 1, 1, 1, 0.5, 0.5, 0.5, 0.25],
                    top_k=[0, 0, 0, 0, 0, 0, 0, 4])
    assert list(tok) == [0, 1, 4, 7, 0, 2, 3, 0]
    assert list(prob) == [0.125] * 4 + [0.25] * 3 + [1.0]


def test_masked_logits(gpu):
    """-infinity, the type's lowest value, NaN and +infinity among the logits; rows with nothing left."""
    rng = np.random.default_rng(8)
    low = np.finfo(np.float32).min
    logits = rng.standard_normal((9, 300)).astype(np.float32)
    logits[0, ::2] = -np.inf
    logits[1, 1::2] = low
    logits[2, 5:] = np.nan
    logits[3, 7] = logits[3, 200] = np.inf
    logits[4, :] = low
    logits[5, :] = -np.inf
    logits[6, :] = np.nan
    logits[7, :] = -np.inf
    logits[7, 299] = low
    logits[8, :200] = low
    u = [0.3, 0.9, 0.99, 0.6, 0.5, 0.5, 0.5, 0.5, 0.5]
    for t in (1.0, 0.0, 1e-30, 1e30):
        for kw in ({}, {"top_k": [3] * 9}, {"top_p": [0.5] * 9}, {"min_p": [0.5] * 9}):
            check(gpu, logits, u, temperature=[t] * 9, **kw)
    tok, prob = run(gpu, logits, u)
    assert tok[5] == tok[6] == -1 and prob[5] == prob[6] == 0 and tok[7] == 299 and tok[3] == 200


def test_settings_out_of_range(gpu):
    """Settings that switch a step off, or that are brought into range."""
    rng = np.random.default_rng(9)
    logits = (rng.standard_normal((12, 500)) * 2).astype(np.float32)
    nan = np.nan
    check(gpu, logits, [0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.8, 0.9, -1.0, 1.0, nan],
          temperature=[nan, -1, 1, 1, 1, 1, 1, 1, np.inf, 1, 1, 1], top_k=[5, 5, -3, 10 ** 9, 500, 0, 0, 0, 0, 0, 0, 0],
          top_p=[1, 1, 1, 1, 1, -0.5, nan, 1.5, 1, 1, 0.5, 1], min_p=[0, 0, 0, 0, nan, -1, 0, 2, 0, 0, 0, 0])


def test_temperature_zero_is_argmax(gpu):
    rng = np.random.default_rng(10)
    logits = rng.standard_normal((3, 70001)).astype(np.float32)
    logits[1, 69000] = logits[1, 123] = 9.0
    tok, prob = run(gpu, logits, [0.9] * 3, temperature=[0] * 3)
    assert list(tok) == [int(np.argmax(r)) for r in logits] and list(prob) == [1.0] * 3


def test_draws_follow_the_probabilities(gpu):
    """u over an even grid: each token comes as often as its probability says, within one grid step at each end."""
    rng = np.random.default_rng(11)
    row = (rng.standard_normal(40) * 1.5).astype(np.float32)
    m = 4096
    tok, prob = run(gpu, np.tile(row, (m, 1)), (np.arange(m) + 0.5) / m, temperature=[0.8] * m)
    p = np.exp(row.astype(np.float64) / np.float64(np.float32(0.8)))
    p /= p.sum()
    assert np.all(np.abs(np.bincount(tok, minlength=40) / m - p) <= 1.0 / m + 1e-9)
    assert np.allclose(prob, p[tok], rtol=2.0 ** -23, atol=0)


def test_replayed_from_a_graph(gpu):
    """Captured once; each replay has the logits and numbers that it finds, on the workspace that eager calls use too."""
    rng = np.random.default_rng(12)
    m, n = 6, 40000
    L, U = gpu.DeviceBuffer(4 * m * n), gpu.DeviceBuffer(4 * m)
    T, K, P = buf(gpu, np.zeros(m), np.int32), buf(gpu, [0, 0, 50, 50, 0, 0], np.int32), gpu.DeviceBuffer(4 * m)
    top_p = buf(gpu, [1, 0.9, 1, 0.9, 0.5, 1], np.float32)
    ws = gpu.sample_workspace(m, n)
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.sample(L, m, n, n, U, T, ws, None, K, top_p, None, P, stream))
    for i in range(4):
        logits = (rng.standard_normal((m, n)) * (0.2 + 2 * i)).astype(np.float32)
        u = rng.random(m).astype(np.float32)
        L.upload(logits)
        U.upload(u)
        graph.launch(stream)
        stream.synchronize()
        got = T.download(np.int32), P.download(np.float32)
        eager = run(gpu, logits, u, None, [0, 0, 50, 50, 0, 0], [1, 0.9, 1, 0.9, 0.5, 1], None, ws=ws)
        assert np.array_equal(got[0], eager[0]) and np.array_equal(got[1], eager[1])
        for r in range(m):
            assert got[0][r] == ref.sample(logits[r], u[r], 1.0, [0, 0, 50, 50, 0, 0][r],
                                           np.float32([1, 0.9, 1, 0.9, 0.5, 1][r]))[0]
    graph.close()


@pytest.mark.parametrize("n", [4500, 40000])
@pytest.mark.parametrize("step", [0.5, 3.0])
def test_long_rows_of_few_values(gpu, n, step):
    """Few distinct values in rows too long for one list: every border falls among thousands of equals."""
    rng = np.random.default_rng(13)
    m = 12
    logits = (np.round(rng.standard_normal((m, n)) / step) * step).astype(np.float32)
    u = rng.random(m)
    check(gpu, logits, u, **settings(rng, m))
    check(gpu, logits, u, temperature=[1.0] * m, top_k=[0, 1, 30, 1000, 1025, 4000] * 2,
          top_p=[1.0] * 6 + [0.3, 0.9, 0.5, 0.999, 0.7, 0.0], min_p=[0, 0, 0, 0.1, 0.5, 1e-3] * 2)


@pytest.mark.parametrize("t", [1.0, 1e4])
def test_an_outlier_above_a_narrow_rest(gpu, t):
    """One logit far above thousands that share its bins' last ones, drawn at a high temperature."""
    rng = np.random.default_rng(14)
    logits = (rng.standard_normal((4, 30000)) * 1e-3).astype(np.float32)
    logits[:, 777] = 5e3
    check(gpu, logits, [0.2, 0.9, 0.5, 0.99], temperature=[t] * 4, top_k=[0, 100, 0, 9000], top_p=[1, 1, 0.8, 0.9],
          min_p=[0, 0, 0.01, 0.2])


@pytest.mark.parametrize("n", [50, 4500])
def test_more_rows_than_one_workspace_holds(gpu, n):
    """1,100 rows with settings of their own: the rows behind the first 1,024 give what they give alone."""
    rng = np.random.default_rng(15)
    m = 1100
    logits = (rng.standard_normal((m, n)) * 2).astype(np.float32)
    u, kw = rng.random(m), settings(rng, m)
    tok, prob = run(gpu, logits, u, **kw)
    part = {k: v[1000:] for k, v in kw.items()}
    alone = run(gpu, logits[1000:], u[1000:], **part)
    assert np.array_equal(tok[1000:], alone[0]) and np.array_equal(prob[1000:], alone[1])
    few = np.r_[0:4, 1020:1030]
    check(gpu, logits[few], u[few], **{k: v[few] for k, v in kw.items()})
    check_few = [ref.sample(logits[r], np.float32(u[r]), np.float32(kw["temperature"][r]), int(kw["top_k"][r]),
                            np.float32(kw["top_p"][r]), np.float32(kw["min_p"][r]))[0] for r in few]
    assert list(tok[few]) == check_few


@pytest.mark.parametrize("n", [900, 6177, 12362, 58032])
@pytest.mark.parametrize("t,spread", [(1.0, 1e-21), (2.0, 1e-17), (1e5, 1e-20), (1.0, 2e-16), (1e-6, 1e-20), (30.0, 1e-13)])
def test_min_p_of_one_among_masses_that_round_to_one(gpu, n, t, spread):
    """Logits closer than a unit of mass: their masses are equal, but an e below 1 in 64 bits is not kept."""
    rng = np.random.default_rng(n)
    m = 8
    logits = (rng.standard_normal((m, n)) * spread).astype(np.float32)
    check(gpu, logits, rng.random(m), temperature=[t] * m, top_k=[0, 0, 5000, n - 1, 1025, 50, n - 1, 0],
          top_p=[1, 0.3, 1, 0.3, 0.9, 1, 1, 0.999], min_p=[1.0] * m)


@pytest.mark.parametrize("n", [900, 20000])
def test_min_p_at_the_smallest_logits(gpu, n):
    """min_p's border between the row's last logits, where the bins end: exact to the logit."""
    logits = (-np.arange(n) * 2.0 ** -12).astype(np.float32)[None]  # each a candidate of its own
    for at in (n - 1, n - 2, n - 40, n // 2):
        min_p = np.float32(np.exp(np.float64(logits[0, at])))
        z = np.log(np.float64(min_p))
        kept = int((logits[0].astype(np.float64) >= z).sum())
        e = np.exp(logits[0, :kept].astype(np.float64))
        tok, prob = run(gpu, logits, [1.0], min_p=[min_p])  # (u of 1: the last that counts)
        assert tok[0] == kept - 1
        assert abs(prob[0] - e[-1] / e.sum()) <= 2.0 ** -24 * prob[0] + 2.0 ** -42 * n


@pytest.mark.parametrize("n", [40, 3000, 9000])
@pytest.mark.parametrize("t", [5e-38, 1.2e-38, 1e-41, 1e-44, 1e-30])
def test_smallest_temperatures(gpu, n, t):
    """Temperatures whose inverse leaves fp32's range, logits a few of them apart."""
    rng = np.random.default_rng(n)
    m = 6
    logits = (-rng.random((m, n)) * 20 * np.float64(np.float32(t))).astype(np.float32)
    logits[0] = np.round(rng.standard_normal(n)) * 1e30
    check(gpu, logits, rng.random(m), temperature=[t] * m, top_k=[0, 0, 30, 0, 2000, 0], top_p=[1, 1, 1, 0.5, 0.9, 1],
          min_p=[0, 0, 0, 0, 0, 0.3])
