"""GPU parity of rqmv_logprobs against oracle/paged.py.

Bars. With d = x - m <= 0 and p the probabilities: a term e^d is off by 2^-24 |d| each for the rounded
difference, its product with log2 e and that constant, and 2^-22 for the exponential; moving a slice's sum to the row's
largest logit, and a wave's to its slice's, costs as much again, with differences no larger than |d|:
9 * 2^-24 |d| + 3 * 2^-22 in all. All terms have one sign, so sums of them add (64 in a row + 22
joins) * 2^-24 relative. So s is off by Es = 9 * 2^-24 sum p |d| + 3 * 2^-22 + 90 * 2^-24, relative; log s by that and 2^-23 of
itself; a log probability by that, 2^-24 |d| and 2^-24 of itself; t / s by 10 * 2^-24 sum p d^2 + (Es +
3 * 2^-22 + 120 * 2^-24) sum p |d|, and the entropy by the two together and 2^-24 of itself.
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu


def run(gpu, x, tokens=None, top=0, ld=None, entropy=True, offset=0, stream=None):
    rows, n = x.shape
    ld = ld or n
    host = np.full(offset + rows * ld + 8, np.nan, np.float32)
    for r in range(rows):
        host[offset + r * ld:offset + r * ld + n] = x[r]
    whole = gpu.DeviceBuffer.from_array(host)
    X = whole.view(4 * offset, whole.nbytes - 4 * offset)
    f32 = lambda k: gpu.DeviceBuffer.from_array(np.full(k, 7, np.float32))  # noqa: E731
    out = {"logprob": f32(rows) if tokens is not None else None, "entropy": f32(rows) if entropy else None,
           "top_tokens": f32(rows * top) if top else None, "top_logprobs": f32(rows * top) if top else None}
    T = gpu.DeviceBuffer.from_array(np.asarray(tokens, np.int32)) if tokens is not None else None
    gpu.logprobs(X, rows, n, ld, tokens=T, top=top, workspace=gpu.logprobs_workspace(rows, n, top), stream=stream, **out)
    gpu.synchronize()
    return {k: v.download(np.int32 if k == "top_tokens" else np.float32) for k, v in out.items() if v is not None}


def check(gpu, x, tokens=None, top=0, **kw):
    x = np.asarray(x, np.float32)
    got = run(gpu, x, tokens, top, **kw)
    for r in range(len(x)):
        lp, h, best, best_lp = ref.logprobs(x[r], None if tokens is None else int(tokens[r]), top)
        v = np.where(np.isnan(x[r]), -np.inf, x[r]).astype(np.float64)
        if v.max() == np.inf:
            v = np.where(v == np.inf, 0.0, -np.inf)
        if top:
            assert got["top_tokens"][r * top:(r + 1) * top].tolist() == best
        if v.max() == -np.inf:
            es = et = log_s = 0.0
            d = v
        else:
            d = v - v.max()
            s = np.exp(d).sum()
            p, a = np.exp(d) / s, np.abs(np.where(d > -1e4, d, 0.0))
            es = 9 * 2.0 ** -24 * (p * a).sum() + 3 * 2.0 ** -22 + 90 * 2.0 ** -24
            et = 10 * 2.0 ** -24 * (p * a * a).sum() + (es + 3 * 2.0 ** -22 + 120 * 2.0 ** -24) * (p * a).sum()
            log_s = np.log(s)

        def near(value, want, token):
            if not 0 <= token < len(d) or want == -np.inf:
                assert value == want
                return
            bar = es + 2.0 ** -23 * log_s + 2.0 ** -24 * (abs(d[token]) + abs(want))
            assert abs(value - want) <= bar, (r, token, value, want, bar)

        if tokens is not None:
            near(got["logprob"][r], lp, int(tokens[r]))
        for i in range(top):
            near(got["top_logprobs"][r * top + i], best_lp[i], best[i])
        if "entropy" in got:
            assert abs(got["entropy"][r] - h) <= es + 2.0 ** -23 * log_s + et + 2.0 ** -24 * h, (r, got["entropy"][r], h)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 255, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 5000, 16384, 16385, 32000,
                               50257])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_sizes(gpu, n, rows, top):
    rng = np.random.default_rng(n + rows)
    x = rng.standard_normal((rows, n)).astype(np.float32) * np.array([1.0, 6.0, 0.1])[:rows, None]
    check(gpu, x, rng.integers(0, n, rows), min(top, n))


@pytest.mark.parametrize("rows,n", [(700, 20000), (600, 16384), (300, 40001), (2000, 100)])
@pytest.mark.parametrize("top", [0, 5])
def test_many_rows(gpu, rows, n, top):
    """Rows enough for the large slices."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    got = run(gpu, x, rng.integers(0, n, rows), top)
    assert all(np.isfinite(v).all() for v in got.values())
    some = rng.permutation(rows)[:12]
    tokens = rng.integers(0, n, rows)
    got = run(gpu, x, tokens, top)
    want = run(gpu, x[some], tokens[some], top)  # (the small slices)
    for i, r in enumerate(some):
        lp, h, best, _ = ref.logprobs(x[r], int(tokens[r]), top)
        bar = 2.0 ** -17 * (1 + abs(lp) / 4)  # (the exact bars: `want` is checked below)
        assert abs(got["logprob"][r] - lp) <= bar and abs(got["entropy"][r] - h) <= bar
        if top:
            assert got["top_tokens"][r * top:(r + 1) * top].tolist() == best
            assert np.abs(got["top_logprobs"][r * top:(r + 1) * top] - want["top_logprobs"][i * top:(i + 1) * top]).max() <= bar
    check(gpu, x[some], tokens[some], top)


@pytest.mark.parametrize("offset,ld", [(0, 5003), (1, 5000), (3, 5001), (2, 5006), (4, 5004)])
@pytest.mark.parametrize("top", [0, 7])
def test_alignment_and_strides(gpu, offset, ld, top):
    rng = np.random.default_rng(ld)
    check(gpu, rng.standard_normal((4, 5000)), rng.integers(0, 5000, 4), top, ld=ld, offset=offset)


@pytest.mark.parametrize("n", [500, 5000, 40000])
def test_rows_of_few_or_equal_logits(gpu, n):
    """Equal logits, a few values, masked ones, none at all: the lowest index first among equals."""
    rng = np.random.default_rng(n)
    inf, nan = np.inf, np.nan
    x = np.zeros((12, n), np.float32)
    x[1] = rng.integers(-3, 3, n)
    x[2] = np.where(rng.random(n) < 0.9, -inf, 1.0)
    x[3] = -inf
    x[4] = nan
    x[5] = -inf
    x[5, [n // 3, n - 1]] = 2.0, nan
    x[6] = np.where(np.arange(n) % 100 < 3, 5.0, -30.0)
    x[7] = rng.standard_normal(n)
    x[7, [5, n // 2, n - 1]] = inf
    x[8] = -0.0
    x[8, ::2] = 0.0
    x[9] = rng.standard_normal(n) * 1e-38
    x[10] = rng.standard_normal(n) * 1e30
    x[11] = -3.4e38
    tokens = rng.integers(0, n, 12)
    tokens[7] = n // 2
    tokens[5] = n // 3
    for top in (0, 1, 32):
        check(gpu, x, tokens, top)


def test_tokens_outside_the_row(gpu):
    x = np.random.default_rng(2).standard_normal((4, 300))
    check(gpu, x, [-1, 300, 2 ** 31 - 1, -2 ** 31])


def test_outputs_by_themselves(gpu):
    x = np.random.default_rng(3).standard_normal((2, 9000)).astype(np.float32)
    whole = run(gpu, x, [4, 5], 6)
    assert run(gpu, x, [4, 5], entropy=False)["logprob"].tolist() == whole["logprob"].tolist()
    assert run(gpu, x)["entropy"].tolist() == whole["entropy"].tolist()
    X = gpu.DeviceBuffer.from_array(x)
    T, L = gpu.DeviceBuffer(4 * 12), gpu.DeviceBuffer(4 * 12)
    ws = gpu.logprobs_workspace(2, 9000, 6)
    gpu.logprobs(X, 2, 9000, 9000, top=6, top_tokens=T, workspace=ws)
    gpu.logprobs(X, 2, 9000, 9000, top=6, top_logprobs=L, workspace=ws)
    gpu.synchronize()
    assert T.download(np.int32).tolist() == whole["top_tokens"].tolist()
    assert L.download(np.float32).tolist() == whole["top_logprobs"].tolist()


def test_a_row_does_not_depend_on_the_others(gpu):
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((5, 30000)) * 4).astype(np.float32)
    tokens = rng.integers(0, 30000, 5)
    whole = run(gpu, x, tokens, 8)
    for r in range(5):
        one = run(gpu, x[r:r + 1], tokens[r:r + 1], 8)
        for k, v in one.items():
            assert np.array_equal(v, whole[k].reshape(5, -1)[r])


@pytest.mark.parametrize("rows,n,top", [(3, 30000, 20), (700, 20000, 0), (5, 2000, 4)])
def test_replayed_from_a_graph(gpu, rows, n, top):
    rng = np.random.default_rng(5)
    X, T = gpu.DeviceBuffer(4 * rows * n), gpu.DeviceBuffer(4 * rows)
    out = {k: gpu.DeviceBuffer(4 * rows * max(w, 1)) for k, w in (("logprob", 1), ("entropy", 1), ("top_tokens", top),
                                                                 ("top_logprobs", top))}
    if not top:
        out["top_tokens"] = out["top_logprobs"] = None
    ws, stream = gpu.logprobs_workspace(rows, n, top), gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.logprobs(X, rows, n, n, tokens=T, top=top, workspace=ws, stream=stream, **out))
    for _ in range(3):
        x = rng.standard_normal((rows, n)).astype(np.float32)
        tokens = rng.integers(0, n, rows).astype(np.int32)
        X.upload(x)
        T.upload(tokens)
        graph.launch(stream)
        stream.synchronize()
        want = run(gpu, x, tokens, top)
        for k, v in want.items():
            assert np.array_equal(out[k].download(v.dtype), v)
    graph.close()


@pytest.mark.parametrize("slices", [5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256])
@pytest.mark.parametrize("top", [1, 31, 32])
def test_joins_of_any_number_of_slices(gpu, slices, top):
    """Slices of 1024 logits, the last of one, a few or all; the likeliest tokens all in one slice, or far apart."""
    rng = np.random.default_rng(slices)
    for n in (1024 * slices - 1023, 1024 * slices - 1000, 1024 * slices):
        x = rng.standard_normal((3, n)).astype(np.float32)
        x[1, -40 if n % 1024 == 0 else 2048 - 40:][:40] += 10
        x[2, ::max(n // 20, 1)] = 7  # (equal ones)
        check(gpu, x, rng.integers(0, n, 3), top)


@pytest.mark.parametrize("rows,n", [(4, 8191), (4, 8192), (4, 8193), (520, 8192), (520, 8193), (600, 16000), (300, 32000)])
@pytest.mark.parametrize("top", [0, 32])
def test_rows_next_to_the_borders_of_the_forms(gpu, rows, n, top):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((rows, n)).astype(np.float32) * 3
    check(gpu, x, rng.integers(0, n, rows), top)


def test_the_largest_row(gpu):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 1 << 20)).astype(np.float32)
    check(gpu, x, [1 << 19], 32)
