"""rqmv_logprobs of the longest rows (slices of 1,024, 2,048 and 4,096 logits a wave), and of more long rows than a grid has
in y, with the bars of test_gpu_logprobs.py."""
import numpy as np
import pytest

from tests.test_gpu_logprobs import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [262143, 262144, 262145, 500000, 524288, 524289, 1000003, 1 << 20])
@pytest.mark.parametrize("top", [0, 1, 32])
def test_long_rows(gpu, n, top):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((2, n)).astype(np.float32) * np.array([[1.0], [4.0]], np.float32)
    x[1, -3:] = 30.0  # (the likeliest in the last, partial slice)
    check(gpu, x, [n - 1, n // 2], top)


@pytest.mark.parametrize("n,top", [(8193, 0), (4097, 3)])
def test_more_rows_than_a_grid_has_in_y(gpu, n, top):
    """Rows by slices: a row's outputs are what it has among few."""
    rng = np.random.default_rng(n)
    few, rows = 509, 65540
    x = (rng.standard_normal((few, n)) * 3).astype(np.float32)
    tokens = rng.integers(0, n, few)
    check(gpu, x[:12], tokens[:12], top)
    want = run(gpu, x, tokens, top)
    at = np.arange(rows) % few
    got = run(gpu, x[at], tokens[at], top)
    for k, v in got.items():
        assert np.array_equal(v.reshape(rows, -1), want[k].reshape(few, -1)[at]), k
