"""What keys and values of 8 bits cost attention: over the pages' values against over the rows before they were rounded, in 64 bits.

The step of a group is 1 to 2 times amax / 127 of sixteen rows of all dims, so with normal values (amax about 3.6) it is 0.03 to 0.06 and
a value is off by 0.01 to 0.02 of its standard deviation; a channel ten times larger than the rest makes that 0.1 to 0.2 of theirs."""
import numpy as np
import pytest

from oracle import paged as ref


def off(larger, queries, seed=0, n=2048, hd=128):
    """Relative 2-norm of the outputs' error, over 32 queries; two key channels `larger` times the others, and their queries as much smaller
    as keeps the scores' spread."""
    rng = np.random.default_rng(seed)
    k, v = rng.standard_normal((n, 1, hd)), rng.standard_normal((n, 1, hd))
    q = rng.standard_normal((32, hd)) * queries
    k[..., :2] *= larger
    q[:, :2] /= np.sqrt(larger)
    empty = np.zeros((n // 64, 1, 64, hd), np.int8), np.zeros((n // 64, 1, 4), np.uint8)

    def kept(y):
        return ref.values_q8(*ref.store_q8(*empty, y, range(n))).transpose(0, 2, 1, 3).reshape(n, hd)

    def attend(keys, values):
        s = q @ keys.T / np.sqrt(hd)
        e = np.exp(s - s.max(1, keepdims=True))
        return e / e.sum(1, keepdims=True) @ values

    want = attend(k[:, 0], v[:, 0])
    return np.linalg.norm(attend(kept(k), kept(v)) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("larger,queries,low,high", [(1, 1.5, 0.012, 0.025), (1, 4.0, 0.018, 0.035), (10, 1.5, 0.07, 0.18),
                                                     (30, 1.5, 0.2, 0.6)])
def test_attention_over_rounded_keys_and_values(larger, queries, low, high):
    assert low < off(larger, queries) < high
