"""Which form of rqmv_paged_attention_q8 takes a batch, by the size of its workspace, and the form for many rows with its keys split.

The workspace serves both types of rows. The form for few rows has parts wherever the table reaches more than 256
positions; the one for many rows has none where its keys are whole, and with S splits a part of head_dim + 2 floats for each split,
token and query head, and 8 bytes for each token and head of a group. So a size of 0 over a longer table says that both
types take the form for many rows, keys whole.
"""
import numpy as np
import pytest

from tests.test_gpu_paged_attention import LARGE
from tests.test_gpu_paged_q8 import Case8

pytestmark = pytest.mark.gpu

# (nq, nkv, block, sequences, splits) at 128 dims, fp16 rows
SPLIT = [(64, 1, 32, [(261, 700)], 3), (64, 1, 16, [(100, 900), (161, 30)], 3), (32, 2, 64, [(590, 500)], 3),
         (32, 8, 16, [(700, 130), (180, 260)], 2), (16, 2, 128, [(1040, 150)], 3)]


def workspace(gpu, tokens, seqs, positions, nq, nkv, hd, block=16):
    batch = gpu.PagedBatch(seqs, tokens, -(-positions // block))
    some = gpu.DeviceBuffer(256)
    return gpu.paged_attention_q8_workspace_size(batch, gpu.PagedCacheQ8(some, some, some, some, 1, block, nkv, hd), nq)


def split_size(tokens, nq, nkv, hd, splits):
    return splits * tokens * nq * (hd * 4 + 8) + tokens * (nq // nkv) * 8


@pytest.mark.parametrize("nq,nkv,hd,block", LARGE)
def test_sizes_with_many_rows(gpu, nq, nkv, hd, block):
    """The batches of test_many_rows and of the tests of masked places, where their tables are long enough to say."""
    for tokens, seqs in ((272, 1), (272, 4), (277, 2), (270, 1)):
        assert workspace(gpu, tokens, seqs, 600, nq, nkv, hd, block) == 0


@pytest.mark.parametrize("hd", [64, 256])
def test_keys_are_never_split_at_64_and_256_dims(gpu, hd):
    """From the fewest rows on that take the form for many, the tiles take more than half of the CUs."""
    for nq, nkv in ((64, 1), (128, 2), (126, 18), (132, 44), (130, 26), (32, 8), (8, 8), (1, 1), (1024, 1024), (1024, 1), (200, 200)):
        first = next(t for t in range(1, 40000) if t * nq // 32 > 1024 and t * (nq // nkv) > 128)
        for tokens in (first, first + 1, first + 31, 2 * first):
            assert workspace(gpu, tokens, 1, 6000, nq, nkv, hd) == 0, (nq, nkv, tokens)
        assert workspace(gpu, first - 1, 1, 6000, nq, nkv, hd) > 0


@pytest.mark.parametrize("window", [0, 333])
@pytest.mark.parametrize("nq,nkv,block,seqs,splits", SPLIT)
def test_many_rows_split_keys(gpu, nq, nkv, block, seqs, splits, window):
    c = Case8(seqs, nq, nkv, 128, block, True, len(seqs) + nq, extra_rows=1)
    assert workspace(gpu, c.rows, len(seqs), c.width * block, nq, nkv, 128, block) == split_size(c.rows, nq, nkv, 128, splits)
    c.check(gpu, window=window)
    Case8(seqs, nq, nkv, 128, block, True, 28, spread=3.0).check(gpu, window=window, scale=0.3)


def test_many_rows_split_keys_of_masked_places(gpu):
    """NaN groups that nobody uses, one in the middle that rows of all splits see, and one at the end."""
    nq, nkv, block, new, ctx = 64, 1, 32, 270, 500
    c = Case8([(new, ctx)], nq, nkv, 128, block, True, 11)
    assert workspace(gpu, new, 1, c.width * block, nq, nkv, 128, block) == split_size(new, nq, nkv, 128, 3)
    clean = c.run(gpu)
    used = np.zeros((c.blocks, c.block // 16), bool)
    p = np.arange(new + ctx)
    used[c.table[0, p // block], p % block // 16] = True
    for cache in (c.k, c.v):
        parts = cache.reshape(c.blocks, nkv, c.block // 16, 16, 128)
        parts.transpose(0, 2, 1, 3, 4)[~used] = np.nan
    c.encode()
    assert np.array_equal(c.run(gpu), clean)
    for name, at in (("v", new + ctx - 1), ("k", new + ctx - 40), ("v", ctx + 20)):
        getattr(c, name)[c.table[0, at // block], 0, at % block, 5] = np.nan
        c.encode()
        first = max(at // 16 * 16 - ctx, 0)  # (the group's first position)
        got = c.run(gpu)
        assert np.array_equal(got[:first], clean[:first]) and np.isnan(got[first:]).all()
