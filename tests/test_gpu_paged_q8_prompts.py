"""The append to 8-bit pages in calls of more than 512 rows (its form for prompts), and the values of a large cache, against the
64-bit references of oracle/paged.py. Codes and scales are equal, queries rqmv_qk_norm_rope's bit for bit (run_append)."""
import numpy as np
import pytest

from oracle import paged as ref
from tests.test_gpu_paged_q8 import pages_of, random_pages, run_append

pytestmark = pytest.mark.gpu


def in_order(rng, tokens, blocks, block):
    """Sequences in order over shuffled pages, each from any position of its first page on."""
    pages, slots = list(rng.permutation(blocks)), []
    while len(slots) < tokens:
        p, end = int(rng.integers(0, block)), int(rng.integers(1, 400))
        page = pages.pop()
        for i in range(p, p + end):
            if i > p and i % block == 0:
                page = pages.pop()
            slots.append(int(page) * block + i % block)
    return slots[:tokens]


def rolling(rng, tokens, blocks, block):
    """Several groups at a time in turns, rows without a slot between them; a group's rows within 32."""
    groups, slots, live = list(rng.permutation(blocks * block // 16)), [], []
    for row in range(tokens):
        live = [g for g in live if g[0] > row - 32 and g[1]]
        pick = rng.random()
        if pick < 0.1:
            slots.append(-1 if pick < 0.05 else blocks * block + int(rng.integers(0, 100)))
            continue
        if not live or (len(live) < 6 and pick < 0.25):
            live.append((row, list(rng.permutation(16)[:rng.integers(1, 17)]), groups.pop()))
        _, left, g = live[rng.integers(0, len(live))]
        slots.append(int(g) * 16 + int(left.pop()))
    return slots


def one_each(rng, tokens, blocks, block):
    """A decode step of as many requests: a row a group."""
    return (rng.permutation(blocks * block // 16)[:tokens] * 16 + rng.integers(0, 16, tokens)).tolist()


def check(gpu, tokens, make, nq, nkv, hd, rot, block, x_f16, q_f16, norm, seed):
    rng = np.random.default_rng(seed)
    blocks, rows, wide = -(-tokens * 16 // block) + 40, 500, (nq + 2 * nkv) * hd
    slots = np.array(make(rng, tokens, blocks, block), np.int32)
    stored = slots[(slots >= 0) & (slots < blocks * block)]
    assert len(slots) == tokens and len(np.unique(stored)) == len(stored)
    for g in np.unique(stored // 16):
        at = np.nonzero(slots // 16 == g)[0]
        assert at[-1] - at[0] < 32
    x = rng.standard_normal((tokens, wide)) * np.exp2(rng.integers(-3, 4, (tokens, 1)))
    x = x.astype(np.float16 if x_f16 else np.float32)
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if norm else None
    pos = rng.integers(0, rows, tokens)
    old = [random_pages(rng, blocks, nkv, block, hd) for _ in range(2)]
    table = gpu.rope_table(rot, 10000.0, rows)
    _, got = run_append(gpu, x, nq, (old[0][0], old[1][0]), (old[0][1], old[1][1]), slots, pos, table, rows, rot, w, 1e-5,
                        x_f16, q_f16)
    cs = table.download(np.float32).reshape(rows, rot // 2, 2)
    _, k, v = ref.qk_norm_rope(x, nq, nkv, hd, *(w or (None, None)), np.float32(1e-5), cs, rot, pos)
    for (c, s), y, at in ((old[0], k, 0), (old[1], v, 2)):
        codes, scale = ref.store_q8(c, s, y, slots)
        assert np.array_equal(got[at + 1], scale)
        live = np.repeat(scale != 255, 16, axis=2)  # (codes of NaN groups stand for nothing)
        assert np.array_equal(got[at][live], codes[live])


@pytest.mark.parametrize("make,tokens", [(in_order, 1000), (rolling, 777), (one_each, 513)])
@pytest.mark.parametrize("nq,nkv,hd,rot,block", [(3, 2, 64, 64, 16), (4, 1, 128, 96, 64), (2, 1, 256, 256, 256)])
@pytest.mark.parametrize("x_f16,q_f16,norm", [(False, False, True), (False, True, False), (True, True, True),
                                              (True, False, False)])
def test_append_of_many_rows(gpu, make, tokens, nq, nkv, hd, rot, block, x_f16, q_f16, norm):
    check(gpu, tokens, make, nq, nkv, hd, rot, block, x_f16, q_f16, norm, hd + tokens)


@pytest.mark.parametrize("make", [in_order, rolling, one_each])
def test_append_of_a_prefill_step(gpu, make):
    """Many heads: runs of each in their own part of the grid."""
    check(gpu, 3480, make, 8, 3, 128, 128, 32, False, True, True, 3480)


@pytest.mark.parametrize("tokens", [511, 512, 513, 528, 529])
def test_append_next_to_the_border_of_the_forms(gpu, tokens):
    check(gpu, tokens, rolling, 2, 2, 64, 32, 32, False, False, True, tokens)


def test_values_of_a_large_cache(gpu):
    """More pieces than one pass of the grid: every value, to the last."""
    rng = np.random.default_rng(2)
    blocks, nkv, block, hd = 2403, 2, 128, 128
    codes = rng.integers(-127, 128, (2, blocks, nkv, block, hd), np.int8)
    assert codes[0].size // 16 > 2 * 8192 * 256  # two passes and a part
    scale = rng.integers(100, 140, (2, blocks, nkv, block // 16)).astype(np.uint8)
    scale[rng.random(scale.shape) < 0.01] = 255
    out = gpu.PagedCache.allocate(blocks, block, nkv, hd)
    gpu.paged_values_q8(pages_of(gpu, codes[0], codes[1], scale[0], scale[1]), out)
    gpu.synchronize()
    for i, buf in enumerate((out.k, out.v)):
        got = buf.download(np.uint16).view(np.float16).reshape(codes[0].shape)
        for b in range(0, blocks, 100):
            want = ref.values_q8(codes[i, b:b + 100], scale[i, b:b + 100])
            assert np.array_equal(got[b:b + 100].astype(np.float64), want, equal_nan=True), b
