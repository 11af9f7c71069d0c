"""Pins of the paged serving references (oracle/paged.py) on the CPU."""
import numpy as np
import pytest
from scipy.special import softmax

from oracle import decode, paged


def test_plan_by_hand():
    table = np.full((3, 4), -1, np.int32)
    table[0, :2] = (7, 8)  # 20 positions in pages of 16
    table[2, 0] = 5        # exactly one page
    got = paged.plan([20, 0, 16], [1, 17, 2], table, [9, 3, 4, 1, 2], 1, 16, 10, 22)
    status, q_start, kv_len, out, positions, slots, head = got
    assert status == 0 and head == 4
    assert list(q_start) == [0, 1, 18, 20] and list(kv_len) == [21, 17, 18]
    assert out.tolist() == [[7, 8, -1, -1], [3, 4, -1, -1], [5, 1, -1, -1]]
    assert list(positions) == [20] + list(range(17)) + [16, 17, 0, 0]
    assert list(slots) == [8 * 16 + 4] + list(range(48, 64)) + [64, 16, 17, -1, -1]


@pytest.mark.parametrize("cached,new,head,status", [([20], [45], 0, 1), ([-1], [1], 0, 1), ([0], [30], 0, 2),
                                                    ([0], [17], 4, 4), ([0], [1], 6, 4), ([0], [40], 4, 6)])
def test_plan_refusals(cached, new, head, status):
    table = np.full((1, 4), -1, np.int32)
    got = paged.plan(cached, new, table, [1, 2, 3, 4, 5], head, 16, 8, 20)
    assert got[0] == status and not got[1].any() and list(got[2]) == cached
    assert np.array_equal(got[3], table) and (got[5] == -1).all() and got[6] == head


def test_norm_and_rotation_by_complex_numbers():
    """Against a complex multiplication."""
    rng = np.random.default_rng(0)
    nq, nkv, hd, eps = 4, 2, 64, 1e-5
    pos = [0, 3, 17]
    x = rng.standard_normal((3, (nq + 2 * nkv) * hd))
    w = rng.standard_normal(hd)
    angle = np.arange(32)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    table = np.stack((np.cos(angle), np.sin(angle)), -1)
    q, k, v = paged.qk_norm_rope(x, nq, nkv, hd, w, w, eps, table, hd, pos)
    for t in range(3):
        heads = x[t].reshape(-1, hd)
        for h in range(nq + nkv):
            y = heads[h] / np.sqrt(np.mean(heads[h] ** 2) + eps) * w
            z = (y[:hd // 2] + 1j * y[hd // 2:]) * np.exp(1j * pos[t] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd))
            got = q[t, h] if h < nq else k[t, h - nq]
            assert np.allclose(got, np.concatenate((z.real, z.imag)), rtol=0, atol=1e-12)
        assert np.array_equal(v[t], heads[nq + nkv:])
    partial = paged.qk_norm_rope(x, nq, nkv, hd, None, None, 0.0, table[:, :8], 16, pos)[0]
    assert np.array_equal(partial[..., 16:], x.reshape(3, -1, hd)[:, :nq, 16:])


@pytest.mark.parametrize("window", [0, 1, 5])
def test_attention_by_brute_force(window):
    rng = np.random.default_rng(1)
    nq, nkv, hd, block, kv, new = 6, 2, 8, 4, 11, 3
    k, v = (rng.standard_normal((5, nkv, block, hd)) for _ in range(2))
    table = np.array([[3, 0, 4]])
    q = rng.standard_normal((4, nq, hd))
    out = paged.attention(q, k, v, [0, new], [kv], table, 3, 0.4, window)
    keys = np.concatenate([k[b] for b in table[0]], 1)[:, :kv]  # [nkv, positions, hd]
    values = np.concatenate([v[b] for b in table[0]], 1)[:, :kv]
    for i in range(new):
        last = kv - new + i
        seen = slice(max(0, last - window + 1) if window else 0, last + 1)
        for h in range(nq):
            w = softmax(0.4 * keys[h // 3, seen] @ q[i, h])
            assert np.allclose(out[i, h], w @ values[h // 3, seen], rtol=0, atol=1e-13)
    assert np.isnan(out[new:]).all()  # a row of no sequence
    gone = paged.attention(q, k, v, [0, new], [kv], np.array([[-1, 5, 9]]), 3, 0.4, window)
    assert not gone[:new].any()


def test_attention_of_one_token_is_the_decode_steps():
    rng = np.random.default_rng(2)
    nq, nkv, hd, kv = 4, 2, 64, 21
    keys, values = (rng.standard_normal((nkv, kv, hd)) for _ in range(2))
    q = rng.standard_normal((1, nq, hd))
    k, v = (np.zeros((2, nkv, 16, hd)) for _ in range(2))
    for cache, src in ((k, keys), (v, values)):
        for p in range(kv):
            cache[p // 16, :, p % 16] = src[:, p]
    out = paged.attention(q, k, v, [0, 1], [kv], np.array([[0, 1]]), 2, hd ** -0.5)
    assert np.allclose(out[0].reshape(-1), decode.attention(q[0], keys, values, kv).reshape(-1), rtol=0, atol=1e-12)


def test_sample_takes_each_token_for_its_share_of_u():
    rng = np.random.default_rng(3)
    logits = rng.standard_normal(12).astype(np.float32)
    logits[4] = logits[9]  # equals: the lower index first
    order = sorted(range(12), key=lambda i: (-logits[i], i))
    p = softmax(logits.astype(np.float64) / 0.7)
    steps = 20000
    for kw, kept in (({}, order), ({"top_k": 5}, order[:5]),
                     ({"min_p": 0.2}, [i for i in order if p[i] >= 0.2 * p.max()]),
                     ({"top_p": 0.6}, order[:1 + int(np.sum(np.cumsum(p[order]) < 0.6))]),
                     ({"top_k": 6, "top_p": 0.5, "min_p": 0.05}, None)):
        if kept is None:
            first = order[:6]
            part = np.cumsum(p[first]) / p[first].sum()
            kept = [i for i in first[:1 + int(np.sum(part < 0.5))] if p[i] >= 0.05 * p.max()]
        share = p[kept] / p[kept].sum()
        ends = np.cumsum(share)
        for u in (np.arange(steps // 100) + 0.5) / (steps // 100):
            token, prob = paged.sample(logits, u, 0.7, **kw)
            at = int(np.searchsorted(ends, u, side="right"))
            assert token == kept[at] and abs(prob - share[at]) < 1e-12


def test_sample_edges():
    nan, inf = np.nan, np.inf
    assert paged.sample([nan, -inf, nan], 0.5) == (-1, 0.0)
    assert paged.sample([1.0, 3.0, nan, 3.0], 0.99, temperature=0.0) == (1, 1.0)
    assert paged.sample([0.0, 0.0, -inf], 0.5)[0] == 1 and paged.sample([0.0, 0.0], 0.4999)[0] == 0
    assert paged.sample([0.0, 1.0, 0.0], 1.0)[0] == 2 and paged.sample([0.0, 1.0], -1.0)[0] == 1
    assert paged.sample([0.0, 1.0, 0.5], 0.9, top_p=0.0) == (1, 1.0)
