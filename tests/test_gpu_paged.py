"""GPU parity of the paged serving operators' tables, norms, rotation and
append (rqmv_paged_plan, rqmv_qk_norm_rope) against the host references of
oracle/paged.py.

Bars: the tables are whole numbers and equal. Norms and rotation are fp32
arithmetic: the sum of squares over at most 256 values in a tree has at most
13 roundings on any path, halved by the square root, then a division, a root, a reciprocal
and two products (1/2 step each, 2^-24 relative), and the rotation adds two
products and a sum relative to the pair's length (sqrt(2) of the larger
magnitude): under 16 half steps, 16 * 2^-24 of the pair's length. Values
rounded to fp16 add half a step of fp16 (2^-11 relative, 2^-25 below its normal
range).
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu


def i32(gpu, a):
    return gpu.DeviceBuffer.from_array(np.asarray(a, np.int32))


# -------------------------------------------------------------------- plan ----

def make_plan(seqs, block, seed, new_hi=9, ctx_hi=200, spare=5):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, ctx_hi + 1, seqs)
    new = rng.integers(0, new_hi + 1, seqs)
    cached[rng.random(seqs) < 0.2] = 0
    cached[rng.random(seqs) < 0.2] //= block
    cached[rng.random(seqs) < 0.2] *= 0
    held = [ref.pages(int(c), block) for c in cached]
    need = [ref.pages(int(c + n), block) for c, n in zip(cached, new)]
    width = max(max(need), 1) + 2
    blocks = sum(need) + spare
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((seqs, width), -7, np.int32)
    at = 0
    for s in range(seqs):
        table[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    return [int(c) for c in cached], [int(n) for n in new], table, ids[at:], blocks


def run_plan(gpu, cached, new, table, free, head, block, blocks, tokens, stride=None, alias=False):
    seqs, width = table.shape
    stride = stride or width
    wide = np.full((seqs, stride), -9, np.int32)
    wide[:, :width] = table
    T, C = i32(gpu, wide), i32(gpu, cached)
    S, P, L = i32(gpu, [-1] * (seqs + 1)), i32(gpu, [-2] * tokens), i32(gpu, [-3] * tokens)
    H, ST = i32(gpu, [head]), i32(gpu, [-4])
    KV = C if alias else i32(gpu, [-5] * seqs)
    HO = H if alias else i32(gpu, [-6])
    batch = gpu.PagedBatch(seqs, tokens, width, S, KV, T, P, L, stride)
    cache = gpu.PagedCache(None, None, blocks, block, 1, 64)
    gpu.paged_plan(batch, cache, C, i32(gpu, new), i32(gpu, free) if len(free) else None, len(free), H, HO, ST)
    gpu.synchronize()
    got = T.download(np.int32).reshape(seqs, stride)
    assert np.all(got[:, width:] == -9)
    return (int(ST.download(np.int32)[0]), S.download(np.int32), KV.download(np.int32), got[:, :width],
            P.download(np.int32), L.download(np.int32), int(HO.download(np.int32)[0]))


def same(got, want):
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("seqs,block,tokens,new_hi", [(1, 16, 1, 1), (1, 256, 700, 700), (7, 16, 64, 9),
                                                      (64, 32, 64, 1), (300, 64, 2048, 11), (300, 16, 2049, 11),
                                                      (1025, 16, 9000, 9), (2500, 128, 2500, 1)])
def test_plan(gpu, seqs, block, tokens, new_hi):
    cached, new, table, free, blocks = make_plan(seqs, block, seqs + tokens, new_hi)
    tokens = max(tokens, sum(new))
    want = ref.plan(cached, new, table, free, 0, block, blocks, tokens)
    assert want[0] == 0
    same(run_plan(gpu, cached, new, table, free, 0, block, blocks, tokens), want)
    same(run_plan(gpu, cached, new, table, free, 0, block, blocks, tokens, table.shape[1] + 3, alias=True), want)


def test_plan_most_sequences(gpu):
    """8192 sequences, one new row for every other one: more than 48 KiB of starts."""
    cached = [i % 33 for i in range(8192)]
    new = [i % 2 for i in range(8192)]
    table = np.full((8192, 3), -1, np.int32)
    at = 0
    for s in range(8192):
        for p in range(ref.pages(cached[s], 16)):
            table[s, p] = at
            at += 1
    free = np.arange(at, at + 4096)
    want = ref.plan(cached, new, table, free, 3, 16, at + 4096, 5000)
    assert want[0] == 0
    same(run_plan(gpu, cached, new, table, free, 3, 16, at + 4096, 5000), want)


@pytest.mark.parametrize("tokens", [40, 4000])
def test_plan_all_or_nothing(gpu, tokens):
    cached, new, table, free, blocks = make_plan(12, 16, 5, new_hi=2)
    need = sum(ref.pages(c + n, 16) - ref.pages(c, 16) for c, n in zip(cached, new))
    room = table.shape[1] * 16
    cases = [(cached, new, free[:need], 0, 0), (cached, new, free[:max(need - 1, 0)], 0, 4), (cached, new, free, -1, 4),
             (cached, new, free, len(free) + 1, 4), (cached[:-1] + [-1], new, free, 0, 1),
             (cached, new[:-1] + [-3], free, 0, 1), (cached[:-1] + [room], new[:-1] + [1], free, 0, 1),
             (cached[:-1] + [2 ** 31 - 1], new[:-1] + [2 ** 31 - 1], free, 0, 1),
             (cached, [n + tokens for n in new], free, 0, None)]
    assert need >= 1
    for c, n, f, head, status in cases:
        want = ref.plan(c, n, table, f, head, 16, blocks, tokens)
        assert status is None or want[0] == status
        same(run_plan(gpu, c, n, table, f, head, 16, blocks, tokens), want)


def test_plan_bad_pages_get_no_slot(gpu):
    """Table or pool entries outside the cache: the rows on them have slot -1."""
    table = np.array([[5, -3, -1], [99, -1, -1]], np.int32)
    free = [2 ** 31 - 1, 3]
    want = ref.plan([20, 3], [20, 2], table, free, 0, 16, 10, 24)
    assert want[0] == 0 and (want[5][:22] == -1).sum() >= 12
    same(run_plan(gpu, [20, 3], [20, 2], table, free, 0, 16, 10, 24), want)


def test_plan_replayed_from_a_graph(gpu):
    """A captured plan, lengths and pool carried on in place: every replay takes one more token a sequence."""
    cached, new, table, free, blocks = make_plan(9, 16, 3, spare=60)
    new, width = [1] * 9, table.shape[1] + 4
    table = np.concatenate((table, np.full((9, 4), -7, np.int32)), 1)
    batch = gpu.PagedBatch(9, 12, width, i32(gpu, [0] * 10), i32(gpu, cached), i32(gpu, table), i32(gpu, [0] * 12),
                           i32(gpu, [0] * 12))
    cache = gpu.PagedCache(None, None, blocks, 16, 1, 64)
    N, F, H, ST = i32(gpu, new), i32(gpu, free), i32(gpu, [0]), i32(gpu, [9])
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.paged_plan(batch, cache, batch.kv_len, N, F, len(free), H, H, ST, stream))
    head = 0
    for _ in range(20):
        want = ref.plan(cached, new, table, free, head, 16, blocks, 12)
        assert want[0] == 0
        graph.launch(stream)
        stream.synchronize()
        got = (int(ST.download(np.int32)[0]), batch.q_start.download(np.int32), batch.kv_len.download(np.int32),
               batch.block_table.download(np.int32).reshape(9, width), batch.positions.download(np.int32),
               batch.slots.download(np.int32), int(H.download(np.int32)[0]))
        same(got, want)
        cached, table, head = [int(v) for v in want[2]], want[3], want[6]
    graph.close()


# -------------------------------------------------- norms, rotation, append ----

def half_steps(x):
    """Half a step of fp16 at x."""
    return np.maximum(np.abs(x) * 2.0 ** -11, 2.0 ** -25)


@pytest.mark.parametrize("nq,nkv,hd,rot,block", [(4, 2, 64, 64, 16), (32, 8, 128, 128, 64), (5, 1, 256, 256, 256),
                                                 (6, 3, 128, 32, 32), (3, 3, 64, 8, 128), (7, 7, 256, 192, 16)])
@pytest.mark.parametrize("tokens", [1, 3, 77])
@pytest.mark.parametrize("x_f16,q_f16,norm", [(False, False, True), (False, True, True), (True, True, False),
                                              (True, False, True), (False, False, False)])
def test_qk_norm_rope(gpu, nq, nkv, hd, rot, block, tokens, x_f16, q_f16, norm):
    rng = np.random.default_rng(nq * hd + tokens)
    rows, blocks, wide, pad = 300, tokens // block + 3, (nq + 2 * nkv) * hd, 24
    x = (rng.standard_normal((tokens, wide + pad)) * 3).astype(np.float16 if x_f16 else np.float32)
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    pos = rng.integers(-5, rows + 5, tokens)  # some outside the table: its nearest row
    slots = rng.permutation(blocks * block)[:tokens].astype(np.int32)
    if tokens > 2:
        slots[0], slots[2] = -1, blocks * block  # outside the cache: nothing stored
    X = gpu.DeviceBuffer.from_array(x.view(np.uint16) if x_f16 else x)
    ldq = nq * hd + 8
    qt = np.float16 if q_f16 else np.float32
    Q = gpu.DeviceBuffer.from_array(np.full((tokens, ldq), 7, qt).view(np.uint16 if q_f16 else np.float32))
    table = gpu.rope_table(rot, 10000.0, rows)
    old = rng.standard_normal((2, blocks, nkv, block, hd)).astype(np.float16)
    K, V = (gpu.DeviceBuffer.from_array(o.view(np.uint16)) for o in old)
    cache = gpu.PagedCache(K, V, blocks, block, nkv, hd)
    batch = gpu.PagedBatch(1, tokens, 1, positions=i32(gpu, pos), slots=i32(gpu, slots))
    norms = {"q_norm": gpu.DeviceBuffer.from_array(w[0]), "k_norm": gpu.DeviceBuffer.from_array(w[1])} if norm else {}
    gpu.qk_norm_rope(batch, cache, X, gpu.DTYPE_F16 if x_f16 else gpu.DTYPE_F32, wide + pad, nq, table, rows, Q,
                     gpu.DTYPE_F16 if q_f16 else gpu.DTYPE_F32, ldq, eps=1e-5, rot_dim=rot, **norms)
    gpu.synchronize()
    cs = table.download(np.float32).reshape(rows, rot // 2, 2)
    q, k, v = ref.qk_norm_rope(x[:, :wide], nq, nkv, hd, w[0] if norm else None, w[1] if norm else None, 1e-5, cs, rot,
                               pos)

    def length(h):  # of each value's rotation pair (of the value itself past the rotated dims)
        n = np.abs(h)
        n[..., :rot] = np.tile(np.hypot(h[..., :rot // 2], h[..., rot // 2:rot]), 2)
        return n

    got = Q.download(np.uint16 if q_f16 else np.float32).view(qt).reshape(tokens, ldq)
    assert np.all(got[:, nq * hd:] == 7)
    off = np.abs(got[:, :nq * hd].reshape(q.shape).astype(np.float64) - q)
    assert np.all(off <= 16 * 2.0 ** -24 * length(q) + (half_steps(q) * (1 + 2.0 ** -11) if q_f16 else 0))
    for buf, new, was, exact in ((K, k, old[0], False), (V, v, old[1], True)):
        cache_now = buf.download(np.uint16).view(np.float16).reshape(blocks, nkv, block, hd)
        want = was.astype(np.float64)
        bar = np.zeros_like(want)
        for t in range(tokens):
            if 0 <= slots[t] < blocks * block:
                want[slots[t] // block, :, slots[t] % block] = new[t]
                bar[slots[t] // block, :, slots[t] % block] = half_steps(new[t]) * (1 + 2.0 ** -11) + \
                    (0 if exact else 16 * 2.0 ** -24 * length(new[t]))
        assert np.all(np.abs(cache_now.astype(np.float64) - want) <= bar)


def test_qk_norm_rope_in_place(gpu):
    """q_out = qkv: the queries' columns change, the keys' and values' stay."""
    rng = np.random.default_rng(4)
    nq, nkv, hd, tokens, wide = 8, 2, 128, 19, 12 * 128
    x = rng.standard_normal((tokens, wide)).astype(np.float32)
    out = []
    for same_buffer in (False, True):
        X, Q = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer(x.nbytes)
        K, V = gpu.DeviceBuffer(2 * 32 * nkv * hd), gpu.DeviceBuffer(2 * 32 * nkv * hd)
        batch = gpu.PagedBatch(1, tokens, 1, positions=i32(gpu, range(tokens)), slots=i32(gpu, range(tokens)))
        gpu.qk_norm_rope(batch, gpu.PagedCache(K, V, 2, 16, nkv, hd), X, gpu.DTYPE_F32, wide, nq,
                         gpu.rope_table(hd, 10000.0, 64), 64, X if same_buffer else Q, gpu.DTYPE_F32, wide)
        gpu.synchronize()
        out.append((X if same_buffer else Q).download(np.float32).reshape(tokens, wide)[:, :nq * hd])
        assert np.array_equal(X.download(np.float32).reshape(tokens, wide)[:, nq * hd:], x[:, nq * hd:])
    assert np.array_equal(out[0], out[1])


def test_qk_norm_rope_matches_the_single_token_form(gpu):
    """Without norms, at a whole-head rotation, the cache rows are those of rqmv_rope_kv within an fp16 rounding."""
    rng = np.random.default_rng(9)
    nq, nkv, hd, pos = 4, 2, 64, 37
    x = rng.standard_normal((nq + 2 * nkv) * hd).astype(np.float32)
    X, Y = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer.from_array(x)
    bufs = [gpu.DeviceBuffer(2 * 64 * nkv * hd) for _ in range(4)]
    gpu.rope_kv(X, i32(gpu, [pos]), nq, nkv, hd, 10000.0, bufs[0], bufs[1], 64)
    batch = gpu.PagedBatch(1, 1, 1, positions=i32(gpu, [pos]), slots=i32(gpu, [pos]))
    gpu.qk_norm_rope(batch, gpu.PagedCache(bufs[2], bufs[3], 1, 64, nkv, hd), Y, gpu.DTYPE_F32, 0, nq,
                     gpu.rope_table(hd, 10000.0, 64), 64, Y, gpu.DTYPE_F32, 0)
    gpu.synchronize()
    k0, v0, k1, v1 = (b.download(np.uint16).view(np.float16).reshape(nkv, 64, hd)[:, pos].astype(np.float64)
                      for b in bufs)
    assert np.array_equal(v0, v1)
    assert np.all(np.abs(k0 - k1) <= 2 * half_steps(k0) * (1 + 2.0 ** -10) + 2.0 ** -22 * 6)
    q0, q1 = (b.download(np.float32)[:nq * hd].astype(np.float64) for b in (X, Y))
    assert np.all(np.abs(q0 - q1) <= 2.0 ** -21 * 6)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_qk_norm_rope_keeps_non_finite_heads_apart(gpu, bad):
    """A NaN or an infinity spoils its own head of its own row and nothing else."""
    rng = np.random.default_rng(2)
    nq, nkv, hd, tokens = 4, 2, 128, 3
    x = rng.standard_normal((tokens, (nq + 2 * nkv) * hd)).astype(np.float32)
    x[1, 2 * hd + 5] = bad       # query head 2 of row 1
    x[2, (nq + 1) * hd + 9] = bad  # key head 1 of row 2
    X, Q = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer(4 * tokens * nq * hd)
    K, V = gpu.DeviceBuffer(2 * 16 * nkv * hd), gpu.DeviceBuffer(2 * 16 * nkv * hd)
    w = gpu.DeviceBuffer.from_array(np.ones(hd, np.float32))
    batch = gpu.PagedBatch(1, tokens, 1, positions=i32(gpu, [3, 4, 5]), slots=i32(gpu, [0, 1, 2]))
    gpu.qk_norm_rope(batch, gpu.PagedCache(K, V, 1, 16, nkv, hd), X, gpu.DTYPE_F32, (nq + 2 * nkv) * hd, nq,
                     gpu.rope_table(hd, 10000.0, 16), 16, Q, gpu.DTYPE_F32, nq * hd, w, w)
    gpu.synchronize()
    q = Q.download(np.float32).reshape(tokens, nq, hd)
    k = K.download(np.uint16).view(np.float16).reshape(nkv, 16, hd)[:, :tokens]
    assert not np.isfinite(q[1, 2]).any() or np.isnan(q[1, 2]).any()
    q[1, 2] = 0
    assert np.isfinite(q).all()
    assert not np.isfinite(k[1, 2]).all() and np.isfinite(k[0]).all() and np.isfinite(k[1, :2]).all()
