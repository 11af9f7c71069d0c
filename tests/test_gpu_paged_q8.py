"""GPU parity of the 8-bit pages (rqmv_qk_norm_rope_q8, rqmv_paged_values_q8,
rqmv_paged_attention_q8) against the 64-bit references of oracle/paged.py.

Codes and scales are whole numbers and equal the reference's: both are rounded
from 64-bit keys. (The two sum a head's squares in different orders, so a key is
the same to 2^-48 and a code could differ where a key lies that close to a
border; the inputs below have none.) Queries are rqmv_qk_norm_rope's, bit for
bit. Attention has the bars of test_gpu_paged_attention.py on the values that the pages stand for, and one term more.
Those bars take every error of a weight relative to the weight, but weights have smallest steps too: fp32 rows carry
2^15 w (w <= 1 of the row's largest) as two fp16 parts, the second rounded to within 2^-25, so w to within 2^-40; fp16
rows carry 2^6 w as one, w to within 2^-31 of the largest. With random fp16 values that is far below the rest, but codes
are often exactly 0: where the value of the one key that matters is, the row is the sum of weights of 1e-10 and less. (Seed
27 of test_many_rows_split_keys, fp32: row 85, head 30 has sum w |v| = 3.3e-11. The two-part weights alone, taken in
numpy, put it off by 1.2e-12, 11.9 times the relative bars.) A row of n keys is off by
n 2^-40 (n 2^-31) times the largest |v| at most, its weight sum being 1 or more.
"""
import numpy as np
import pytest

from oracle import paged as ref
from tests.test_gpu_paged_attention import HEADS, LARGE, SPLIT, Case

pytestmark = pytest.mark.gpu


def i32(gpu, a):
    return gpu.DeviceBuffer.from_array(np.asarray(a, np.int32))


def u8(gpu, a):
    return gpu.DeviceBuffer.from_array(np.ascontiguousarray(a).view(np.uint8))


def random_pages(rng, blocks, nkv, block, hd):
    """Codes and scale bytes as earlier steps left them: groups of unlike size, a few of them NaN."""
    codes = rng.integers(-127, 128, (blocks, nkv, block, hd)).astype(np.int8)
    scale = rng.integers(115, 125, (blocks, nkv, block // 16)).astype(np.uint8)
    scale[rng.random(scale.shape) < 0.05] = 255
    return codes, scale


def pages_of(gpu, k, v, ks, vs):
    blocks, nkv, block, hd = k.shape
    return gpu.PagedCacheQ8(u8(gpu, k), u8(gpu, v), u8(gpu, ks), u8(gpu, vs), blocks, block, nkv, hd)


def pages_back(cache, shape):
    groups = shape[:2] + (shape[2] // 16,)
    return (cache.k.download(np.int8).reshape(shape), cache.k_scale.download(np.uint8).reshape(groups),
            cache.v.download(np.int8).reshape(shape), cache.v_scale.download(np.uint8).reshape(groups))


# ------------------------------------------------------------------ values ----

@pytest.mark.parametrize("nkv,hd,block", [(1, 64, 16), (3, 128, 32), (2, 256, 256)])
def test_values(gpu, nkv, hd, block):
    """Every scale byte with codes of every size; bytes outside 103..136 count as the nearest."""
    rng = np.random.default_rng(nkv)
    blocks = -(-256 * 16 // (block * nkv))
    codes = rng.integers(-127, 128, (2, blocks, nkv, block, hd)).astype(np.int8)
    scale = np.resize(np.arange(256), (2, blocks, nkv, block // 16)).astype(np.uint8)
    scale[1] = scale[1][::-1]
    cache = pages_of(gpu, codes[0], codes[1], scale[0], scale[1])
    out = gpu.PagedCache.allocate(blocks, block, nkv, hd)
    gpu.paged_values_q8(cache, out)
    gpu.synchronize()
    for i, buf in enumerate((out.k, out.v)):
        got = buf.download(np.uint16).view(np.float16).reshape(codes[0].shape).astype(np.float64)
        assert np.array_equal(got, ref.values_q8(codes[i], scale[i]), equal_nan=True)


# ------------------------------------------------------------------ append ----

def run_append(gpu, x, nq, codes, scale, slots, pos, table, rows, rot, norm, eps, x_f16=False, q_f16=False, stream=None,
               into=None):
    """One call; (queries, pages after it)."""
    k, v = codes
    blocks, nkv, block, hd = k.shape
    tokens, wide = x.shape
    X = gpu.DeviceBuffer.from_array(x.view(np.uint16) if x_f16 else x)
    qt, ldq = (np.float16 if q_f16 else np.float32), nq * hd + 8
    Q = gpu.DeviceBuffer.from_array(np.full((tokens, ldq), 7, qt).view(np.uint16 if q_f16 else np.float32))
    cache = pages_of(gpu, k, v, *scale)
    batch = gpu.PagedBatch(1, tokens, 1, positions=i32(gpu, pos), slots=i32(gpu, slots))
    norms = {"q_norm": gpu.DeviceBuffer.from_array(norm[0]), "k_norm": gpu.DeviceBuffer.from_array(norm[1])} if norm else {}
    dt = {True: gpu.DTYPE_F16, False: gpu.DTYPE_F32}
    args = (X, dt[x_f16], wide, nq, table, rows, Q, dt[q_f16], ldq)
    gpu.qk_norm_rope_q8(batch, cache, *args, eps=eps, rot_dim=rot, stream=stream, **norms)
    gpu.synchronize()
    q = Q.download(np.uint16 if q_f16 else np.float32).view(qt).reshape(tokens, ldq)
    # the queries of the form over fp16 pages
    plain = gpu.PagedCache.allocate(blocks, block, nkv, hd)
    gpu.qk_norm_rope(batch, plain, *args, eps=eps, rot_dim=rot, stream=stream, **norms)
    gpu.synchronize()
    same = Q.download(np.uint16 if q_f16 else np.float32).view(qt).reshape(tokens, ldq)
    bits = np.uint16 if q_f16 else np.uint32
    assert np.array_equal(q.view(bits), same.view(bits))
    return q, pages_back(cache, k.shape)


def runs(rng, tokens, blocks, block, longest):
    """Slots in runs of up to `longest` within a group, groups in any order, slots within them too."""
    slots, groups = [], rng.permutation(blocks * block // 16)
    for g in groups:
        n = int(rng.integers(1, longest + 1))
        at = rng.permutation(16)[:n] if rng.random() < 0.5 else np.arange(n) + rng.integers(0, 17 - n)
        slots += [int(g) * 16 + int(a) for a in at]
        if len(slots) >= tokens:
            break
    return np.array(slots[:tokens], np.int32)


@pytest.mark.parametrize("nq,nkv,hd,rot,block", [(4, 2, 64, 64, 16), (32, 8, 128, 128, 64), (5, 1, 256, 256, 256),
                                                 (6, 3, 128, 32, 32), (3, 3, 64, 8, 128), (7, 7, 256, 192, 16)])
@pytest.mark.parametrize("tokens,longest", [(1, 1), (3, 2), (77, 16), (61, 1)])
@pytest.mark.parametrize("x_f16,q_f16,norm", [(False, False, True), (False, True, False), (True, True, True),
                                              (True, False, False)])
def test_append(gpu, nq, nkv, hd, rot, block, tokens, longest, x_f16, q_f16, norm):
    rng = np.random.default_rng(nq * hd + tokens)
    rows, blocks, wide, pad = 300, -(-tokens * 16 // block) + 2, (nq + 2 * nkv) * hd, 24
    size = np.exp2(rng.integers(-3, 4, tokens))[:, None]  # rows of unlike size
    x = (rng.standard_normal((tokens, wide + pad)) * size).astype(np.float16 if x_f16 else np.float32)
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if norm else None
    pos = rng.integers(-5, rows + 5, tokens)  # some outside the table: its nearest row
    slots = runs(rng, tokens, blocks, block, longest)
    if tokens > 3:
        slots[[0, tokens // 2]] = -1, blocks * block  # outside the cache: nothing stored
    old = [random_pages(rng, blocks, nkv, block, hd) for _ in range(2)]
    table = gpu.rope_table(rot, 10000.0, rows)
    q, got = run_append(gpu, x, nq, (old[0][0], old[1][0]), (old[0][1], old[1][1]), slots, pos, table, rows, rot, w, 1e-5,
                        x_f16, q_f16)
    assert np.all(q[:, nq * hd:] == 7)
    cs = table.download(np.float32).reshape(rows, rot // 2, 2)
    _, k, v = ref.qk_norm_rope(x[:, :wide], nq, nkv, hd, *(w or (None, None)), np.float32(1e-5), cs, rot, pos)
    for (c, s), y, at in ((old[0], k, 0), (old[1], v, 2)):
        codes, scale = ref.store_q8(c, s, y, slots)
        assert np.array_equal(got[at + 1], scale)
        live = np.repeat(scale != 255, 16, axis=2)  # (codes of NaN groups stand for nothing)
        assert np.array_equal(got[at][live], codes[live])


def test_append_rows_of_several_groups_in_turn(gpu):
    """Two groups' rows alternating, rows without a slot between them: a group's 32 rows apart at most."""
    rng = np.random.default_rng(6)
    nq, nkv, hd, block = 2, 2, 64, 16
    slots = np.full(100, -1, np.int32)
    slots[3:35:2] = 16 + rng.permutation(16)
    slots[4:36:2] = 48 + rng.permutation(16)
    slots[36:66:3] = 64 + rng.permutation(16)[:10]
    slots[[69, 99]] = 80, 97
    x = rng.standard_normal((100, (nq + 2 * nkv) * hd)).astype(np.float32) * np.exp2(rng.integers(-3, 4, (100, 1))).astype(np.float32)
    old = [random_pages(rng, 8, nkv, block, hd) for _ in range(2)]
    table = gpu.rope_table(hd, 10000.0, 128)
    _, got = run_append(gpu, x, nq, (old[0][0], old[1][0]), (old[0][1], old[1][1]), slots, np.arange(100), table, 128, hd,
                        None, 0.0)
    _, k, v = ref.qk_norm_rope(x, nq, nkv, hd, None, None, 0.0, table.download(np.float32).reshape(128, hd // 2, 2), hd,
                               np.arange(100))
    for (c, s), y, at in ((old[0], k, 0), (old[1], v, 2)):
        codes, scale = ref.store_q8(c, s, y, slots)
        assert np.array_equal(got[at + 1], scale)
        live = np.repeat(scale != 255, 16, axis=2)
        assert np.array_equal(got[at][live], codes[live])


def test_append_extreme_values(gpu):
    """Zeros, the smallest and the largest magnitudes that a scale reaches, and what lies past them."""
    rng = np.random.default_rng(1)
    nq, nkv, hd, block = 1, 1, 64, 16
    sizes = [0.0, 1e-38, 2.0 ** -25, 2.0 ** -24, 3e-6, 127.0, 127.49999, 127.5, 32000.0, 65024.0, 65279.99, 65280.0, 1e6, 3e38]
    for size in sizes:
        x = (rng.uniform(-1, 1, (2, 3 * hd)) * size).astype(np.float32)
        x[0, hd + 3] = x[1, 2 * hd + 9] = size
        old = [random_pages(rng, 2, nkv, block, hd) for _ in range(2)]
        for c, s in old:
            s[:] = 112
        for slots in ([0, 20], [5, 6], [17, 16]):
            _, got = run_append(gpu, x, nq, (old[0][0], old[1][0]), (old[0][1], old[1][1]), slots, [0, 0],
                                gpu.rope_table(hd, 10000.0, 4), 4, hd, None, 0.0)
            for at, i in ((0, 1), (2, 2)):
                codes, scale = ref.store_q8(*old[at // 2], x[:, i * hd:(i + 1) * hd].astype(np.float64)[:, None], slots)
                assert np.array_equal(got[at + 1], scale), (size, slots)
                live = np.repeat(scale != 255, 16, axis=2)
                assert np.array_equal(got[at][live], codes[live]), (size, slots)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_non_finite_values_spoil_their_group_alone(gpu, bad):
    rng = np.random.default_rng(3)
    nq, nkv, hd, block, tokens = 2, 2, 128, 32, 40
    x = rng.standard_normal((tokens, (nq + 2 * nkv) * hd)).astype(np.float32)
    x[20, (nq + 1) * hd + 5] = bad           # key head 1
    x[3, (nq + nkv) * hd + 100] = bad        # value head 0
    old = [random_pages(rng, 3, nkv, block, hd) for _ in range(2)]
    for c, s in old:
        s[:] = 120
    slots = np.arange(tokens, dtype=np.int32)
    w = [np.ones(hd, np.float32)] * 2
    _, got = run_append(gpu, x, nq, (old[0][0], old[1][0]), (old[0][1], old[1][1]), slots, slots,
                        gpu.rope_table(hd, 10000.0, 64), 64, hd, w, 1e-6)
    spoilt = [np.argwhere(got[i] == 255).tolist() for i in (1, 3)]
    assert spoilt == [[[0, 1, 1]], [[0, 0, 0]]]
    # anew from its first row on
    x[:] = 1.0
    _, again = run_append(gpu, x, nq, (got[0], got[2]), (got[1], got[3]), slots, slots,
                          gpu.rope_table(hd, 10000.0, 64), 64, hd, w, 1e-6)
    assert not (again[1] == 255).any() and not (again[3] == 255).any()


def test_append_token_by_token(gpu):
    """Four sequences of growing keys, a token a call: the reference's codes after every step, and every row within a
    step of the last scale of what was stored."""
    rng = np.random.default_rng(8)
    nq, nkv, hd, block, seqs, steps = 2, 2, 64, 16, 4, 35
    blocks = seqs * 3
    pages = rng.permutation(blocks).reshape(seqs, 3)
    host = [random_pages(rng, blocks, nkv, block, hd) for _ in range(2)]
    cache = pages_of(gpu, host[0][0], host[1][0], host[0][1], host[1][1])
    table = gpu.rope_table(hd, 10000.0, 64)
    cs = table.download(np.float32).reshape(64, hd // 2, 2)
    SL, PO = i32(gpu, [0] * seqs), i32(gpu, [0] * seqs)
    batch = gpu.PagedBatch(seqs, seqs, 3, positions=PO, slots=SL)
    X, Q = gpu.DeviceBuffer(4 * seqs * 6 * hd), gpu.DeviceBuffer(4 * seqs * nq * hd)
    stored = [np.zeros((blocks * block, nkv, hd)) for _ in range(2)]
    for step in range(steps):
        x = (rng.standard_normal((seqs, 6 * hd)) * 1.13 ** step).astype(np.float32)
        slots = pages[:, step // block] * block + step % block
        X.upload(x)
        SL.upload(slots.astype(np.int32))
        PO.upload(np.full(seqs, step, np.int32))
        gpu.qk_norm_rope_q8(batch, cache, X, gpu.DTYPE_F32, 6 * hd, nq, table, 64, Q, gpu.DTYPE_F32, nq * hd)
        gpu.synchronize()
        _, k, v = ref.qk_norm_rope(x, nq, nkv, hd, None, None, 0.0, cs, hd, np.full(seqs, step))
        got = pages_back(cache, host[0][0].shape)
        for i, y in enumerate((k, v)):
            host[i] = ref.store_q8(*host[i], y, slots)
            stored[i][slots] = y
            assert np.array_equal(got[2 * i], host[i][0]) and np.array_equal(got[2 * i + 1], host[i][1])
    for i in range(2):
        values = ref.values_q8(*host[i]).transpose(0, 2, 1, 3)
        size = np.repeat(2.0 ** (host[i][1] - 127.0), 16, axis=2).transpose(0, 2, 1)
        for p in range(steps):
            at = pages[:, p // block], p % block
            off = np.abs(values[at] - stored[i].reshape(blocks, block, nkv, hd)[at])
            assert np.all(off <= size[at][..., None])


def test_append_in_place_and_from_a_graph(gpu):
    """q_out = qkv; a captured append replays with the slots and positions it then finds, as an eager one does."""
    rng = np.random.default_rng(4)
    nq, nkv, hd, tokens, block, blocks = 8, 2, 128, 19, 16, 12
    wide = (nq + 2 * nkv) * hd
    old = [random_pages(rng, blocks, nkv, block, hd) for _ in range(2)]
    eager, replayed = (pages_of(gpu, old[0][0], old[1][0], old[0][1], old[1][1]) for _ in range(2))
    X, Y = gpu.DeviceBuffer(4 * tokens * wide), gpu.DeviceBuffer(4 * tokens * wide)
    SL, PO = i32(gpu, [0] * tokens), i32(gpu, [0] * tokens)
    batch = gpu.PagedBatch(1, tokens, 1, positions=PO, slots=SL)
    table, stream = gpu.rope_table(hd, 10000.0, 64), gpu.Stream()
    gpu.synchronize()
    call = lambda x, c: gpu.qk_norm_rope_q8(batch, c, x, gpu.DTYPE_F32, wide, nq, table, 64, x, gpu.DTYPE_F32, wide,  # noqa: E731
                                            stream=stream)
    graph = gpu.Graph(stream, lambda: call(Y, replayed))
    for step in range(6):
        x = rng.standard_normal((tokens, wide)).astype(np.float32)
        X.upload(x)
        Y.upload(x)
        SL.upload(runs(rng, tokens, blocks, block, 16))
        PO.upload(rng.integers(0, 64, tokens).astype(np.int32))
        graph.launch(stream)
        stream.synchronize()
        call(X, eager)
        stream.synchronize()
        got = X.download(np.float32).reshape(tokens, wide)
        assert np.array_equal(got, Y.download(np.float32).reshape(tokens, wide))
        assert np.array_equal(got[:, nq * hd:], x[:, nq * hd:])
        for a, b in zip(pages_back(eager, old[0][0].shape), pages_back(replayed, old[0][0].shape)):
            assert np.array_equal(a, b)
    graph.close()


def test_append_past_4_gib(gpu):
    """A cache of more than 2^32 codes per tensor: the groups at its end are what those at its start are."""
    rng = np.random.default_rng(5)
    nq, nkv, hd, block, tokens = 2, 8, 256, 256, 40
    blocks = (1 << 32) // (nkv * hd * block) + 3
    cache = gpu.PagedCacheQ8.allocate(blocks, block, nkv, hd)
    assert cache.k.nbytes > 1 << 32
    x = rng.standard_normal((tokens, (nq + 2 * nkv) * hd)).astype(np.float32)
    X, Q = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer(4 * tokens * nq * hd)
    table = gpu.rope_table(hd, 10000.0, 64)
    got = []
    for b in (0, blocks - 1):
        slots = b * block + 32 + np.arange(tokens)
        batch = gpu.PagedBatch(1, tokens, 1, positions=i32(gpu, np.arange(tokens)), slots=i32(gpu, slots))
        gpu.qk_norm_rope_q8(batch, cache, X, gpu.DTYPE_F32, x.shape[1], nq, table, 64, Q, gpu.DTYPE_F32, nq * hd)
        gpu.synchronize()
        n, s = nkv * block * hd, nkv * block // 16
        part = [buf.view(b * w, w).download(np.uint8) for buf, w in ((cache.k, n), (cache.v, n), (cache.k_scale, s),
                                                                    (cache.v_scale, s))]
        part = [p.reshape(nkv, -1, w)[:, r] for p, w, r in zip(part, (hd, hd, 1, 1), [slice(32, 72)] * 2 + [slice(2, 5)] * 2)]
        got.append(part)
    assert all(np.array_equal(a, b) for a, b in zip(*got)) and got[0][0].any()


# --------------------------------------------------------------- attention ----

class Case8(Case):
    """A batch over 8-bit pages: k and v hold the values that codes and scales stand for."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.encode()

    def encode(self):
        """Codes and scales of what k and v hold now (a group with a NaN or an infinity is NaN), and k and v theirs."""
        self.codes = {}
        for name in ("k", "v"):
            x = getattr(self, name).astype(np.float64)
            blocks, nkv, block, hd = x.shape
            g = x.reshape(blocks, nkv, block // 16, 16 * hd)
            bad = ~np.isfinite(g).all(-1)
            g = np.where(bad[..., None], 0.0, g)
            top = np.abs(g).max(-1)
            e = np.clip(np.ceil(np.log2(np.maximum(top, 1e-30) / 127.0)).astype(int), -24, 9)
            codes = np.clip(np.rint(g * 2.0 ** -e[..., None]), -127, 127).astype(np.int8).reshape(x.shape)
            scale = np.where(bad, 255, e + 127).astype(np.uint8)
            self.codes[name], self.codes[name + "_scale"] = codes, scale
            setattr(self, name, ref.values_q8(codes, scale).astype(np.float16))

    def check(self, gpu, scale=None, window=0, adds=1, **kw):
        """`adds`: how often a value is added (the few-rows form adds those of scales above 2^5 up to 16 times)."""
        got = self.run(gpu, scale, window, **kw)
        out, size = self.want(scale, window)
        live = int(self.q_start[-1])
        assert np.all(got[live:] == 7)  # rows of no sequence
        got, out, size = got[:live].astype(np.float64), out[:live], size[:live]
        assert np.all(np.isfinite(got))
        sc = self.hd ** -0.5 if scale is None else scale
        q = np.abs(self.q[:live].astype(np.float64))
        kmax, vmax = float(np.abs(self.k).max()), float(np.abs(self.v).max())
        s = sc * q.sum(-1, keepdims=True) * kmax  # at least every |s| and every sum of magnitudes
        e = s * (self.hd / 8 + 8 + 4) * 2.0 ** -24 + 2.0 ** -22
        if not self.f16:
            e = e + sc * q.max(-1, keepdims=True) * 2.0 ** -21 * kmax * self.hd
        n = max(self.kv_len, default=0)
        sums = (n / 16 * adds + 40) * 2.0 ** -24
        bar = (np.expm1(2 * e) + (2.0 ** -11 if self.f16 else 2.0 ** -21) + sums) * size
        bar = bar + max(n, 0) * vmax * (2.0 ** -31 if self.f16 else 2.0 ** -40)
        if self.f16:
            bar = bar + 2.0 ** -11 * np.abs(out) * 1.01 + 2.0 ** -25
        off = np.abs(got - out)
        assert np.all(off <= bar), float(np.nanmax(off / np.maximum(bar, 1e-300)))

    def cache8(self, gpu):
        c = self.codes
        return pages_of(gpu, c["k"], c["v"], c["k_scale"], c["v_scale"])

    def run(self, gpu, scale=None, window=0, pad=0, stride=None, stream=None):
        dt = np.float16 if self.f16 else np.float32
        rows, row = max(self.rows, 1), self.nq * self.hd
        q = np.full((rows, row + pad), 3, dt)
        q[:, :row] = self.q.reshape(rows, row)
        bits = np.uint16 if self.f16 else np.uint32
        Q = gpu.DeviceBuffer.from_array(q.view(bits))
        O = gpu.DeviceBuffer.from_array(np.full((rows, row + pad), 7, dt).view(bits))
        stride = stride or self.width
        table = np.full((len(self.kv_len), stride), -1, np.int32)
        table[:, :self.width] = self.table
        batch = gpu.PagedBatch(len(self.kv_len), rows, self.width, i32(gpu, self.q_start), i32(gpu, self.kv_len),
                               i32(gpu, table), table_stride=stride)
        cache = self.cache8(gpu)
        ws = gpu.paged_attention_q8_workspace(batch, cache, self.nq)
        gpu.paged_attention_q8(batch, cache, Q, gpu.DTYPE_F16 if self.f16 else gpu.DTYPE_F32, row + pad, self.nq, O,
                               row + pad, ws, scale, window, stream)
        gpu.synchronize()
        out = O.download(bits).view(dt).reshape(rows, row + pad)
        assert np.all(out[:, row:] == 7)
        return out[:, :row].reshape(rows, self.nq, self.hd)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", HEADS)
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 63, 64, 127, 300])
def test_one_new_token(gpu, nq, nkv, hd, block, ctx, f16):
    Case8([(1, ctx)], nq, nkv, hd, block, f16, ctx).check(gpu)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", HEADS)
@pytest.mark.parametrize("seqs", [[(1, 70), (0, 50), (1, 0), (1, 513), (0, 0), (2, 33)], [(5, 95), (3, 200), (7, 0)],
                                  [(130, 0)], [(65, 3), (1, 80), (0, 9), (97, 131)]])
def test_batches(gpu, nq, nkv, hd, block, seqs, f16):
    Case8(seqs, nq, nkv, hd, block, f16, len(seqs), extra_rows=3).check(gpu, pad=8, stride=70)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 400), (3, 77), (2, 0)], [(90, 0), (70, 150)]])
@pytest.mark.parametrize("window", [1, 17, 64, 5000])
def test_windows(gpu, seqs, window, f16):
    Case8(seqs, 4, 2, 128, 16, f16, window).check(gpu, window=window)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 4999), (1, 30)], [(40, 2500)]])
def test_split_keys(gpu, seqs, f16):
    Case8(seqs, 8, 2, 128, 32, f16, 5).check(gpu)
    Case8(seqs, 8, 2, 64, 32, f16, 6, spread=4.0).check(gpu, scale=0.5)
    Case8(seqs, 2, 1, 256, 16, f16, 7).check(gpu, window=1500)


def test_many_sequences(gpu):
    """More sequences than a workgroup counts by itself."""
    Case8([(i % 3, (7 * i) % 40) for i in range(700)], 2, 1, 64, 16, True, 8).check(gpu)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", LARGE)
@pytest.mark.parametrize("seqs,window", [([(270, 0)], 0), ([(150, 3), (1, 80), (0, 9), (119, 331)], 0),
                                         ([(270, 200)], 33), ([(200, 1), (75, 500)], 128)])
def test_many_rows(gpu, nq, nkv, hd, block, seqs, window, f16):
    Case8(seqs, nq, nkv, hd, block, f16, 20 + len(seqs), extra_rows=2).check(gpu, window=window, pad=8)


@pytest.mark.parametrize("nq,nkv,hd,block,f16", SPLIT)
@pytest.mark.parametrize("seqs,window", [([(261, 700)], 0), ([(100, 900), (161, 30)], 0), ([(262, 800)], 333)])
def test_many_rows_split_keys(gpu, nq, nkv, hd, block, seqs, window, f16):
    Case8(seqs, nq, nkv, hd, block, f16, 25 + len(seqs), extra_rows=1).check(gpu, window=window)
    Case8(seqs, nq, nkv, hd, block, f16, 27, spread=3.0).check(gpu, window=window, scale=0.3)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,new,ctx", [(4, 2, 64, 1, 37), (4, 2, 64, 5, 219), (4, 2, 128, 100, 77),
                                               (4, 2, 256, 5, 90), (128, 2, 64, 270, 45), (128, 2, 128, 270, 45),
                                               (128, 2, 256, 270, 45), (64, 1, 128, 270, 45)])
def test_masked_places_never_touch_the_result(gpu, nq, nkv, hd, new, ctx, f16):
    """NaN in every group that no position uses; then in the last one, for the rows from its first position on."""
    c = Case8([(new, ctx)], nq, nkv, hd, 32, f16, 11)
    clean = c.run(gpu)
    used = np.zeros((c.blocks, c.block // 16), bool)
    p = np.arange(new + ctx)
    used[c.table[0, p // 32], p % 32 // 16] = True
    for cache in (c.k, c.v):
        parts = cache.reshape(c.blocks, nkv, c.block // 16, 16, hd)
        parts.transpose(0, 2, 1, 3, 4)[~used] = np.nan
    c.encode()
    assert np.array_equal(c.run(gpu), clean)
    last = new + ctx - 1
    hurt = np.zeros(clean.shape, bool)
    for name, head, rows in (("v", nkv - 1, slice(nq - nq // nkv, nq)), ("k", 0, slice(0, nq // nkv))):
        getattr(c, name)[c.table[0, last // 32], head, last % 32, 5] = np.nan
        c.encode()
        hurt[max(last // 16 * 16 - ctx, 0):new, rows] = True
        got = c.run(gpu)
        assert np.array_equal(got[~hurt], clean[~hurt]) and np.isnan(got[hurt]).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,new,ctx", [(4, 2, 64, 1, 200), (4, 2, 128, 5, 219), (4, 2, 256, 3, 90),
                                               (128, 2, 64, 270, 45), (128, 2, 128, 270, 45), (128, 2, 256, 270, 45)])
def test_scales_from_the_smallest_to_the_largest(gpu, nq, nkv, hd, new, ctx, f16):
    """Groups of keys and values of every size that a scale reaches, side by side."""
    c = Case8([(new, ctx)], nq, nkv, hd, 16, f16, 12)
    rng = np.random.default_rng(hd)
    for x, lo in ((c.k, 0), (c.v, -20)):
        size = np.exp2(rng.integers(lo, 14, (c.blocks, nkv, 1, 1)))
        x[:] = np.clip(x.astype(np.float64) * size, -65000, 65000).astype(np.float16)
    c.k[:, :, :, hd // 2:] = c.k[:, :, :, hd // 2:] * np.float16(0.25)
    c.encode()
    assert max(c.codes[n].max() for n in ("k_scale", "v_scale")) >= 134 and c.codes["v_scale"].min() < 110
    c.check(gpu, scale=1e-5, adds=16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", [(4, 2, 64, 16), (4, 2, 128, 64), (128, 2, 128, 16), (128, 2, 256, 16)])
def test_absent_pages_are_not_attended_to(gpu, nq, nkv, hd, block, f16):
    for new, ctx in ((1, 200), (90, 210)):
        c = Case8([(new, ctx), (new, ctx)], nq, nkv, hd, block, f16, 13)
        c.table[0, 0] = -1
        c.table[0, 2] = c.blocks
        c.table[1, :] = 2 ** 31 - 1  # nothing left: zeros
        c.check(gpu)
        assert not c.run(gpu)[new:2 * new].any()


@pytest.mark.parametrize("f16", [False, True])
def test_lengths_and_starts_out_of_range(gpu, f16):
    """Positions past the table, kv_len below the new tokens, starts that decrease or leave the rows."""
    Case8([(1, 100), (2, 90)], 2, 1, 64, 16, f16, 14, max_blocks=4).check(gpu)
    Case8([(270, 100)], 128, 2, 64, 16, f16, 34, max_blocks=9).check(gpu)
    c = Case8([(6, 0), (70, 10)], 2, 1, 64, 16, f16, 15)
    c.kv_len[:] = (3, 40)
    c.check(gpu)
    c.kv_len[:] = (0, -5)
    assert not c.run(gpu)[:76].any()
    c = Case8([(2, 20), (3, 20)], 2, 1, 64, 16, f16, 16)
    for start in ([0, 2, 400], [-9, 2, 5], [0, 5, 2], [7, 7, 7]):
        c.q_start = np.array(start, np.int32)
        c.run(gpu, pad=8)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs,nq,nkv,hd", [([(1, 300), (2, 5)], 4, 2, 128), ([(140, 33)], 4, 2, 64),
                                            ([(270, 30)], 128, 2, 128), ([(262, 800)], 64, 1, 128)])
def test_in_place_and_from_a_graph(gpu, seqs, nq, nkv, hd, f16):
    """out = q; each replay has the bits of an eager call."""
    c = Case8(seqs, nq, nkv, hd, 16, f16, 17)
    want = c.run(gpu)
    bits, row = (np.uint16 if f16 else np.uint32), nq * hd
    Q = gpu.DeviceBuffer.from_array(c.q.view(bits))
    batch = gpu.PagedBatch(len(seqs), c.rows, c.width, i32(gpu, c.q_start), i32(gpu, c.kv_len), i32(gpu, c.table))
    cache = c.cache8(gpu)
    ws, stream = gpu.paged_attention_q8_workspace(batch, cache, nq), gpu.Stream()
    gpu.synchronize()
    graph = gpu.Graph(stream, lambda: gpu.paged_attention_q8(batch, cache, Q, 1 if f16 else 0, row, nq, Q, row, ws,
                                                             stream=stream))
    for _ in range(3):
        Q.upload(c.q.view(bits))
        graph.launch(stream)
        stream.synchronize()
        assert np.array_equal(Q.download(bits).reshape(-1), want.view(bits).reshape(-1))
        ws.fill_zero()
        gpu.synchronize()
    graph.close()


def test_attention_past_4_gib(gpu):
    """Pages past 2^32 codes give what the same pages at the start give."""
    nkv, hd, block = 8, 128, 128
    blocks = (1 << 32) // (nkv * hd * block) + 100
    c = Case8([(2, 300), (70, 100)], 16, nkv, hd, block, True, 19)
    want = c.run(gpu)
    big = gpu.PagedCacheQ8.allocate(blocks, block, nkv, hd)
    small = c.cache8(gpu)
    assert big.k.nbytes > 1 << 32
    for name in ("k", "v", "k_scale", "v_scale"):
        src, dst = getattr(small, name), getattr(big, name)
        gpu._hip(gpu.lib().hip.hipMemcpy(dst.ptr + dst.nbytes - src.nbytes, src.ptr, src.nbytes, 3), "hipMemcpy")
    batch = gpu.PagedBatch(2, 72, c.width, i32(gpu, c.q_start), i32(gpu, c.kv_len),
                           i32(gpu, np.where(c.table < 0, -1, c.table + blocks - c.blocks)))
    Q, O = gpu.DeviceBuffer.from_array(c.q.view(np.uint16)), gpu.DeviceBuffer(c.q.nbytes)
    gpu.paged_attention_q8(batch, big, Q, 1, 16 * hd, 16, O, 16 * hd, gpu.paged_attention_q8_workspace(batch, big, 16))
    gpu.synchronize()
    assert np.array_equal(O.download(np.uint16).reshape(-1), want.view(np.uint16).reshape(-1))
