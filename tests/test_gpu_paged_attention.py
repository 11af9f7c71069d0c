"""GPU parity of rqmv_paged_attention against the f64 reference of
oracle/paged.py.

Bars. Per row, with w the reference's weights (sum 1) and A = sum w |v|:
 - a score s = scale q.k is off by at most E, counted here per element: fp32
   rows carry q to 2^-21 of the row's largest magnitude (two fp16 parts) and every
   product and sum of the dot rounds to 2^-24 of the magnitudes' sum (head_dim / 8 + 8
   roundings in a row), fp16 rows only the latter; then the product with the scale
   and the reference, 4 * 2^-24 |s|, and 2^-22 for the exponential. Weights
   are then off by a factor e^(+-E), their quotient by e^(2 E).
 - fp16 rows: each weight is rounded to fp16 (2^-11 relative, or 2^-25 of the
   scale where the largest is 2^6 or more: 2^-31), and so is the output (2^-11).
   fp32 rows: weights in two parts, 2^-21.
 - sums of n products: (n / 16 + 40) * 2^-24 of A, and the joins of waves and splits
   lie within the 40.
So |out - ref| <= (e^(2 E) - 1 + weights + sums) A + output rounding.
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu


def i32(gpu, a):
    return gpu.DeviceBuffer.from_array(np.asarray(a, np.int32))


class Case:
    """A batch of sequences (new, cached) over a shuffled pool, on the host."""

    def __init__(self, seqs, nq, nkv, hd, block, f16, seed, spread=1.0, extra_rows=0, max_blocks=None):
        rng = np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.block, self.f16 = nq, nkv, hd, block, f16
        need = [ref.pages(c + n, block) for n, c in seqs]
        self.width = max_blocks or max(max(need), 1)
        self.blocks = sum(need) + 2
        ids = rng.permutation(self.blocks)
        self.table = np.full((len(seqs), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            n = min(n, self.width)
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.q_start = np.concatenate(([0], np.cumsum([n for n, _ in seqs]))).astype(np.int32)
        self.kv_len = np.array([n + c for n, c in seqs], np.int32)
        self.rows = int(self.q_start[-1]) + extra_rows
        dt = np.float16 if f16 else np.float32
        self.q = (rng.standard_normal((max(self.rows, 1), nq, hd)) * spread).astype(dt)
        self.k = rng.standard_normal((self.blocks, nkv, block, hd)).astype(np.float16)
        self.v = rng.standard_normal((self.blocks, nkv, block, hd)).astype(np.float16)

    def run(self, gpu, scale=None, window=0, pad=0, stride=None, stream=None):
        dt = np.float16 if self.f16 else np.float32
        rows, row = max(self.rows, 1), self.nq * self.hd
        q = np.full((rows, row + pad), 3, dt)
        q[:, :row] = self.q.reshape(rows, row)
        bits = np.uint16 if self.f16 else np.uint32
        Q = gpu.DeviceBuffer.from_array(q.view(bits))
        self.sentinel = np.full((rows, row + pad), 7, dt)
        O = gpu.DeviceBuffer.from_array(self.sentinel.view(bits))
        stride = stride or self.width
        table = np.full((len(self.kv_len), stride), -1, np.int32)
        table[:, :self.width] = self.table
        batch = gpu.PagedBatch(len(self.kv_len), rows, self.width, i32(gpu, self.q_start), i32(gpu, self.kv_len),
                               i32(gpu, table), table_stride=stride)
        cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(self.k.view(np.uint16)),
                               gpu.DeviceBuffer.from_array(self.v.view(np.uint16)), self.blocks, self.block, self.nkv,
                               self.hd)
        ws = gpu.paged_attention_workspace(batch, cache, self.nq)
        gpu.paged_attention(batch, cache, Q, gpu.DTYPE_F16 if self.f16 else gpu.DTYPE_F32, row + pad, self.nq, O,
                            row + pad, ws, scale, window, stream)
        gpu.synchronize()
        out = O.download(bits).view(dt).reshape(rows, row + pad)
        assert np.all(out[:, row:] == 7)
        return out[:, :row].reshape(rows, self.nq, self.hd)

    def want(self, scale=None, window=0):
        scale = self.hd ** -0.5 if scale is None else scale
        out = ref.attention(self.q, self.k, self.v, self.q_start, self.kv_len, self.table, self.width, scale, window)
        size = ref.attention(self.q, self.k, np.abs(self.v), self.q_start, self.kv_len, self.table, self.width, scale,
                             window)
        return out, size

    def check(self, gpu, scale=None, window=0, **kw):
        got = self.run(gpu, scale, window, **kw)
        out, size = self.want(scale, window)
        live = int(self.q_start[-1])
        assert np.all(got[live:] == 7)  # rows of no sequence
        got, out, size = got[:live].astype(np.float64), out[:live], size[:live]
        assert np.all(np.isfinite(got))
        sc = self.hd ** -0.5 if scale is None else scale
        q = np.abs(self.q[:live].astype(np.float64))
        kmax = float(np.abs(self.k).max())
        s = sc * q.sum(-1, keepdims=True) * kmax  # at least every |s| and every sum of magnitudes
        e = s * (self.hd / 8 + 8 + 4) * 2.0 ** -24 + 2.0 ** -22
        if not self.f16:
            e = e + sc * q.max(-1, keepdims=True) * 2.0 ** -21 * kmax * self.hd
        sums = (max(self.kv_len, default=0) / 16 + 40) * 2.0 ** -24
        w = 2.0 ** -11 + 2.0 ** -31 * max(self.kv_len, default=0) if self.f16 else 2.0 ** -21
        bar = (np.expm1(2 * e) + w + sums) * size + (2.0 ** -11 * np.abs(out) * 1.01 + 2.0 ** -25 if self.f16 else 0)
        off = np.abs(got - out)
        assert np.all(off <= bar), float(np.nanmax(off / np.maximum(bar, 1e-300)))


HEADS = [(4, 2, 64, 16), (32, 8, 128, 64), (6, 6, 128, 16), (14, 2, 64, 32), (4, 1, 256, 128), (10, 2, 256, 16),
         (40, 1, 64, 256)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", HEADS)
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 31, 63, 64, 127, 128, 300])
def test_one_new_token(gpu, nq, nkv, hd, block, ctx, f16):
    Case([(1, ctx)], nq, nkv, hd, block, f16, ctx).check(gpu)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", HEADS)
@pytest.mark.parametrize("seqs", [[(1, 70), (0, 50), (1, 0), (1, 513), (0, 0), (2, 33)], [(5, 95), (3, 200), (7, 0)],
                                  [(1, 5)] * 9 + [(1, 900)]])
def test_decode_batches(gpu, nq, nkv, hd, block, seqs, f16):
    Case(seqs, nq, nkv, hd, block, f16, len(seqs), extra_rows=3).check(gpu, pad=8, stride=70)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", HEADS)
@pytest.mark.parametrize("seqs", [[(130, 0)], [(65, 3), (1, 80), (0, 9), (97, 131)], [(64, 64), (200, 100)]])
def test_prompts(gpu, nq, nkv, hd, block, seqs, f16):
    Case(seqs, nq, nkv, hd, block, f16, 1 + len(seqs), extra_rows=2).check(gpu, pad=16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 400), (3, 77), (2, 0)], [(90, 0), (70, 150)]])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 5000])
def test_windows(gpu, seqs, window, f16):
    Case(seqs, 4, 2, 128, 16, f16, window).check(gpu, window=window)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 4999), (1, 30)], [(40, 2500)]])
def test_split_keys(gpu, seqs, f16):
    """Keys over many workgroups and their join, peaked scores among them."""
    Case(seqs, 8, 2, 128, 32, f16, 5).check(gpu)
    Case(seqs, 8, 2, 64, 32, f16, 6, spread=4.0).check(gpu, scale=0.5)
    Case(seqs, 2, 1, 256, 16, f16, 7).check(gpu, window=1500)


def test_many_sequences(gpu):
    """More sequences than one search step tells apart."""
    seqs = [(i % 3, (7 * i) % 40) for i in range(700)]
    Case(seqs, 2, 1, 64, 16, True, 8).check(gpu)


@pytest.mark.parametrize("f16", [False, True])
def test_scores_that_grow_along_the_keys(gpu, f16):
    """The reference moves at every step: key i has i times the same direction."""
    for new in (1, 150):
        c = Case([(new, 700)], 4, 1, 64, 16, f16, 9)
        order = c.table[0, np.arange(700 + new) // 16], np.arange(700 + new) % 16
        c.k[order[0], 0, order[1]] = (np.arange(700 + new)[:, None] / 256.0 * np.ones(64)).astype(np.float16)
        c.q[:] = 1.0
        c.check(gpu, scale=1.0)
        c.q[:] = -1.0
        c.check(gpu, scale=1.0)


@pytest.mark.parametrize("new,ctx", [(1, 37), (3, 200), (100, 50)])
def test_extreme_rows_fp32(gpu, new, ctx):
    """fp32 queries past fp16's range and far below it."""
    c = Case([(new, ctx)], 4, 2, 128, 16, False, 10)
    c.q[:, 0] *= 1e6
    c.q[:, 1] *= 1e-6
    c.q[:, 2] *= 1e-30
    c.q[0, 3, 0] = 1e5
    c.check(gpu, scale=1e-6)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,ctx", [(1, 37), (5, 219), (100, 77), (300, 0)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_masked_places_never_touch_the_result(gpu, new, ctx, bad, f16):
    """NaN and infinities in every row of the cache that no position uses, and in the last token's key and value,
    which only that token's rows may see."""
    c = Case([(new, ctx), (new, ctx)], 4, 2, 64, 16, f16, 11)
    clean = c.run(gpu)
    used = np.zeros((c.blocks, c.block), bool)
    for s in range(2):
        p = np.arange(new + ctx)
        used[c.table[s, p // 16], p % 16] = True
    for cache in (c.k, c.v):
        cache.transpose(0, 2, 1, 3)[~used] = bad
    got = c.run(gpu)
    assert np.array_equal(got, clean)
    if new > 1:
        last = new + ctx - 1
        c.v[c.table[0, last // 16], 1, last % 16, 5] = bad
        got = c.run(gpu)
        hurt = np.zeros(got.shape, bool)
        hurt[new - 1, 2:, 5] = True  # kv head 1's query heads of sequence 0's last row
        assert np.array_equal(got[~hurt], clean[~hurt]) and not np.isfinite(got[hurt]).any()
        c.k[c.table[0, last // 16], 0, last % 16, 3] = np.nan
        got = c.run(gpu)
        hurt[new - 1, :2] = True
        assert np.array_equal(got[~hurt], clean[~hurt]) and not np.isfinite(got[hurt]).any()


@pytest.mark.parametrize("f16", [False, True])
def test_non_finite_values_that_all_rows_see(gpu, f16):
    for new in (1, 80):
        c = Case([(new, 300)], 2, 1, 64, 16, f16, 12)
        c.v[c.table[0, 3], 0, 5, 9] = np.inf
        got = c.run(gpu)
        assert not np.isfinite(got[:, :, 9]).any()
        got[:, :, 9] = 0
        assert np.isfinite(got).all()
        c = Case([(new, 300)], 2, 1, 64, 16, f16, 12)
        c.q[new - 1, 1, 0] = np.nan
        got = c.run(gpu)
        assert np.isnan(got[new - 1, 1]).all()
        got[new - 1, 1] = 0
        assert np.isfinite(got).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("block", [16, 64])
def test_absent_pages_are_not_attended_to(gpu, block, f16):
    for new, ctx in ((1, 200), (3, 150), (90, 210)):
        c = Case([(new, ctx), (new, ctx)], 4, 2, 64, block, f16, 13)
        c.table[0, 0] = -1
        c.table[0, 2] = c.blocks
        c.table[1, :] = 2 ** 31 - 1  # nothing left: zeros
        c.check(gpu)
        assert not c.run(gpu)[new:2 * new].any()


@pytest.mark.parametrize("f16", [False, True])
def test_lengths_the_table_does_not_reach(gpu, f16):
    """Positions past max_blocks pages are not attended to; kv_len below the new tokens leaves rows without keys."""
    c = Case([(1, 100), (2, 90)], 2, 1, 64, 16, f16, 14, max_blocks=4)
    c.check(gpu)
    c = Case([(6, 0), (70, 10)], 2, 1, 64, 16, f16, 15)
    c.kv_len[:] = (3, 40)
    c.check(gpu)
    c.kv_len[:] = (0, -5)
    assert not c.run(gpu)[:76].any()


def test_starts_out_of_range_stay_inside_the_rows(gpu):
    """q_start past the batch's rows or decreasing: whatever the rows hold, nothing outside them is written."""
    c = Case([(2, 20), (3, 20)], 2, 1, 64, 16, True, 16)
    for start in ([0, 2, 400], [-9, 2, 5], [0, 5, 2], [7, 7, 7]):
        c.q_start = np.array(start, np.int32)
        c.run(gpu, pad=8)


@pytest.mark.parametrize("f16", [False, True])
def test_in_place(gpu, f16):
    """out = q."""
    for seqs in ([(1, 300), (2, 5)], [(140, 33)]):
        c = Case(seqs, 4, 2, 128, 16, f16, 17)
        want = c.run(gpu)
        bits = np.uint16 if f16 else np.uint32
        Q = gpu.DeviceBuffer.from_array(c.q.view(bits))
        batch = gpu.PagedBatch(len(seqs), c.rows, c.width, i32(gpu, c.q_start), i32(gpu, c.kv_len), i32(gpu, c.table))
        cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                               gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, 16, 2, 128)
        gpu.paged_attention(batch, cache, Q, 1 if f16 else 0, 512, 4, Q, 512,
                            gpu.paged_attention_workspace(batch, cache, 4))
        gpu.synchronize()
        assert np.array_equal(Q.download(bits).reshape(-1), want.view(bits).reshape(-1))


@pytest.mark.parametrize("f16", [False, True])
def test_same_result_every_time_and_from_a_graph(gpu, f16):
    """Captured once, replayed as the lengths grow; each replay has the bits of an eager call."""
    c = Case([(1, 40), (1, 700)], 8, 2, 128, 16, f16, 18, max_blocks=60)
    free = [b for b in range(c.blocks) if b not in c.table]
    c.table[0, 3], c.table[1, 44] = free[0], free[1]  # pages for the positions to come
    bits, size = (np.uint16, 2) if f16 else (np.uint32, 4)
    KV = i32(gpu, c.kv_len)
    batch = gpu.PagedBatch(2, 2, c.width, i32(gpu, c.q_start), KV, i32(gpu, c.table))
    cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                           gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, 16, 2, 128)
    Q = gpu.DeviceBuffer.from_array(c.q.view(bits))
    O, E = gpu.DeviceBuffer(2 * 1024 * size), gpu.DeviceBuffer(2 * 1024 * size)
    ws = gpu.paged_attention_workspace(batch, cache, 8)
    stream = gpu.Stream()
    call = lambda out, s: gpu.paged_attention(batch, cache, Q, 1 if f16 else 0, 1024, 8, out, 1024, ws, stream=s)  # noqa: E731
    graph = gpu.Graph(stream, lambda: call(O, stream))
    for step in range(12):
        KV.upload(c.kv_len + step)
        graph.launch(stream)
        stream.synchronize()
        call(E, stream)
        stream.synchronize()
        assert np.array_equal(O.download(bits), E.download(bits))
    graph.close()


def test_offsets_past_4_gib(gpu):
    """A cache of more than 2^32 bytes per tensor: pages at its end give what the same pages at its start give."""
    nkv, hd, block, blocks = 8, 128, 128, 17000
    c = Case([(2, 300), (70, 100)], 16, nkv, hd, block, True, 19)
    want = c.run(gpu)
    K, V = gpu.DeviceBuffer(2 * blocks * nkv * block * hd), gpu.DeviceBuffer(2 * blocks * nkv * block * hd)
    assert K.nbytes > 1 << 32
    page = 2 * nkv * block * hd
    for buf, src in ((K, c.k), (V, c.v)):
        small = gpu.DeviceBuffer.from_array(src.view(np.uint16))
        at = (blocks - c.blocks) * page
        gpu._hip(gpu.lib().hip.hipMemcpy(buf.ptr + at, small.ptr, small.nbytes, 3), "hipMemcpy")
    batch = gpu.PagedBatch(2, 72, c.width, i32(gpu, c.q_start), i32(gpu, c.kv_len),
                           i32(gpu, np.where(c.table < 0, -1, c.table + blocks - c.blocks)))
    cache = gpu.PagedCache(K, V, blocks, block, nkv, hd)
    Q, O = gpu.DeviceBuffer.from_array(c.q.view(np.uint16)), gpu.DeviceBuffer(c.q.nbytes)
    gpu.paged_attention(batch, cache, Q, 1, 16 * hd, 16, O, 16 * hd, gpu.paged_attention_workspace(batch, cache, 16))
    gpu.synchronize()
    assert np.array_equal(O.download(np.uint16).reshape(-1), want.view(np.uint16).reshape(-1))


# Batches of so many rows that the large tiles take them (more than 1024 tiles of 32 rows over all heads), and
# of heads over one kv head, where those tiles' keys are split as well.
LARGE = [(128, 2, 64, 16), (126, 18, 64, 64), (128, 1, 128, 16), (132, 44, 128, 32), (128, 2, 256, 16),
         (130, 26, 256, 128)]
SPLIT = [(64, 1, 64, 16, False), (64, 1, 128, 16, False), (64, 1, 128, 32, True), (32, 1, 256, 16, False)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,block", LARGE)
@pytest.mark.parametrize("seqs,window", [([(270, 0)], 0), ([(150, 3), (1, 80), (0, 9), (119, 331)], 0),
                                         ([(270, 200)], 33), ([(200, 1), (75, 500)], 128)])
def test_many_rows(gpu, nq, nkv, hd, block, seqs, window, f16):
    Case(seqs, nq, nkv, hd, block, f16, 20 + len(seqs), extra_rows=2).check(gpu, window=window, pad=8)


@pytest.mark.parametrize("nq,nkv,hd,block,f16", SPLIT)
@pytest.mark.parametrize("seqs,window", [([(261, 700)], 0), ([(100, 900), (161, 30)], 0), ([(262, 800)], 333),
                                         ([(270, 3)], 0)])
def test_many_rows_split_keys(gpu, nq, nkv, hd, block, seqs, window, f16):
    Case(seqs, nq, nkv, hd, block, f16, 25 + len(seqs), extra_rows=1).check(gpu, window=window)
    Case(seqs, nq, nkv, hd, block, f16, 27, spread=3.0).check(gpu, window=window, scale=0.3)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd", [(128, 2, 64), (128, 2, 128), (128, 2, 256), (64, 1, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_many_rows_masked_places(gpu, nq, nkv, hd, bad, f16):
    """As test_masked_places_never_touch_the_result, at many rows."""
    new, ctx = 270, 45
    c = Case([(new, ctx)], nq, nkv, hd, 16, f16, 30)
    clean = c.run(gpu)
    used = np.zeros((c.blocks, c.block), bool)
    p = np.arange(new + ctx)
    used[c.table[0, p // 16], p % 16] = True
    for cache in (c.k, c.v):
        cache.transpose(0, 2, 1, 3)[~used] = bad
    assert np.array_equal(c.run(gpu), clean)
    hurt = np.zeros(clean.shape, bool)
    for at, dim in ((new + ctx - 1, 5), (200, 40)):  # a value is for the rows from its position on
        c.v[c.table[0, at // 16], nkv - 1, at % 16, dim] = bad
        hurt[at - ctx:, nq - nq // nkv:, dim] = True
        got = c.run(gpu)
        assert np.array_equal(got[~hurt], clean[~hurt]) and not np.isfinite(got[hurt]).any()
    c.k[c.table[0, 250 // 16], 0, 250 % 16, 3] = np.nan
    hurt[250 - ctx:, :nq // nkv] = True
    got = c.run(gpu)
    assert np.array_equal(got[~hurt], clean[~hurt]) and not np.isfinite(got[hurt]).any()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd", [(128, 2, 64), (128, 2, 128), (128, 2, 256), (64, 1, 128)])
def test_many_rows_absent_pages(gpu, nq, nkv, hd, f16):
    c = Case([(200, 100), (75, 10)], nq, nkv, hd, 16, f16, 31)
    c.table[0, 0] = -1
    c.table[0, 2] = c.blocks
    c.table[1, :] = -2 ** 31  # nothing left: zeros
    c.check(gpu)
    assert not c.run(gpu)[200:275].any()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,new", [(4, 2, 1), (4, 2, 60), (128, 2, 270)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_non_finite_values_beside_an_absent_page(gpu, nq, nkv, new, bad, f16):
    """Every row sees key 35; the pages around its own are absent."""
    c = Case([(new, 200)], nq, nkv, 128, 16, f16, 32)
    c.table[0, [1, 3]] = -1
    clean = c.run(gpu)
    c.v[c.table[0, 2], 1, 3, 7] = bad
    got = c.run(gpu)
    hurt = np.zeros(got.shape, bool)
    hurt[:, nq // 2:, 7] = True
    assert np.array_equal(got[~hurt], clean[~hurt]) and not np.isfinite(got[hurt]).any()


def test_many_extreme_rows_fp32(gpu):
    for hd in (64, 128, 256):
        c = Case([(270, 30)], 128, 2, hd, 16, False, 33)
        c.q[:, 0] *= 1e6
        c.q[:, 1] *= 1e-6
        c.q[:, 2] *= 1e-30
        c.q[0, 3, 0] = 1e5
        c.check(gpu, scale=1e-6)


@pytest.mark.parametrize("f16", [False, True])
def test_many_rows_lengths(gpu, f16):
    """Positions past the table, and kv_len below the new tokens."""
    Case([(270, 100)], 128, 2, 64, 16, f16, 34, max_blocks=9).check(gpu)
    c = Case([(200, 0), (75, 10)], 128, 1, 128, 16, f16, 35)
    c.kv_len[:] = (3, 40)
    c.check(gpu)
    c.kv_len[:] = (0, -5)
    assert not c.run(gpu)[:275].any()


@pytest.mark.parametrize("nq,nkv,hd,block,f16", SPLIT + [(128, 2, 64, 16, True), (128, 2, 256, 16, True)])
def test_many_rows_in_place_from_a_graph(gpu, nq, nkv, hd, block, f16):
    """out = q; each replay has the bits of an eager call on the same rows."""
    c = Case([(200, 0), (62, 400)], nq, nkv, hd, block, f16, 36)
    bits, row = (np.uint16 if f16 else np.uint32), nq * hd
    KV = i32(gpu, c.kv_len)
    batch = gpu.PagedBatch(2, c.rows, c.width, i32(gpu, c.q_start), KV, i32(gpu, c.table))
    cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                           gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, block, nkv, hd)
    Q = gpu.DeviceBuffer.from_array(c.q.view(bits))
    O = gpu.DeviceBuffer(c.q.nbytes)
    ws = gpu.paged_attention_workspace(batch, cache, nq)
    stream = gpu.Stream()
    call = lambda q, out: gpu.paged_attention(batch, cache, q, 1 if f16 else 0, row, nq, out, row, ws,  # noqa: E731
                                              stream=stream)
    graph = gpu.Graph(stream, lambda: call(Q, Q))
    for step in range(4):
        KV.upload(c.kv_len - 9 * step)
        Q.upload(c.q.view(bits))
        call(Q, O)
        stream.synchronize()
        graph.launch(stream)
        stream.synchronize()
        assert np.array_equal(Q.download(bits), O.download(bits))
    graph.close()


def test_two_streams_with_a_workspace_each(gpu):
    """Two batches at once on two streams, again and again, give what each gives alone."""
    cases = [Case([(1, 3000), (3, 50)], 32, 8, 128, 16, True, 37), Case([(261, 700)], 64, 1, 128, 16, True, 38)]
    want = [c.run(gpu) for c in cases]
    runs = []
    for c in cases:
        batch = gpu.PagedBatch(len(c.kv_len), c.rows, c.width, i32(gpu, c.q_start), i32(gpu, c.kv_len), i32(gpu, c.table))
        cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                               gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, 16, c.nkv, 128)
        runs.append((batch, cache, gpu.DeviceBuffer.from_array(c.q.view(np.uint16)), gpu.DeviceBuffer(c.q.nbytes),
                     gpu.paged_attention_workspace(batch, cache, c.nq), gpu.Stream()))
    for _ in range(8):
        for c, (batch, cache, q, out, ws, stream) in zip(cases, runs):
            gpu.paged_attention(batch, cache, q, 1, c.nq * 128, c.nq, out, c.nq * 128, ws, stream=stream)
    for c, run, w in zip(cases, runs, want):
        run[5].synchronize()
        assert np.array_equal(run[3].download(np.uint16).reshape(-1), w.view(np.uint16).reshape(-1))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("seqs,window", [([(i % 3, (7 * i) % 40) for i in range(257)] + [(2, 5000), (40, 900)], 0),
                                         ([(1, 2300)] + [(1, 3)] * 511 + [(1, 700)], 0),
                                         ([(0, 9)] * 300 + [(1, 1500), (0, 0), (3, 2000)] + [(0, 4)] * 1000, 1100)])
def test_more_sequences_than_threads(gpu, seqs, window, f16):
    """Items found by the launch before, long sequences among short ones and empty ones."""
    Case(seqs, 4, 2, 64, 16, f16, 40, extra_rows=2).check(gpu, window=window)
    c = Case(seqs, 2, 1, 128, 32, f16, 41)
    c.table[5, :] = -1
    c.check(gpu, window=window)


def test_many_starts_out_of_order_stay_inside_the_rows(gpu):
    c = Case([(2, 600)] * 300, 2, 1, 64, 16, True, 42)
    for start in (np.arange(301)[::-1] * 2, np.where(np.arange(301) % 2, 600, 0), np.full(301, -3), np.arange(301) * 9):
        c.q_start = start.astype(np.int32)
        c.run(gpu, pad=8)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,new,ctx", [(4, 2, 128, 1, 700), (4, 1, 64, 3, 40), (8, 4, 256, 2, 300),
                                               (128, 2, 64, 270, 30), (128, 2, 128, 270, 30), (128, 2, 256, 270, 30)])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e20])
def test_scores_whose_last_bit_passes_one(gpu, nq, nkv, hd, new, ctx, scale, f16):
    """Scores of 10^5 and more: where the largest leads by 10^-4 of itself (a dot's rounding takes up to
    (hd / 8 + 8) 2^-24 < 3e-6 of the magnitudes' sum, here up to ten times the score) its value is the row's."""
    c = Case([(new, ctx)], nq, nkv, hd, 16, f16, 43)
    c.q *= 100 if f16 else 1e5
    got = c.run(gpu, scale=scale).astype(np.float64)
    assert np.isfinite(got).all()
    at = np.arange(new + ctx)
    k, v = (x[c.table[0, at // 16], :, at % 16].astype(np.float64) for x in (c.k, c.v))
    some = 0
    for h in range(nq):
        g = h // (nq // nkv)
        s = c.q[:, h].astype(np.float64) @ k[:, g].T
        s[at[None, :] > ctx + np.arange(new)[:, None]] = -np.inf
        first = s.argmax(1)
        best = np.take_along_axis(s, first[:, None], 1)[:, 0]
        np.put_along_axis(s, first[:, None], -np.inf, 1)
        size = np.abs(c.q[:, h].astype(np.float64)) @ np.abs(k[:, g]).T
        sure = best - s.max(1) > 1e-4 * size.max(1) if s.shape[1] > 1 else np.ones(new, bool)
        some += sure.sum()
        assert np.all(np.abs(got[sure, h] - v[first[sure], g]) <= 2.0 ** -10 * np.abs(v[first[sure], g]))
    assert some > new * nq // 2


ROWS_FORMS = [(4, 2, 64, 1), (4, 1, 256, 3), (8, 2, 128, 40), (128, 2, 64, 270), (128, 2, 128, 270), (128, 2, 256, 270),
              (64, 1, 128, 262)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,new", ROWS_FORMS)
@pytest.mark.parametrize("ctx", [0, 5, 900])
def test_rows_whose_scores_are_all_minus_infinity(gpu, nq, nkv, hd, new, ctx, f16):
    """An infinite query opposite to every key that it sees: e^(-inf - -inf) is undefined, and the row is NaN, not the zeros
    of a row without keys."""
    c = Case([(new, ctx)], nq, nkv, hd, 16, f16, 50)
    c.k[..., 0] = -np.abs(c.k[..., 0]) - np.float16(0.25)
    if ctx + new >= 32:
        c.table[0, (ctx + new) // 32] = -1  # (an absent page among them, not the first)
    clean = c.run(gpu)
    assert np.isfinite(clean).all()
    hurt = np.zeros(clean.shape, bool)
    for row, head in ((0, 0), (new - 1, nq - 1), (new // 2, nq // 2)):
        c.q[row, head, 0] = np.inf
        hurt[row, head] = True
    got = c.run(gpu)
    assert np.isnan(got[hurt]).all() and np.array_equal(got[~hurt], clean[~hurt])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,new", ROWS_FORMS)
def test_infinite_keys(gpu, nq, nkv, hd, new, f16):
    """A key whose score is -infinity weighs nothing beside finite ones (fp32 rows, whose queries are two parts, may
    be NaN instead), and a row that sees only such keys is NaN; a score of +infinity makes the row NaN."""
    ctx = 1500
    c = Case([(new, ctx)], nq, nkv, hd, 16, f16, 51)
    c.q[..., 0] = 8.0
    at = lambda p: (c.table[0, p // 16], slice(None), p % 16, 0)  # noqa: E731
    far = np.r_[0:1100, 1300, ctx - 1]  # (whole parts of split keys among them)
    for p in far:
        c.k[at(p)] = -60000.0  # a score of -480000 / sqrt(head_dim): a weight of zero
    clean = c.run(gpu)
    assert np.isfinite(clean).all()
    for p in far:
        c.k[at(p)] = -np.inf
    got = c.run(gpu)
    if f16:
        assert np.array_equal(got, clean)
    else:
        whole = np.isfinite(got).all(-1)
        assert np.array_equal(got[whole], clean[whole])
    c.k[at(1200)] = np.inf
    assert not np.isfinite(c.run(gpu)).any()
    c.k[..., 0] = -np.inf
    assert not np.isfinite(c.run(gpu)).any()
    c.table[:] = -1  # no key at all
    assert not c.run(gpu).any()


@pytest.mark.parametrize("hd,nq,nkv,new", [(64, 4, 2, 3), (128, 4, 2, 40), (256, 4, 1, 2), (64, 128, 2, 270),
                                           (128, 128, 2, 270), (256, 128, 2, 270)])
def test_factors_of_scores_at_the_ends_of_fp32(gpu, hd, nq, nkv, new):
    """fp32 rows: tiny queries at a small scale, and queries near the type's end at a large one whose keys are zero there:
    all scores are 0 or within 2^-60 of it, so each row is the mean of the values that it sees."""
    ctx = 37
    c = Case([(new, ctx)], nq, nkv, hd, 16, False, 52)
    at = np.arange(new + ctx)
    values = c.v[c.table[0, at // 16], :, at % 16].astype(np.float64)  # [keys, nkv, hd]

    def check(scale):
        got = c.run(gpu, scale=scale).astype(np.float64)
        for i in range(new):
            seen = values[:ctx + i + 1]
            want = np.repeat(seen.mean(0), nq // nkv, 0)
            size = np.repeat(np.abs(seen).mean(0), nq // nkv, 0)
            # weights of 1 are exact; sums of up to 307 values, the division
            assert np.all(np.abs(got[i] - want) <= (307 / 16 + 40) * 2.0 ** -24 * size), scale

    c.q[:] *= np.float32(1e-30)
    for scale in (1e-20, 1e-30, 1e-38, 1e-42):
        check(scale)
    c.q[:] = 0
    c.q[..., 1] = 3e38
    c.k[..., 1] = 0
    for scale in (1e4, 1e10, 1e30):
        check(scale)


STARTS = [(128, 2, 64, True), (128, 2, 128, False), (128, 2, 256, True), (128, 2, 256, False), (64, 1, 128, True),
          (64, 1, 64, False), (4, 2, 64, True), (2, 1, 128, False)]


@pytest.mark.parametrize("nq,nkv,hd,f16", STARTS)
@pytest.mark.parametrize("starts", [
    [0, 270, 3, 4, 5, 270], [270, 200, 100, 50, 20, 0], [0, 260, 0, 260, 0, 270], [-9, 400, -9, 400, -9, 400],
    [200, 210, 220, 230, 240, 270], [270] * 6, [-7] * 6, [2 ** 31 - 1] * 6, [0, -2 ** 31, 2 ** 31 - 1, 5, -1, 9],
    [0, 0, 60, 60, 270, 270]])
def test_starts_of_any_values_stay_inside_the_rows(gpu, nq, nkv, hd, f16, starts):
    """Nothing before or behind the batch's rows is written, nor a row that no sequence could have."""
    c = Case([(54, 100), (54, 0), (54, 300), (54, 7), (54, 64)], nq, nkv, hd, 16, f16, 54)
    dt, bits = (np.float16, np.uint16) if f16 else (np.float32, np.uint32)
    row, guard, size = nq * hd, 300, np.dtype(dt).itemsize
    Q = gpu.DeviceBuffer.from_array(c.q.view(bits))
    O = gpu.DeviceBuffer.from_array(np.full((c.rows + 2 * guard, row), 7, dt).view(bits))
    batch = gpu.PagedBatch(5, c.rows, c.width, i32(gpu, starts), i32(gpu, c.kv_len), i32(gpu, c.table))
    cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                           gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, 16, nkv, hd)
    gpu.paged_attention(batch, cache, Q, 1 if f16 else 0, row, nq, O.view(guard * row * size, c.rows * row * size), row,
                        gpu.paged_attention_workspace(batch, cache, nq))
    gpu.synchronize()
    out = O.download(bits).view(dt).reshape(c.rows + 2 * guard, row)
    may = np.zeros(len(out), bool)  # rows between a start and the next one
    for a, b in zip(starts, starts[1:]):
        may[guard + min(max(a, 0), c.rows):guard + min(max(b, 0), c.rows)] = True
    assert np.all(out[~may] == 7)
    if sorted(starts) == starts and starts[0] >= 0:
        assert np.all(out[may] != 7)


@pytest.mark.parametrize("nq,nkv,hd", [(128, 2, 64), (128, 2, 128), (128, 2, 256)])
@pytest.mark.parametrize("less", [21, 23])
def test_long_tail_of_small_weights(gpu, nq, nkv, hd, less):
    """A first key over 40,000 equal ones of 2^-21 and 2^-23 of its weight, below fp16's normal range as the product takes
    them: they count alike in the sum of the values and in the divisor. Their weights are whole steps of fp16
    (the score's rounding, 23 * 2^-23, is far below half of one), and adding them to the first's loses nothing, so
    the row is off by its output's rounding and a few of fp32."""
    new, ctx = 270, 40000
    c = Case([(new, ctx)], nq, nkv, hd, 256, True, 53)
    c.q[:] = 0
    c.q[..., 3] = 4
    c.k[..., 3] = 0
    c.k[c.table[0, 0], :, 0, 3] = 8
    c.v[:] = 1
    c.v[c.table[0, 0], :, 0] = 0
    scale = np.float32(less * np.log(2) / 32)
    t = np.exp(-32 * np.float64(scale))
    n = ctx + np.arange(new)[:, None, None]
    want = n * t / (1 + n * t)
    got = c.run(gpu, scale=float(scale)).astype(np.float64)
    assert np.all(np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -17) * want), np.max(np.abs(got / want - 1))


def test_most_rows_of_256_dims(gpu):
    """2^26 rows (token, head) of 256 dims, 32 GiB in place: the last token's keys are split, its parts joined; every
    other token sees no key."""
    tokens, seqs, heads, hd = 1 << 20, 8192, 64, 256
    c = Case([(1, 271)], heads, heads, hd, 16, True, 55)
    want = c.run(gpu)
    row = 2 * heads * hd
    Q = gpu.DeviceBuffer(tokens * row)
    gpu._hip(gpu.lib().hip.hipMemset(Q.ptr, 0x3C, Q.nbytes), "hipMemset")
    small = gpu.DeviceBuffer.from_array(c.q.view(np.uint16))
    gpu._hip(gpu.lib().hip.hipMemcpy(Q.ptr + Q.nbytes - row, small.ptr, row, 3), "hipMemcpy")
    start = np.minimum(np.arange(seqs + 1) * 129, tokens - 1)
    start[-1] = tokens
    kv = np.zeros(seqs, np.int32)
    kv[-1] = 272
    table = np.full((seqs, c.width), -1, np.int32)
    table[-1] = c.table[0]
    batch = gpu.PagedBatch(seqs, tokens, c.width, i32(gpu, start), i32(gpu, kv), i32(gpu, table))
    cache = gpu.PagedCache(gpu.DeviceBuffer.from_array(c.k.view(np.uint16)),
                           gpu.DeviceBuffer.from_array(c.v.view(np.uint16)), c.blocks, 16, heads, hd)
    gpu.paged_attention(batch, cache, Q, 1, heads * hd, heads, Q, heads * hd,
                        gpu.paged_attention_workspace(batch, cache, heads))
    gpu.synchronize()
    last = Q.view(Q.nbytes - 64 * row, 64 * row).download(np.uint16).reshape(64, -1)
    assert np.array_equal(last[-1], want.view(np.uint16).reshape(-1))
    assert not last[:-1].any()
    Q.close()
