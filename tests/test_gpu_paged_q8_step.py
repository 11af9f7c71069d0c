"""A serving step over 8-bit pages in a row, as a serving program runs it: prompts
of three requests through one step, then decode steps from one captured graph
(tables, the norm before the block, projection, norms and rotation into 8-bit
pages, attention, output, the norms and residual between the blocks, head,
sampling, log probabilities). After every step each operator's outputs are
checked against the 64-bit references on the device's own inputs to it, so that
a code next to a border is the same on both sides.

Bars: products within rel-L2 1e-3 of the restatement, their own bar; codes, tables and tokens equal;
attention (fp32 rows, up to 40 keys of magnitude about 1) and norms within 2^-17 of the magnitudes that are
summed, some 20 times what their own tests allow at these sizes; log probabilities and entropies within 2^-18 (1 + |value|).
"""
import numpy as np
import pytest

import oracle
from oracle import paged as ref
from rqmv import synth
from tests.test_gpu_paged_q8 import pages_back

pytestmark = pytest.mark.gpu

D, NQ, NKV, HD, VOCAB, BLOCK, ROWS, TOP = 256, 4, 2, 64, 5000, 16, 64, 8
QKV = (NQ + 2 * NKV) * HD
EPS, SCALE = 1e-5, 0.5


def i32(gpu, a):
    return gpu.DeviceBuffer.from_array(np.asarray(a, np.int32))


class Server:
    def __init__(self, gpu, seed):
        self.gpu = gpu
        rng = np.random.default_rng(seed)
        w = {"qkv": ("q4_k", QKV, D), "o": ("q4_k", D, NQ * HD), "head": ("q8_0", VOCAB, D)}
        blocks = {k: synth.weights(f, r, c, seed + i) for i, (k, (f, r, c)) in enumerate(w.items())}
        self.w = {k: gpu.Weight(f, r, c, blocks[k]) for k, (f, r, c) in w.items()}
        self.host = {k: oracle.dequant_rows(f, blocks[k], r, c).astype(np.float64) for k, (f, r, c) in w.items()}
        self.embed = rng.standard_normal((VOCAB, D)).astype(np.float32)
        near = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
        self.norms = {"q": near(HD), "k": near(HD), "in": near(D), "post": near(D), "out": near(D),
                      "gate": np.tanh(rng.standard_normal((1, D))).astype(np.float32)}
        self.dev = {k: gpu.DeviceBuffer.from_array(v) for k, v in self.norms.items()}
        self.dev["embed"] = gpu.DeviceBuffer.from_array(self.embed)
        self.blocks = 24
        self.cache = gpu.PagedCacheQ8.allocate(self.blocks, BLOCK, NKV, HD)
        for buf in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale):
            buf.upload(rng.integers(0, 256, buf.nbytes).astype(np.uint8) | 1)  # (what another program left)
        self.table = gpu.rope_table(HD, 10000.0, ROWS)

    def buffers(self, rows, batch):
        f = lambda n: self.gpu.DeviceBuffer(4 * n)  # noqa: E731
        return {"x": f(rows * D), "h": f(rows * D), "qkv": f(rows * QKV), "q": f(rows * NQ * HD), "a": f(rows * NQ * HD),
                "o": f(rows * D), "x2": f(rows * D), "h2": f(rows * D), "logits": f(rows * VOCAB), "u": f(rows),
                "token": f(rows), "prob": f(rows), "logprob": f(rows), "entropy": f(rows), "top_tokens": f(rows * TOP),
                "top_logprobs": f(rows * TOP), "ws": self.gpu.sample_workspace(rows, VOCAB),
                "lp_ws": self.gpu.logprobs_workspace(rows, VOCAB, TOP),
                "attn_ws": self.gpu.paged_attention_q8_workspace(batch, self.cache, NQ)}

    def layer(self, batch, b, rows, temperature, stream):
        g = self.gpu
        g.block_norm(b["x"], rows, D, pre_norm=self.dev["in"], eps=EPS, out=b["h"], stream=stream)
        self.w["qkv"].matvec(b["h"], g.DTYPE_F32, rows, D, b["qkv"], QKV, stream)
        g.qk_norm_rope_q8(batch, self.cache, b["qkv"], g.DTYPE_F32, QKV, NQ, self.table, ROWS, b["q"], g.DTYPE_F32, NQ * HD,
                          self.dev["q"], self.dev["k"], EPS, stream=stream)
        g.paged_attention_q8(batch, self.cache, b["q"], g.DTYPE_F32, NQ * HD, NQ, b["a"], NQ * HD, b["attn_ws"],
                             stream=stream)
        self.w["o"].matvec(b["a"], g.DTYPE_F32, rows, NQ * HD, b["o"], D, stream)
        g.block_norm(b["x"], rows, D, delta=b["o"], post_norm=self.dev["post"], gate=self.dev["gate"], scale=SCALE,
                     pre_norm=self.dev["out"], eps=EPS, x_out=b["x2"], out=b["h2"], stream=stream)
        self.w["head"].matvec(b["h2"], g.DTYPE_F32, rows, D, b["logits"], VOCAB, stream)
        g.sample(b["logits"], rows, VOCAB, VOCAB, b["u"], b["token"], b["ws"], temperature, None, None, None, b["prob"],
                 stream)
        g.logprobs(b["logits"], rows, VOCAB, VOCAB, tokens=b["token"], logprob=b["logprob"], entropy=b["entropy"], top=TOP,
                   top_tokens=b["top_tokens"], top_logprobs=b["top_logprobs"], workspace=b["lp_ws"], stream=stream)

    def pages(self):
        return pages_back(self.cache, (self.blocks, NKV, BLOCK, HD))

    def check(self, b, x, before, live, q_start, kv_len, table, positions, slots, u, temperature):
        """Every stage of a step against its reference, on what the stage before left on the device."""
        n = self.norms
        at = {k: b[k].download(np.float32).reshape(len(x), -1)[:live].astype(np.float64) for k in
              ("h", "qkv", "q", "a", "o", "x2", "h2", "logits", "logprob", "entropy", "prob", "top_logprobs")}
        eps = float(np.float32(EPS))

        def close(got, want, size):
            assert np.all(np.abs(got - want) <= 2.0 ** -17 * size)

        def product(got, want):
            assert np.linalg.norm(got - want) <= 1e-3 * np.linalg.norm(want)

        x = x[:live].astype(np.float64)
        _, h = ref.block_norm(x, pre=n["in"], eps=eps)
        close(at["h"], h, np.abs(h))
        product(at["qkv"], at["h"] @ self.host["qkv"].T)
        cs = self.table.download(np.float32).reshape(ROWS, HD // 2, 2)
        q, k, v = ref.qk_norm_rope(at["qkv"], NQ, NKV, HD, n["q"], n["k"], eps, cs, HD, positions[:live])
        close(at["q"], q.reshape(live, -1), 4.0)
        now = self.pages()
        for i, y in ((0, k), (2, v)):
            codes, scale = ref.store_q8(before[i], before[i + 1], y, slots[:live])
            assert np.array_equal(now[i + 1], scale)
            fine = np.repeat(scale != 255, 16, axis=2)
            assert np.array_equal(now[i][fine], codes[fine])
        keys, values = ref.values_q8(now[0], now[1]), ref.values_q8(now[2], now[3])
        q = at["q"].reshape(live, NQ, HD)
        a = ref.attention(q, keys, values, q_start, kv_len, table, table.shape[1], HD ** -0.5)
        size = ref.attention(q, keys, np.abs(values), q_start, kv_len, table, table.shape[1], HD ** -0.5)
        close(at["a"], a.reshape(live, -1), size.reshape(live, -1))
        product(at["o"], at["a"] @ self.host["o"].T)
        x2, h2 = ref.block_norm(x, at["o"], n["post"], n["gate"], SCALE, n["out"], eps)
        close(at["x2"], x2, np.abs(x2) + np.abs(x2 - x))
        close(at["h2"], h2, np.abs(h2) + 1.0)
        product(at["logits"], at["h2"] @ self.host["head"].T)
        logits = at["logits"].astype(np.float32)
        tokens = b["token"].download(np.int32)[:live]
        top = b["top_tokens"].download(np.int32).reshape(-1, TOP)
        for r in range(live):
            t, p = ref.sample(logits[r], np.float32(u[r]), temperature[r])
            assert tokens[r] == t and abs(at["prob"][r, 0] - p) <= 2.0 ** -23
            lp, entropy, best, best_lp = ref.logprobs(logits[r], t, TOP)
            assert top[r].tolist() == best
            for got, want in ((at["logprob"][r, 0], lp), (at["entropy"][r, 0], entropy), *zip(at["top_logprobs"][r], best_lp)):
                assert abs(got - want) <= 2.0 ** -18 * (1 + abs(want))
        return tokens


def test_prompts_then_captured_decode_steps(gpu):
    rng = np.random.default_rng(31)
    s = Server(gpu, 40)
    new, seqs, rows, width = [5, 17, 1], 3, 24, 4
    free = rng.permutation(s.blocks).astype(np.int32)
    F, H, ST, table = i32(gpu, free), i32(gpu, [0]), i32(gpu, [9]), np.full((seqs, width), -1, np.int32)
    stream = gpu.Stream()

    # the prompts: 23 live rows of 24
    batch = gpu.PagedBatch.allocate(seqs, rows, width)
    b = s.buffers(rows, batch)
    x = s.embed[rng.integers(0, VOCAB, rows)]
    u, temperature = rng.random(rows).astype(np.float32), np.full(rows, 0.8, np.float32)
    b["x"].upload(x)
    b["u"].upload(u)
    before = s.pages()
    gpu.paged_plan(batch, s.cache, i32(gpu, [0] * seqs), i32(gpu, new), F, len(free), H, H, ST, stream)
    s.layer(batch, b, rows, gpu.DeviceBuffer.from_array(temperature), stream)
    stream.synchronize()
    status, q_start, kv_len, table, positions, slots, head = ref.plan([0] * seqs, new, table, free, 0, BLOCK, s.blocks, rows)
    assert status == 0 and int(ST.download(np.int32)[0]) == 0
    assert np.array_equal(batch.slots.download(np.int32), slots)
    tokens = s.check(b, x, before, int(q_start[-1]), q_start, kv_len, table, positions, slots, u, temperature)
    last = [int(tokens[q_start[i + 1] - 1]) for i in range(seqs)]

    # one decode step of every request, captured with its plan and embeddings; lengths and pool go on in place
    step = gpu.PagedBatch(seqs, seqs, width, i32(gpu, [0] * (seqs + 1)), batch.kv_len, batch.block_table,
                          i32(gpu, [0] * seqs), i32(gpu, [0] * seqs))
    d = s.buffers(seqs, step)
    ones, temperature = i32(gpu, [1] * seqs), np.array([0.0, 0.8, 1.2], np.float32)
    T = gpu.DeviceBuffer.from_array(temperature)
    d["token"].upload(np.array(last, np.int32))
    gpu.synchronize()

    def enqueue():
        gpu.paged_plan(step, s.cache, step.kv_len, ones, F, len(free), H, H, ST, stream)
        for i in range(seqs):
            gpu.embed_row(s.dev["embed"], VOCAB, D, d["token"].view(4 * i, 4), d["x"].view(4 * D * i, 4 * D), stream)
        s.layer(step, d, seqs, T, stream)

    graph = gpu.Graph(stream, enqueue)
    for _ in range(14):  # past a page's end for every request
        u = rng.random(seqs).astype(np.float32)
        d["u"].upload(u)
        before = s.pages()
        graph.launch(stream)
        stream.synchronize()
        assert int(ST.download(np.int32)[0]) == 0
        status, q_start, kv_len, table, positions, slots, head = ref.plan(
            [int(v) for v in kv_len], [1] * seqs, table, free, head, BLOCK, s.blocks, seqs)
        assert np.array_equal(step.kv_len.download(np.int32), kv_len)
        last = [int(t) for t in s.check(d, s.embed[last], before, seqs, q_start, kv_len, table, positions, slots, u, temperature)]
    graph.close()
