"""The paged serving operators in a row, as a serving program runs them: prompts
of three requests through one step, then decode steps from one captured graph
(tables, projection, norms and rotation, attention, output, head, sampling),
against a host restatement in 64 bits; and drawn tokens in DecodeModel.

Bars: logits within rel-L2 1e-3 of the restatement, the quantized products' own
bar; tables equal; tokens those that oracle/paged.py draws from the device's
logits.
"""
import gc

import numpy as np
import pytest

import oracle
from oracle import paged as ref
from rqmv import synth
from rqmv.decode import DecodeModel, DecoderShape

pytestmark = pytest.mark.gpu

D, NQ, NKV, HD, VOCAB, BLOCK, ROWS = 256, 4, 2, 64, 512, 16, 64
QKV = (NQ + 2 * NKV) * HD
EPS = 1e-5


def i32(gpu, a):
    return gpu.DeviceBuffer.from_array(np.asarray(a, np.int32))


class Server:
    """One attention layer and a head on the device, and the same on the host."""

    def __init__(self, gpu, seed):
        self.gpu = gpu
        rng = np.random.default_rng(seed)
        w = {"qkv": ("q4_k", QKV, D), "o": ("q4_k", D, NQ * HD), "head": ("q8_0", VOCAB, D)}
        blocks = {k: synth.weights(f, r, c, seed + i) for i, (k, (f, r, c)) in enumerate(w.items())}
        self.w = {k: gpu.Weight(f, r, c, blocks[k]) for k, (f, r, c) in w.items()}
        self.host = {k: oracle.dequant_rows(f, blocks[k], r, c).astype(np.float64) for k, (f, r, c) in w.items()}
        self.embed = rng.standard_normal((VOCAB, D)).astype(np.float32)
        self.norms = [(1 + 0.1 * rng.standard_normal(HD)).astype(np.float32) for _ in range(2)]
        self.blocks = 24
        self.cache = gpu.PagedCache.allocate(self.blocks, BLOCK, NKV, HD)
        self.table = gpu.rope_table(HD, 10000.0, ROWS)
        self.dev = {"embed": gpu.DeviceBuffer.from_array(self.embed),
                    "qn": gpu.DeviceBuffer.from_array(self.norms[0]), "kn": gpu.DeviceBuffer.from_array(self.norms[1])}
        self.k = np.zeros((self.blocks, NKV, BLOCK, HD), np.float16)  # the host's pages
        self.v = np.zeros_like(self.k)

    def buffers(self, rows):
        f = lambda n: self.gpu.DeviceBuffer(4 * n)  # noqa: E731
        return {"x": f(rows * D), "qkv": f(rows * QKV), "q": f(rows * NQ * HD), "a": f(rows * NQ * HD), "y": f(rows * D),
                "logits": f(rows * VOCAB), "u": f(rows), "token": f(rows), "prob": f(rows),
                "ws": self.gpu.sample_workspace(rows, VOCAB)}

    def layer(self, batch, b, rows, temperature, top_k, stream):
        """Everything between the activations in b["x"] and the tokens in b["token"]."""
        g = self.gpu
        self.w["qkv"].matvec(b["x"], g.DTYPE_F32, rows, D, b["qkv"], QKV, stream)
        g.qk_norm_rope(batch, self.cache, b["qkv"], g.DTYPE_F32, QKV, NQ, self.table, ROWS, b["q"], g.DTYPE_F32,
                       NQ * HD, self.dev["qn"], self.dev["kn"], EPS, stream=stream)
        g.paged_attention(batch, self.cache, b["q"], g.DTYPE_F32, NQ * HD, NQ, b["a"], NQ * HD, b["attn_ws"],
                          stream=stream)
        self.w["o"].matvec(b["a"], g.DTYPE_F32, rows, NQ * HD, b["y"], D, stream)
        self.w["head"].matvec(b["y"], g.DTYPE_F32, rows, D, b["logits"], VOCAB, stream)
        g.sample(b["logits"], rows, VOCAB, VOCAB, b["u"], b["token"], b["ws"], temperature, top_k, None, None, b["prob"],
                 stream)

    def reference(self, x, q_start, kv_len, table, positions, slots):
        """The same on the host; appends to the host's pages. Logits of the live rows."""
        live = int(q_start[-1])
        cs = self.table.download(np.float32).reshape(ROWS, HD // 2, 2)
        q, k, v = ref.qk_norm_rope(x[:live].astype(np.float64) @ self.host["qkv"].T, NQ, NKV, HD, self.norms[0],
                                   self.norms[1], EPS, cs, HD, positions[:live])
        for t in range(live):
            self.k[slots[t] // BLOCK, :, slots[t] % BLOCK] = k[t].astype(np.float16)
            self.v[slots[t] // BLOCK, :, slots[t] % BLOCK] = v[t].astype(np.float16)
        a = ref.attention(q, self.k, self.v, q_start, kv_len, table, table.shape[1], HD ** -0.5)
        return a.reshape(live, -1) @ self.host["o"].T @ self.host["head"].T

    def check(self, b, want, u, temperature, top_k):
        live = len(want)
        logits = b["logits"].download(np.float32).reshape(-1, VOCAB)[:live]
        assert np.linalg.norm(logits - want) <= 1e-3 * np.linalg.norm(want)
        tokens, probs = b["token"].download(np.int32), b["prob"].download(np.float32)
        for r in range(live):
            t, p = ref.sample(logits[r], np.float32(u[r]), temperature[r], top_k[r])
            assert tokens[r] == t and abs(probs[r] - p) <= 2.0 ** -23
        return tokens[:live]


def test_prompts_then_captured_decode_steps(gpu):
    rng = np.random.default_rng(31)
    s = Server(gpu, 40)
    new, seqs, rows, width = [5, 17, 1], 3, 24, 4
    free = rng.permutation(s.blocks).astype(np.int32)
    F, H, ST, table = i32(gpu, free), i32(gpu, [0]), i32(gpu, [9]), np.full((seqs, width), -1, np.int32)
    stream = gpu.Stream()

    # the prompts: 23 live rows of 24
    batch = gpu.PagedBatch.allocate(seqs, rows, width)
    b = s.buffers(rows)
    b["attn_ws"] = gpu.paged_attention_workspace(batch, s.cache, NQ)
    prompt = rng.integers(0, VOCAB, rows)
    x = s.embed[prompt]
    u, temperature, top_k = rng.random(rows).astype(np.float32), [0.8] * rows, [40] * rows
    b["x"].upload(x)
    b["u"].upload(u)
    cached = i32(gpu, [0] * seqs)
    gpu.paged_plan(batch, s.cache, cached, i32(gpu, new), F, len(free), H, H, ST, stream)
    s.layer(batch, b, rows, gpu.DeviceBuffer.from_array(np.array(temperature, np.float32)), i32(gpu, top_k), stream)
    stream.synchronize()
    status, q_start, kv_len, table, positions, slots, head = ref.plan([0] * seqs, new, table, free, 0, BLOCK, s.blocks, rows)
    assert status == 0 and int(ST.download(np.int32)[0]) == 0
    assert np.array_equal(batch.block_table.download(np.int32).reshape(seqs, width), table)
    tokens = s.check(b, s.reference(x, q_start, kv_len, table, positions, slots), u, temperature, top_k)
    last = [int(tokens[q_start[i + 1] - 1]) for i in range(seqs)]

    # one decode step of every request, captured with its plan and embeddings; lengths and pool go on in place
    step = gpu.PagedBatch(seqs, seqs, width, i32(gpu, [0] * (seqs + 1)), batch.kv_len, batch.block_table,
                          i32(gpu, [0] * seqs), i32(gpu, [0] * seqs))
    d = s.buffers(seqs)
    d["attn_ws"] = gpu.paged_attention_workspace(step, s.cache, NQ)
    ones = i32(gpu, [1] * seqs)
    T, K = gpu.DeviceBuffer.from_array(np.array([0.0, 0.8, 1.2], np.float32)), i32(gpu, [0, 0, 20])
    d["token"].upload(np.array(last, np.int32))

    def enqueue():
        gpu.paged_plan(step, s.cache, step.kv_len, ones, F, len(free), H, H, ST, stream)
        for i in range(seqs):
            gpu.embed_row(s.dev["embed"], VOCAB, D, d["token"].view(4 * i, 4), d["x"].view(4 * D * i, 4 * D), stream)
        s.layer(step, d, seqs, T, K, stream)

    graph = gpu.Graph(stream, enqueue)
    for _ in range(14):  # past a page's end for every request
        u = rng.random(seqs).astype(np.float32)
        d["u"].upload(u)
        graph.launch(stream)
        stream.synchronize()
        assert int(ST.download(np.int32)[0]) == 0
        status, q_start, kv_len, table, positions, slots, head = ref.plan(
            [int(v) for v in kv_len], [1] * seqs, table, free, head, BLOCK, s.blocks, seqs)
        assert np.array_equal(step.kv_len.download(np.int32), kv_len)
        assert np.array_equal(step.slots.download(np.int32), slots)
        want = s.reference(s.embed[last], q_start, kv_len, table, positions, slots)
        last = [int(t) for t in s.check(d, want, u, [0.0, 0.8, 1.2], [0, 0, 20])]
    graph.close()


@pytest.mark.parametrize("captured", [False, True])
def test_decoder_draws_its_tokens(gpu, captured):
    """DecodeModel steps with a Sampling: tokens drawn from the step's logits, and at temperature 0 the argmax's."""
    shape = DecoderShape(layers=1, d=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=5000)
    syn = synth.DecoderSynth(shape, seed=3, norm_std=0.1)
    model = DecodeModel(shape, 32, syn.embed(), syn.out_norm(), syn.head())
    model.set_layer(0, syn.layer(0))
    model.set_cache(0, *syn.cache(0, 8))
    stream = gpu.Stream()
    sampling = model.sampling(temperature=0.9, top_k=50, top_p=0.95)
    model.set_position(7, 8)
    graph = model.capture(stream, sampling) if captured else None
    rng = np.random.default_rng(1)
    for _ in range(8):
        u = float(rng.random())
        sampling.set_random(u)
        if captured:
            model.replay(graph, stream)
        else:
            model.step(stream, sampling)
        stream.synchronize()
        want, p = ref.sample(model.read_logits(), np.float32(u), np.float32(0.9), 50, np.float32(0.95))
        assert model.read_token() == want and abs(sampling.read_prob() - p) <= 2.0 ** -23
    greedy = []
    for kw in ({}, {"sampling": model.sampling(temperature=0.0)}):
        model.set_position(7, 8)
        got = []
        for _ in range(4):
            model.step(stream, **kw)
            stream.synchronize()
            got.append(model.read_token())
        greedy.append(got)
    assert greedy[0] == greedy[1]
    # a graph outlives the name of its Sampling
    graph = model.capture(stream, model.sampling(temperature=0.0))
    gc.collect()
    junk = [gpu.DeviceBuffer.from_array(np.full(1 << 18, 0x7FC00000, np.uint32)) for _ in range(4)]
    model.set_position(7, 8)
    got = []
    for _ in range(4):
        model.replay(graph, stream)
        stream.synchronize()
        got.append(model.read_token())
    assert got == greedy[0] and len(junk) == 4
    graph.close()


def test_replays_of_a_drawing_step_go_one_at_a_time(gpu):
    """Several replays at once would draw with one random number; at temperature 0 none is drawn with."""
    shape = DecoderShape(layers=1, d=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=5000)
    syn = synth.DecoderSynth(shape, seed=3, norm_std=0.1)
    model = DecodeModel(shape, 32, syn.embed(), syn.out_norm(), syn.head())
    model.set_layer(0, syn.layer(0))
    model.set_cache(0, *syn.cache(0, 8))
    stream = gpu.Stream()
    tokens = []
    for sampling in (None, model.sampling(temperature=0.0)):
        graph = model.capture(stream, sampling)
        model.set_position(7, 8)
        model.replay(graph, stream, 4)
        stream.synchronize()
        tokens.append(model.read_token())
        graph.close()
    assert tokens[0] == tokens[1]
    graph = model.capture(stream, model.sampling(temperature=0.9))
    model.set_position(7, 8)
    with pytest.raises(ValueError, match="one random number"):
        model.replay(graph, stream, 2)
    assert model.read_position() == 8
    graph.sampling.set_random(0.5)
    model.replay(graph, stream)
    stream.synchronize()
    assert model.read_token() == ref.sample(model.read_logits(), np.float32(0.5), np.float32(0.9))[0]
    graph.close()
