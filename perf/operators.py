"""Performance cases of the paged serving operators.

What a program that serves several requests at once asks of the library around
its quantized products: the step's block tables and slot maps, the norms and
the rotation of queries and keys with the append to the paged cache, attention
of each sequence's new tokens over its pages, and the choice of the next tokens.

A case is a dict; `kind` says which operator it is:
  plan       rqmv.paged_plan
  qkv        rqmv.qk_norm_rope
  attention  rqmv.paged_attention
  sample     rqmv.sample

The lengths of a case's sequences follow from its `mix` alone, so that its work
is known without its inputs; tensors are drawn on the device from the seed.
`run` computes the operators from elementary torch operations, or with the
library's kernels where `own` is true.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROPE_BASE = 500000.0
EPS = 1e-6


# ------------------------------------------------------------------ cases ----

def attention(name, seqs, new, ctx, heads, block, x, mix, window=0):
    q_heads, kv_heads, head_dim = heads
    return {"name": name, "kind": "attention", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "x": x,
            "window": window, "mix": mix}


def qkv(name, tokens, heads, block, x, q, norm=True):
    q_heads, kv_heads, head_dim = heads
    return {"name": name, "kind": "qkv", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "block": block, "x": x, "q": q, "norm": norm}


def plan(name, seqs, new, ctx, block, mix):
    return {"name": name, "kind": "plan", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "block": block, "mix": mix}


def listed():
    return [
        # the tables of a decode step: every request has one new token
        plan("plan_decode_64", 64, (1, 1), (1, 8192), 16, 1),
        # the tables of a mixed step: prompts of any length beside decoding requests
        plan("plan_mixed_300", 300, (1, 400), (0, 16384), 32, 2),
        # the new token of one request, fp32 as the products give it
        qkv("qkv_decode_1", 1, (32, 8, 128), 16, "f32", "f32"),
        # an odd number of requests decoded together, queries rounded for the matrix cores
        qkv("qkv_decode_33", 33, (16, 2, 64), 32, "f32", "f16"),
        # a prefill step
        qkv("qkv_prefill_4096", 4096, (32, 8, 128), 64, "f32", "f16"),
        # one request decoding at a context of 4,097
        attention("attention_decode_1", 1, (1, 1), (4096, 4096), (32, 8, 128), 16, "f32", 3),
        # requests of very different lengths decoded together
        attention("attention_decode_32", 32, (1, 1), (60, 8192), (32, 8, 128), 64, "f16", 4),
        # a few speculated tokens of each of eight requests, fp32 throughout
        attention("attention_verify_5", 8, (5, 5), (300, 3000), (16, 2, 64), 32, "f32", 5),
        # ragged prompts from their first token on, wide heads, fp32 throughout
        attention("attention_prompts_f32", 5, (17, 900), (0, 0), (8, 4, 256), 16, "f32", 6),
        # a chunk of a long prompt over what its earlier chunks left in the cache
        attention("attention_chunk_2048", 1, (2048, 2048), (14336, 14336), (32, 8, 128), 128, "f16", 7),
        # the next token of one request
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 128256, "top_k": 50, "flat": False},
        # the next tokens of a batch, each request with its own settings, top-k off for half of them
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": 128256, "top_k": 0, "flat": False},
    ]


MOST_PAIRS = 2048 * 16384 * 32 * 128  # the largest attention: padded (token, key) pairs x query heads x head_dim
HEADS = ((32, 8, 128), (16, 2, 128), (4, 4, 128), (12, 4, 128), (28, 4, 128), (16, 2, 64), (24, 8, 64), (8, 4, 256),
         (8, 1, 256), (32, 2, 64))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "qkv", "attention", "attention", "attention", "sample"))
    heads, block, mix = rng.choice(HEADS), rng.choice((16, 32, 64, 128, 256)), rng.randrange(1 << 30)
    if kind == "plan":
        seqs = _log(rng, 1, 512)
        hi = _log(rng, 1, 16384 // seqs)
        case = plan("", seqs, (rng.choice((1, hi)), hi), (rng.choice((0, 1, 100)), _log(rng, 100, 16384)), block, mix)
    elif kind == "qkv":
        case = qkv("", _log(rng, 1, 4096), heads, block, rng.choice(("f32", "f16")), rng.choice(("f32", "f16")),
                   rng.random() < 0.75)
    elif kind == "attention":
        while True:
            seqs = _log(rng, 1, 64)
            new_hi = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 16, 2048)))
            ctx_hi = rng.choice((0, _log(rng, 10, 14336), _log(rng, 10, 14336)))
            if seqs * new_hi * (new_hi + ctx_hi) * heads[0] * heads[2] <= MOST_PAIRS and \
                    seqs * (new_hi + ctx_hi) * heads[1] * heads[2] <= 1 << 28:
                break
        case = attention("", seqs, (rng.randint(1, new_hi), new_hi), (rng.randint(0, ctx_hi), ctx_hi), heads, block,
                         rng.choice(("f32", "f16", "f16")), mix, rng.choice((0, 0, 0, _log(rng, 16, 4096))))
    else:
        case = {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 128256),
                "top_k": rng.choice((0, 1, 20, 50, 200, 1000)), "flat": rng.random() < 0.25}
    case.pop("name", None)
    return case


def lengths(case):
    """(new, cached) tokens of each sequence."""
    rng = random.Random(case["mix"])
    new, ctx = [], []
    for _ in range(case["seqs"]):
        new.append(_log(rng, case["new_lo"], case["new_hi"]))
        ctx.append(_log(rng, case["ctx_lo"] + 1, case["ctx_hi"] + 1) - 1)
    return new, ctx


# ----------------------------------------------------------------- inputs ----

class Memory:
    """A tensor's memory as the library takes device memory."""

    def __init__(self, t):
        self.keep, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _type(x):
    return torch.float16 if x == "f16" else torch.float32


def _pages(n, block):
    return (n + block - 1) // block


def _plan_inputs(case, seed):
    new, ctx = lengths(case)
    block = case["block"]
    held = [_pages(c, block) for c in ctx]
    need = [_pages(c + n, block) for n, c in zip(new, ctx)]
    width = max(need) + 3
    blocks = sum(need) + 40
    ids = torch.randperm(blocks, device="cuda", generator=_gen(seed)).int()
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < _ints(held)[:, None]
    table[at] = ids[:sum(held)]
    # the pool: blocks that other requests hold by now, then the free ones
    pool = torch.cat((ids[:7], ids[sum(held):]))
    tokens = _pages(sum(new), 64) * 64  # the step's token buffers, a whole number of 64 rows
    return {"new": _ints(new), "ctx": _ints(ctx), "table": table, "free": pool.contiguous(), "head": _ints([7]),
            "tokens": tokens, "blocks": blocks, "width": width}


def _rope_table(head_dim, rows):
    half = head_dim // 2
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * torch.exp(
        -2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / head_dim * math.log(ROPE_BASE))
    return torch.stack((torch.cos(angle), torch.sin(angle)), 2).float().contiguous()


def _qkv_inputs(case, seed):
    g = _gen(seed)
    nq, nkv, hd, t, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["tokens"], case["block"]
    blocks = 2 * _pages(t, block) + 4
    rows = 8192
    x = torch.randn(t, (nq + 2 * nkv) * hd, device="cuda", generator=g) * 2.0
    return {"x": x.to(_type(case["x"])), "rope": _rope_table(hd, rows), "rows": rows, "blocks": blocks,
            "q_norm": 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=g),
            "k_norm": 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=g),
            "pos": torch.randint(0, rows, (t,), device="cuda", generator=g).int(),
            "slots": torch.randperm(blocks * block, device="cuda", generator=g)[:t].int().contiguous(),
            "k": torch.randn(blocks, nkv, block, hd, device="cuda", generator=g).half(),
            "v": torch.randn(blocks, nkv, block, hd, device="cuda", generator=g).half()}


def _attention_inputs(case, seed):
    g = _gen(seed)
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    new, ctx = lengths(case)
    need = [_pages(c + n, block) for n, c in zip(new, ctx)]
    width, blocks = max(need), sum(need) + 3
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < _ints(need)[:, None]
    table[at] = torch.randperm(blocks, device="cuda", generator=g).int()[:sum(need)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return {"q": (torch.randn(start[-1], nq * hd, device="cuda", generator=g) * 1.5).to(_type(case["x"])),
            "k": torch.randn(blocks, nkv, block, hd, device="cuda", generator=g).half(),
            "v": torch.randn(blocks, nkv, block, hd, device="cuda", generator=g).half(),
            "start": _ints(start), "kv_len": _ints([c + n for n, c in zip(new, ctx)]), "table": table,
            "tokens": start[-1], "blocks": blocks, "width": width, "most_new": max(new)}


def _sample_inputs(case, seed):
    g = _gen(seed)
    m, n = case["rows"], case["vocab"]
    logits = torch.randn(m, n, device="cuda", generator=g) * (0.5 if case["flat"] else 3.0)

    def one_of(values):
        at = torch.randint(0, len(values), (m,), device="cuda", generator=g)
        return torch.tensor(values, device="cuda")[at].contiguous()

    top_k = one_of([case["top_k"]] if case["top_k"] else [0, 0, 40, 500]).int()
    return {"logits": logits, "u": torch.rand(m, device="cuda", generator=g), "top_k": top_k,
            "temperature": one_of([0.6, 0.8, 1.0, 1.0, 1.3] + ([0.0] if m > 8 else [])),
            "top_p": one_of([0.8, 0.95, 1.0]), "min_p": one_of([0.0, 0.0, 0.02])}


_INPUTS = {"plan": _plan_inputs, "qkv": _qkv_inputs, "attention": _attention_inputs, "sample": _sample_inputs}


# ---------------------------------------------------------------- prepare ----

def prepare(case, seed):
    t = _INPUTS[case["kind"]](case, seed)
    out = {}
    if case["kind"] == "plan":
        out = {"start": torch.empty(case["seqs"] + 1, dtype=torch.int32, device="cuda"),
               "kv_len": torch.empty(case["seqs"], dtype=torch.int32, device="cuda"),
               "pos": torch.empty(t["tokens"], dtype=torch.int32, device="cuda"),
               "slots": torch.empty(t["tokens"], dtype=torch.int32, device="cuda"),
               "head_out": torch.empty(1, dtype=torch.int32, device="cuda"),
               "status": torch.empty(1, dtype=torch.int32, device="cuda")}
    elif case["kind"] == "qkv":
        out = {"out": torch.empty(case["tokens"], case["q_heads"] * case["head_dim"], dtype=_type(case["q"]),
                                  device="cuda")}
    elif case["kind"] == "attention":
        out = {"out": torch.empty_like(t["q"])}
    else:
        out = {"token": torch.empty(case["rows"], dtype=torch.int32, device="cuda"),
               "prob": torch.empty(case["rows"], device="cuda")}
    t.update(out)
    memory = {k: Memory(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
    return {"case": case, "t": t, "memory": memory}


# -------------------------------------------------------------- plain form ----

def _plain_plan(case, t):
    block, width, tokens = case["block"], t["width"], t["tokens"]
    new, ctx, table = t["new"].long(), t["ctx"].long(), t["table"].long()
    end = torch.cumsum(new, 0)
    held, need = (ctx + block - 1) // block, (ctx + new + block - 1) // block
    taken = torch.cumsum(need - held, 0)
    at = torch.arange(width, device="cuda")[None, :]
    entry = t["head"].long() + (taken - need + held)[:, None] + at - held[:, None]
    fresh = (at >= held[:, None]) & (at < need[:, None])
    table = torch.where(fresh, t["free"].long()[entry.clamp(0, t["free"].numel() - 1)], table)
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(end, token, right=True).clamp(max=case["seqs"] - 1)
    real = token < end[-1]
    pos = torch.where(real, token - (end - new)[seq] + ctx[seq], torch.zeros_like(token))
    slot = table[seq, (pos // block).clamp(max=width - 1)] * block + pos % block
    slot = torch.where(real, slot, torch.full_like(slot, -1))
    return {"start": torch.cat((end.new_zeros(1), end)).int(), "kv_len": (ctx + new).int(), "pos": pos.int(),
            "slots": slot.int(), "table": table.int(), "head": (t["head"] + taken[-1:]).int(),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _plain_qkv(case, t):
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    half = hd // 2
    x = t["x"].float().reshape(case["tokens"], nq + 2 * nkv, hd)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    if case["norm"]:
        w = torch.cat((t["q_norm"].expand(nq, hd), t["k_norm"].expand(nkv, hd)))
        qk = qk / torch.sqrt((qk * qk).mean(2, keepdim=True) + EPS) * w
    cs = t["rope"][t["pos"].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    a, b = qk[..., :half], qk[..., half:]
    qk = torch.cat((a * cos - b * sin, b * cos + a * sin), 2)
    slot = t["slots"].long()
    t["k"][slot // block, :, slot % block] = qk[:, nq:].half()
    t["v"][slot // block, :, slot % block] = v.half()
    return {"q": qk[:, :nq].reshape(case["tokens"], nq * hd).to(_type(case["q"])), "k": t["k"], "v": t["v"]}


def _plain_attention(case, t):
    nq, nkv, hd, block, seqs = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "block", "seqs"))
    group, most = nq // nkv, t["most_new"]
    start, kv_len = t["start"].long(), t["kv_len"].long()
    new = start[1:] - start[:-1]
    # every sequence padded to the longest: its pages in order, its tokens from its first on
    page = t["table"].long().clamp(min=0)
    keys = t["k"][page].float().permute(0, 2, 1, 3, 4).reshape(seqs, nkv, -1, hd)
    values = t["v"][page].float().permute(0, 2, 1, 3, 4).reshape(seqs, nkv, -1, hd)
    token = torch.arange(most, device="cuda")
    row = (start[:-1, None] + token).clamp(max=t["tokens"] - 1)
    q = t["q"].float()[row].reshape(seqs, most, nkv, group, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(seqs, nkv, group * most, hd), keys.transpose(2, 3).contiguous()) / math.sqrt(hd)
    pos = (kv_len - new)[:, None] + token
    at = torch.arange(keys.shape[2], device="cuda")
    seen = at <= pos[..., None]
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]
    s = s.reshape(seqs, nkv, group, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(seqs, nkv, group * most, -1), values).reshape(seqs, nkv, group, most, hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs * most, nq * hd)
    # back to the ragged rows
    every = torch.arange(t["tokens"], device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), every, right=True)
    return o[seq * most + every - start[seq]].to(t["q"].dtype)


def _plain_sample(case, t):
    logits = t["logits"]
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)
    greedy = t["temperature"][:, None] <= 0
    temperature = torch.where(greedy, torch.ones_like(t["temperature"][:, None]), t["temperature"][:, None]).double()
    e = torch.exp((value.double() - value[:, :1].double()) / temperature)
    rank = torch.arange(case["vocab"], device="cuda")
    k = torch.where(t["top_k"] > 0, t["top_k"].long(), case["vocab"])[:, None]
    e = torch.where(rank < k, e, torch.zeros_like(e))
    end = torch.cumsum(e, 1)
    target = t["top_p"].double()[:, None] * end[:, -1:]
    kept = ((end - e < target) | (rank == 0)) & (e >= t["min_p"].double()[:, None])
    e = torch.where(kept, e, torch.zeros_like(e))
    total = e.sum(1, keepdim=True)
    at = (torch.cumsum(e, 1) <= t["u"].double()[:, None] * total).sum(1, keepdim=True)
    at = torch.where(greedy, torch.zeros_like(at), torch.minimum(at, (e > 0).sum(1, keepdim=True) - 1))
    prob = torch.where(greedy, torch.ones_like(total), torch.gather(e, 1, at) / total)
    return {"token": torch.gather(order, 1, at)[:, 0].int(), "prob": prob[:, 0].float()}


_PLAIN = {"plan": _plain_plan, "qkv": _plain_qkv, "attention": _plain_attention, "sample": _plain_sample}


# -------------------------------------------------------- the library's way ----

_ready = []


def _library():
    if not _ready:
        sys.path.insert(0, os.path.join(ROOT, "recipe-dev_amd"))
        import rqmv

        rqmv.init(0)
        _ready.append(rqmv)
    return _ready[0]


class _Kept:
    """What a serving program keeps from step to step: the cache's and the batch's descriptions, a workspace."""

    def __init__(self, case, t, m):
        rqmv = _library()
        kind = case["kind"]
        if kind == "sample":
            size = rqmv.sample_workspace_size(case["rows"], case["vocab"])
        else:
            none = Memory(torch.empty(0, device="cuda"))
            heads = (case.get("kv_heads", 1), case.get("head_dim", 128))
            self.cache = rqmv.PagedCache(m.get("k", none), m.get("v", none), t["blocks"], case["block"], *heads)
            self.batch = rqmv.PagedBatch(case.get("seqs", 1), t.get("tokens", case.get("tokens")), t.get("width", 1),
                                         q_start=m.get("start"), kv_len=m.get("kv_len"), block_table=m.get("table"),
                                         positions=m.get("pos"), slots=m.get("slots"))
            size = 0
            if kind == "attention":
                size = rqmv.paged_attention_workspace_size(self.batch, self.cache, case["q_heads"])
        self.workspace = Memory(torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"))


def _run_own(s):
    rqmv = _library()
    case, t, m = s["case"], s["t"], s["memory"]
    if "kept" not in s:
        s["kept"] = _Kept(case, t, m)
    kept, kind = s["kept"], case["kind"]
    f = {"f32": rqmv.DTYPE_F32, "f16": rqmv.DTYPE_F16}
    if kind == "plan":
        rqmv.paged_plan(kept.batch, kept.cache, m["ctx"], m["new"], m["free"], t["free"].numel(), m["head"],
                        m["head_out"], m["status"])
        return {"start": t["start"], "kv_len": t["kv_len"], "pos": t["pos"], "slots": t["slots"], "table": t["table"],
                "head": t["head_out"], "status": t["status"]}
    if kind == "qkv":
        nq, nkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
        norm = {"q_norm": m["q_norm"], "k_norm": m["k_norm"], "eps": EPS} if case["norm"] else {}
        rqmv.qk_norm_rope(kept.batch, kept.cache, m["x"], f[case["x"]], (nq + 2 * nkv) * hd, nq, m["rope"], t["rows"],
                          m["out"], f[case["q"]], nq * hd, **norm)
        return {"q": t["out"], "k": t["k"], "v": t["v"]}
    if kind == "attention":
        row = case["q_heads"] * case["head_dim"]
        rqmv.paged_attention(kept.batch, kept.cache, m["q"], f[case["x"]], row, case["q_heads"], m["out"], row,
                             kept.workspace, window=case["window"])
        return t["out"]
    rqmv.sample(m["logits"], case["rows"], case["vocab"], case["vocab"], m["u"], m["token"], kept.workspace,
                temperature=m["temperature"], top_k=m["top_k"], top_p=m["top_p"], min_p=m["min_p"], prob=m["prob"])
    return {"token": t["token"], "prob": t["prob"]}


# -------------------------------------------------------------------- run ----

def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["kind"]](s["case"], s["t"])


# ------------------------------------------------------------------- work ----

def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 7), "flops": 4.0 * case["rows"] * case["vocab"]}
    if kind == "qkv":
        nq, nkv, hd, t = case["q_heads"], case["kv_heads"], case["head_dim"], case["tokens"]
        size = {"f32": 4, "f16": 2}
        # a row of the rotation table is shared by the tokens at its position, the norms' weights by all
        return {"bytes": float(t * ((nq + 2 * nkv) * hd * size[case["x"]] + nq * hd * size[case["q"]] + 2 * nkv * hd * 2 +
                                    8) + min(t, 8192) * hd * 4 + 8 * hd), "flops": 7.0 * t * (nq + nkv) * hd}
    new, ctx = lengths(case)
    if kind == "plan":
        block = case["block"]
        pages = sum(_pages(c + n, block) - _pages(c, block) for n, c in zip(new, ctx))
        # a token's page is read from the table where its request held it already
        return {"bytes": 4.0 * (4 * len(new) + 4 + 2 * sum(new) + 2 * pages + len(new)), "flops": 8.0 * sum(new)}
    nq, nkv, hd, window = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
    pairs = keys = 0
    for n, c in zip(new, ctx):
        if window:
            pairs += sum(min(c + i + 1, window) for i in range(n))
            keys += min(c + n, n - 1 + window)
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    size = 2 if case["x"] == "f16" else 4
    return {"bytes": float(keys * nkv * hd * 4 + 2 * sum(new) * nq * hd * size), "flops": 4.0 * pairs * nq * hd}


# ------------------------------------------------------------------ exact ----

def _exact_qkv(case, t):
    nq, nkv, hd, block, tokens = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "block", "tokens"))
    x = t["x"].double().reshape(tokens, -1, hd)
    heads = x[:, :nq + nkv].clone()
    if case["norm"]:
        heads /= (heads.square().sum(2, keepdim=True) / hd + EPS).sqrt()
        heads[:, :nq] *= t["q_norm"].double()
        heads[:, nq:] *= t["k_norm"].double()
    pair = torch.view_as_complex(torch.stack(heads.chunk(2, 2), 3).contiguous())
    # the rotation by the table's entries, which are what the operator is given
    turned = torch.view_as_real(pair * torch.view_as_complex(t["rope"][t["pos"].long()].double())[:, None])
    heads = torch.cat((turned[..., 0], turned[..., 1]), 2)
    k, v = t["k"].double(), t["v"].double()
    blk, off = t["slots"].long() // block, t["slots"].long() % block
    k[blk, :, off] = heads[:, nq:]
    v[blk, :, off] = x[:, nq + nkv:]
    return {"q": heads[:, :nq].reshape(tokens, -1), "k": k, "v": v}


def _exact_attention(case, t):
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    new, ctx = lengths(case)
    out, at = [], 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        pages = t["table"][i, :_pages(c + n, block)].long()
        pos = torch.arange(c, c + n, device="cuda")[:, None]
        key_pos = torch.arange(c + n, device="cuda")[None, :]
        hidden = key_pos > pos
        if case["window"]:
            hidden |= key_pos <= pos - case["window"]
        rows = torch.empty(n, nq, hd, dtype=torch.float64, device="cuda")
        for h in range(nq):
            k = t["k"][pages, h // (nq // nkv)].reshape(-1, hd)[:c + n].double()
            v = t["v"][pages, h // (nq // nkv)].reshape(-1, hd)[:c + n].double()
            q = t["q"][at:at + n, h * hd:(h + 1) * hd].double()
            s = (q @ k.t().contiguous() * hd ** -0.5).masked_fill_(hidden, -math.inf)
            rows[:, h] = torch.softmax(s, 1) @ v
        out.append(rows.reshape(n, nq * hd))
        at += n
    return torch.cat(out)


def _exact_sample(case, t):
    """Row by row, from the definition: the probability of the token that the draw gives."""
    probs = []
    host = {k: t[k].cpu() for k in ("logits", "temperature", "top_k", "top_p", "min_p", "u")}
    for i in range(case["rows"]):
        temperature = float(host["temperature"][i])
        if temperature <= 0:
            probs.append(1.0)
            continue
        v = torch.sort(host["logits"][i].double(), descending=True).values
        v = v[:int(host["top_k"][i]) or None]
        p = torch.softmax(v / temperature, 0)
        end = torch.cumsum(p, 0)
        count = int((end < float(host["top_p"][i])).sum()) + 1
        p = p[:count]
        p = p[p >= float(host["min_p"][i]) * p[0]]
        p = p / p.sum()
        at = int((torch.cumsum(p, 0) <= float(host["u"][i])).sum())
        probs.append(float(p[min(at, p.numel() - 1)]))
    return {"token": None, "prob": torch.tensor(probs, dtype=torch.float64)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None
    t = _INPUTS[kind](case, seed)
    return {"qkv": _exact_qkv, "attention": _exact_attention, "sample": _exact_sample}[kind](case, t)
