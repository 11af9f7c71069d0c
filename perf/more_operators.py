"""Performance cases of serving over 8-bit pages: the append, attention, the
probabilities behind the answers, and the norms between the blocks.

What a program that serves requests from a cache of 8 bits asks of the library
around its quantized products: the norms before and after a block with its gate
and the residual stream, queries and keys through their norms and the rotation
with keys and values into 8-bit pages, attention over those pages, and the log
probabilities of the tokens that came or were given.

A page's values are codes times a power of two: int8 codes
[blocks, kv_heads, block, head_dim], and for each 16 positions of a block and
head one scale byte b, which stands for 2^(b - 127).

A case is a dict; `kind` says which operator it is:
  append     rqmv.qk_norm_rope_q8, then rqmv.paged_values_q8 (the pages as the values they stand for)
  attention  rqmv.paged_attention_q8
  logprobs   rqmv.logprobs
  norm       rqmv.block_norm

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
ROWS = 8192             # positions of the rotation table
GROUP = 16              # positions that share a scale
LOW, HIGH = -24, 9      # exponents of a scale


# ------------------------------------------------------------------ cases ----

def _tokens(name, kind, seqs, new, ctx, heads, block, x, mix, **more):
    q_heads, kv_heads, head_dim = heads
    return {"name": name, "kind": kind, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "x": x,
            "mix": mix, **more}


def append(name, seqs, new, ctx, heads, block, x, q, mix, norm=True):
    return _tokens(name, "append", seqs, new, ctx, heads, block, x, mix, q=q, norm=norm)


def attention(name, seqs, new, ctx, heads, block, x, mix, window=0):
    return _tokens(name, "attention", seqs, new, ctx, heads, block, x, mix, window=window)


def logprobs(name, rows, vocab, top, rounded=False):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "rounded": rounded}


def norm(name, rows, n, out, post, gate, pre=True):
    return {"name": name, "kind": "norm", "rows": rows, "n": n, "out": out, "post": post, "gate": gate, "pre": pre}


def listed():
    return [
        # the new token of each of 24 requests
        append("append_decode_24", 24, (1, 1), (0, 8000), (32, 8, 128), 16, "f32", "f32", 1),
        # three speculated tokens of seven requests, wide heads, rows already rounded
        append("append_verify_3", 7, (3, 3), (100, 4000), (8, 4, 256), 32, "f16", "f16", 2),
        # a prefill step: prompts, and chunks of longer ones, of any length
        append("append_prefill_4000", 6, (200, 1500), (0, 3500), (32, 8, 128), 64, "f32", "f16", 3),
        # one request decoding at a context of 8,000
        attention("attention_decode_1", 1, (1, 1), (7999, 7999), (32, 8, 128), 16, "f32", 4),
        # requests of very different lengths decoded together
        attention("attention_decode_48", 48, (1, 1), (100, 12000), (32, 8, 128), 64, "f16", 5),
        # a few speculated tokens of each of six requests, within a window, fp32 throughout
        attention("attention_verify_4", 6, (4, 4), (900, 5000), (16, 2, 64), 32, "f32", 6, window=1000),
        # ragged prompts from their first token on, wide heads, fp32 throughout
        attention("attention_prompts_f32", 5, (17, 900), (0, 0), (8, 4, 256), 32, "f32", 7),
        # a chunk of a long prompt over what its earlier chunks left in the cache
        attention("attention_chunk_2000", 1, (2000, 2000), (12000, 12000), (32, 8, 128), 256, "f16", 8),
        # what the drawn tokens of a batch are reported with: their log probabilities, entropies, twenty alternatives
        logprobs("logprobs_step_17", 17, 128256, 20),
        # the tokens of a prompt scored
        logprobs("logprobs_prompt_1500", 1500, 128256, 0),
        # between two blocks of a decode step: after one, the residual, before the next
        norm("norm_decode_5", 5, 5120, "f32", True, "none"),
        # the same of a prefill step with a gate per channel, rounded for the matrix cores
        norm("norm_prefill_4096", 4096, 4096, "f16", True, "one"),
    ]


MOST_PAIRS = 2000 * 14000 * 32 * 128  # the largest attention: padded (token, key) pairs x query heads x head_dim
MOST_LOGITS = 1500 * 128256
HEADS = ((32, 8, 128), (16, 2, 128), (4, 4, 128), (12, 4, 128), (28, 4, 128), (16, 2, 64), (24, 8, 64), (8, 4, 256),
         (8, 1, 256), (32, 2, 64))
WIDTHS = (64, 512, 1024, 2048, 2880, 4096, 5120, 6144, 8192, 14336)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "append", "attention", "attention", "attention", "logprobs", "norm"))
    heads, block, mix = rng.choice(HEADS), rng.choice((16, 32, 64, 128, 256)), rng.randrange(1 << 30)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        hi = rng.choice((1, _log(rng, 1, 16), _log(rng, 1, 4000 // seqs)))
        case = append("", seqs, (rng.choice((1, hi)), hi), (rng.choice((0, 1, 100)), _log(rng, 100, 4000)), heads,
                      block, rng.choice(("f32", "f16")), rng.choice(("f32", "f16")), mix, rng.random() < 0.75)
    elif kind == "attention":
        while True:
            seqs = _log(rng, 1, 64)
            new_hi = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 16, 2000)))
            ctx_hi = rng.choice((0, _log(rng, 10, 12000), _log(rng, 10, 12000)))
            if seqs * new_hi * (new_hi + ctx_hi) * heads[0] * heads[2] <= MOST_PAIRS and \
                    seqs * (new_hi + ctx_hi) * heads[1] * heads[2] <= 1 << 28:
                break
        case = attention("", seqs, (rng.randint(1, new_hi), new_hi), (rng.randint(0, ctx_hi), ctx_hi), heads, block,
                         rng.choice(("f32", "f16", "f16")), mix, rng.choice((0, 0, 0, _log(rng, 16, 4096))))
    elif kind == "logprobs":
        vocab = _log(rng, 1000, 128256)
        case = logprobs("", _log(rng, 1, min(1500, MOST_LOGITS // vocab)), vocab, rng.choice((0, 0, 1, 5, 20, 32)),
                        rng.random() < 0.25)
    else:
        case = norm("", _log(rng, 1, 4096), rng.choice(WIDTHS), rng.choice(("f32", "f16")), rng.random() < 0.7,
                    rng.choice(("none", "one", "row")), rng.random() < 0.85)
        if case["rows"] * case["n"] > 4096 * 4096:
            case["rows"] = 4096 * 4096 // case["n"]
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


def _rope_table(head_dim, rows):
    half = head_dim // 2
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * torch.exp(
        -2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / head_dim * math.log(ROPE_BASE))
    return torch.stack((torch.cos(angle), torch.sin(angle)), 2).float().contiguous()


def _q8_pages(blocks, kv_heads, block, head_dim, g, spread):
    """Pages as earlier steps left them: normal values whose size differs by group, as codes and scale bytes."""
    y = torch.randn(blocks, kv_heads, block // GROUP, GROUP, head_dim, device="cuda", generator=g)
    y *= torch.exp2(torch.rand(blocks, kv_heads, block // GROUP, 1, 1, device="cuda", generator=g) * spread)
    e = _exponent(y.abs().amax((3, 4)))
    codes = torch.round(y * torch.exp2(-e[..., None, None].float()))
    return codes.to(torch.int8).reshape(blocks, kv_heads, block, head_dim), (e + 127).to(torch.uint8)


def _append_inputs(case, seed):
    g = _gen(seed)
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    new, ctx = lengths(case)
    # the pages that the step writes to, anywhere in the cache; a sequence's are in no order
    held = [_pages(c + n, block) - c // block for n, c in zip(new, ctx)]
    blocks = sum(held) + 2
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed))).tolist()
    pos, slots, at = [], [], 0
    for n, c, pages in zip(new, ctx, held):
        pos += range(c, c + n)
        slots += [ids[at + p // block - c // block] * block + p % block for p in range(c, c + n)]
        at += pages
    pad = -len(pos) % 8  # the step's buffers are a whole number of eight rows
    tokens = len(pos) + pad
    k, k_scale = _q8_pages(blocks, nkv, block, hd, g, 2.0)
    v, v_scale = _q8_pages(blocks, nkv, block, hd, g, 2.0)
    x = torch.randn(tokens, (nq + 2 * nkv) * hd, device="cuda", generator=g) * 2.0
    return {"x": x.to(_type(case["x"])), "rope": _rope_table(hd, ROWS), "blocks": blocks, "tokens": tokens,
            "q_norm": 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=g),
            "k_norm": 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=g),
            "pos": _ints(pos + [0] * pad), "slots": _ints(slots + [-1] * pad),
            "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


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
    k, k_scale = _q8_pages(blocks, nkv, block, hd, g, 0.5)
    v, v_scale = _q8_pages(blocks, nkv, block, hd, g, 1.5)
    return {"q": (torch.randn(start[-1], nq * hd, device="cuda", generator=g) * 1.5).to(_type(case["x"])),
            "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "start": _ints(start),
            "kv_len": _ints([c + n for n, c in zip(new, ctx)]), "table": table, "tokens": start[-1],
            "blocks": blocks, "width": width, "most_new": max(new)}


def _logprobs_inputs(case, seed):
    g = _gen(seed)
    m, n = case["rows"], case["vocab"]
    logits = torch.randn(m, n, device="cuda", generator=g) * 3.0
    if case["rounded"]:  # a head that answers in few bits: equal logits
        logits = torch.round(logits * 16.0) / 16.0
    # half of the tokens are likely ones
    likely = logits.argmax(1)
    token = torch.randint(0, n, (m,), device="cuda", generator=g)
    token = torch.where(torch.rand(m, device="cuda", generator=g) < 0.5, likely, token)
    return {"logits": logits, "tokens": token.int()}


def _norm_inputs(case, seed):
    g = _gen(seed)
    m, n = case["rows"], case["n"]
    t = {"x": torch.randn(m, n, device="cuda", generator=g) * 3.0,
         "delta": torch.randn(m, n, device="cuda", generator=g) * 0.5,
         "post": 1.0 + 0.1 * torch.randn(n, device="cuda", generator=g),
         "pre": 1.0 + 0.1 * torch.randn(n, device="cuda", generator=g)}
    if case["gate"] != "none":
        t["gate"] = torch.tanh(torch.randn(m if case["gate"] == "row" else 1, n, device="cuda", generator=g))
    return t


SCALE = 0.22  # of the residual, where a norm case has one

_INPUTS = {"append": _append_inputs, "attention": _attention_inputs, "logprobs": _logprobs_inputs, "norm": _norm_inputs}


# ---------------------------------------------------------------- prepare ----

def prepare(case, seed):
    t = _INPUTS[case["kind"]](case, seed)
    out = {}
    if case["kind"] == "append":
        out = {"out": torch.empty(t["tokens"], case["q_heads"] * case["head_dim"], dtype=_type(case["q"]), device="cuda"),
               "k_values": torch.empty(t["k"].shape, dtype=torch.float16, device="cuda"),
               "v_values": torch.empty(t["v"].shape, dtype=torch.float16, device="cuda")}
    elif case["kind"] == "attention":
        out = {"out": torch.empty_like(t["q"])}
    elif case["kind"] == "logprobs":
        m, top = case["rows"], case["top"]
        out = {"logprob": torch.empty(m, device="cuda"), "entropy": torch.empty(m, device="cuda"),
               "top_tokens": torch.empty(m, top, dtype=torch.int32, device="cuda"),
               "top_logprobs": torch.empty(m, top, device="cuda")}
    else:
        out = {"x_out": torch.empty_like(t["x"]), "out": torch.empty(t["x"].shape, dtype=_type(case["out"]), device="cuda")}
    t.update(out)
    memory = {k: Memory(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
    return {"case": case, "t": t, "memory": memory}


# -------------------------------------------------------------- plain form ----

def _exponent(a):
    """The smallest e in LOW..HIGH at which a / 2^e rounds to a code (a < 127.5 * 2^e)."""
    m, e = torch.frexp(a.double())
    return torch.where(a > 0, torch.clamp(e - 7 + (m * 128.0 >= 127.5).int(), LOW, HIGH), LOW)


def _values(codes, scale):
    """Codes [blocks, heads, block, dims] with their scale bytes as values, fp32."""
    b, h, n, d = codes.shape
    s = torch.exp2(scale.float() - 127.0)
    return (codes.reshape(b, h, n // GROUP, GROUP, d).float() * s[..., None, None]).reshape(b, h, n, d)


def _store(codes, scale, y, slot, block):
    """Rows y [n, heads, dims] (64 bits: codes lie next to borders) into the pages at their slots."""
    blocks, nkv, _, hd = codes.shape
    groups = blocks * block // GROUP
    old = codes.reshape(blocks, nkv, block // GROUP, GROUP, hd).permute(0, 2, 1, 3, 4).reshape(groups, nkv, GROUP, hd)
    e_old = scale.reshape(blocks, nkv, block // GROUP).permute(0, 2, 1).reshape(groups, nkv).long() - 127
    at = slot // GROUP
    top = torch.zeros(groups, nkv, dtype=torch.float64, device="cuda")
    top.scatter_reduce_(0, at[:, None].expand(-1, nkv), y.abs().amax(2), "amax")
    rows = torch.zeros(groups, dtype=torch.bool, device="cuda")
    rows[at] = True
    fresh = torch.zeros(groups, dtype=torch.float64, device="cuda")
    fresh.scatter_reduce_(0, at, (slot % GROUP == 0).double(), "amax")
    anew = (fresh > 0)[:, None]
    e = _exponent(top).long()
    e = torch.where(rows[:, None], torch.where(anew, e, torch.maximum(e, e_old)), e_old)
    kept = torch.round(old.float() * torch.exp2((e_old - e).clamp(min=-40).float())[..., None, None])
    kept = torch.where(anew[..., None, None], torch.zeros_like(kept), kept)
    kept[at, :, slot % GROUP] = torch.round(y * torch.exp2(-e[at].double())[..., None]).float()
    new = kept.reshape(blocks, block // GROUP, nkv, GROUP, hd).permute(0, 2, 1, 3, 4).reshape(codes.shape)
    codes.copy_(new.to(torch.int8))
    scale.copy_((e + 127).reshape(blocks, block // GROUP, nkv).permute(0, 2, 1).to(torch.uint8))


def _plain_append(case, t):
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    half = hd // 2
    x = t["x"].double().reshape(t["tokens"], nq + 2 * nkv, hd)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    if case["norm"]:
        w = torch.cat((t["q_norm"].expand(nq, hd), t["k_norm"].expand(nkv, hd))).double()
        qk = qk / torch.sqrt((qk * qk).mean(2, keepdim=True) + EPS) * w
    cs = t["rope"][t["pos"].long()][:, None].double()
    cos, sin = cs[..., 0], cs[..., 1]
    a, b = qk[..., :half], qk[..., half:]
    qk = torch.cat((a * cos - b * sin, b * cos + a * sin), 2)
    real = t["slots"] >= 0
    slot = t["slots"][real].long()
    _store(t["k"], t["k_scale"], qk[real, nq:], slot, block)
    _store(t["v"], t["v_scale"], v[real], slot, block)
    return {"q": qk[:, :nq].reshape(t["tokens"], nq * hd).to(_type(case["q"])),
            "k": _values(t["k"], t["k_scale"]).half(), "v": _values(t["v"], t["v_scale"]).half()}


def _plain_attention(case, t):
    nq, nkv, hd, block, seqs = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "block", "seqs"))
    group, most = nq // nkv, t["most_new"]
    start, kv_len = t["start"].long(), t["kv_len"].long()
    new = start[1:] - start[:-1]
    # every sequence padded to the longest: its pages in order, its tokens from its first on
    page = t["table"].long().clamp(min=0).reshape(-1)

    def pages(codes, scale):
        y = _values(codes[page], scale[page]).reshape(seqs, -1, nkv, block, hd)
        return y.permute(0, 2, 1, 3, 4).reshape(seqs, nkv, -1, hd)

    keys, values = pages(t["k"], t["k_scale"]), pages(t["v"], t["v_scale"])
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


def _plain_logprobs(case, t):
    logits = t["logits"]
    largest = logits.amax(1, keepdim=True)
    d = (logits - largest).double()  # (a long sum)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"logprob": (torch.gather(d, 1, t["tokens"].long()[:, None]) - log_total)[:, 0].float(),
           "entropy": (log_total - (e * d).sum(1, keepdim=True) / total)[:, 0].float()}
    if case["top"]:
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_tokens"] = order.int()
        out["top_logprobs"] = (torch.gather(d, 1, order) - log_total).float()
    return out


def _plain_norm(case, t):
    d = t["delta"]
    if case["post"]:
        d = d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) * t["post"]
    if case["gate"] != "none":
        d = d * t["gate"]
    u = t["x"] + SCALE * d
    out = {"x": u}
    if case["pre"]:
        out["y"] = (u / torch.sqrt((u * u).mean(1, keepdim=True) + EPS) * t["pre"]).to(_type(case["out"]))
    return out


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs, "norm": _plain_norm}


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
        kind, size = case["kind"], 0
        if kind == "logprobs":
            size = rqmv.logprobs_workspace_size(case["rows"], case["vocab"], case["top"])
        elif kind in ("append", "attention"):
            shape = (t["blocks"], case["block"], case["kv_heads"], case["head_dim"])
            self.cache = rqmv.PagedCacheQ8(m["k"], m["v"], m["k_scale"], m["v_scale"], *shape)
            self.batch = rqmv.PagedBatch(case["seqs"], t["tokens"], t.get("width", 1), q_start=m.get("start"),
                                         kv_len=m.get("kv_len"), block_table=m.get("table"), positions=m.get("pos"),
                                         slots=m.get("slots"))
            if kind == "attention":
                size = rqmv.paged_attention_q8_workspace_size(self.batch, self.cache, case["q_heads"])
            else:
                self.values = rqmv.PagedCache(m["k_values"], m["v_values"], *shape)
        self.workspace = Memory(torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"))


def _run_own(s):
    rqmv = _library()
    case, t, m = s["case"], s["t"], s["memory"]
    if "kept" not in s:
        s["kept"] = _Kept(case, t, m)
    kept, kind = s["kept"], case["kind"]
    f = {"f32": rqmv.DTYPE_F32, "f16": rqmv.DTYPE_F16}
    if kind == "append":
        nq, nkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
        w = {"q_norm": m["q_norm"], "k_norm": m["k_norm"], "eps": EPS} if case["norm"] else {}
        rqmv.qk_norm_rope_q8(kept.batch, kept.cache, m["x"], f[case["x"]], (nq + 2 * nkv) * hd, nq, m["rope"], ROWS,
                             m["out"], f[case["q"]], nq * hd, **w)
        rqmv.paged_values_q8(kept.cache, kept.values)
        return {"q": t["out"], "k": t["k_values"], "v": t["v_values"]}
    if kind == "attention":
        row = case["q_heads"] * case["head_dim"]
        rqmv.paged_attention_q8(kept.batch, kept.cache, m["q"], f[case["x"]], row, case["q_heads"], m["out"], row,
                                kept.workspace, window=case["window"])
        return t["out"]
    if kind == "logprobs":
        n, top = case["vocab"], case["top"]
        more = {"top": top, "top_tokens": m["top_tokens"], "top_logprobs": m["top_logprobs"]} if top else {}
        rqmv.logprobs(m["logits"], case["rows"], n, n, tokens=m["tokens"], logprob=m["logprob"], entropy=m["entropy"],
                      workspace=kept.workspace, **more)
        return {k: t[k] for k in ("logprob", "entropy") + (("top_tokens", "top_logprobs") if top else ())}
    n, more = case["n"], {}
    if case["post"]:
        more["post_norm"] = m["post"]
    if case["gate"] != "none":
        more.update(gate=m["gate"], ldg=n if case["gate"] == "row" else 0)
    if case["pre"]:
        more.update(pre_norm=m["pre"], out=m["out"], out_dtype=f[case["out"]])
    rqmv.block_norm(m["x"], case["rows"], n, delta=m["delta"], scale=SCALE, eps=EPS, x_out=m["x_out"], **more)
    return {"x": t["x_out"], "y": t["out"]} if case["pre"] else {"x": t["x_out"]}


# -------------------------------------------------------------------- run ----

def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["kind"]](s["case"], s["t"])


# ------------------------------------------------------------------- work ----

def work(case):
    kind = case["kind"]
    size = {"f32": 4, "f16": 2}
    if kind == "logprobs":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 3 + 2 * case["top"]),
                "flops": 6.0 * case["rows"] * case["vocab"]}
    if kind == "norm":
        each = 12 + (size[case["out"]] if case["pre"] else 0) + (4 if case["gate"] == "row" else 0)
        return {"bytes": float(case["n"] * (case["rows"] * each + 12)), "flops": 9.0 * case["rows"] * case["n"]}
    new, ctx = lengths(case)
    nq, nkv, hd, block = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"]
    if kind == "append":
        tokens = (sum(new) + 7) // 8 * 8
        # the rows, their queries and codes; then every page read and its values written, at 1 and 2 bytes
        pages = sum(_pages(c + n, block) - c // block for n, c in zip(new, ctx)) + 2
        table = min(tokens, ROWS) * hd * 4
        return {"bytes": float(tokens * ((nq + 2 * nkv) * hd * size[case["x"]] + nq * hd * size[case["q"]] + 8) +
                               2 * sum(new) * nkv * hd + table + 2 * 3 * pages * block * nkv * hd),
                "flops": 7.0 * tokens * (nq + nkv) * hd + 2.0 * pages * block * nkv * hd}
    window = case["window"]
    pairs = keys = 0
    for n, c in zip(new, ctx):
        if window:
            pairs += sum(min(c + i + 1, window) for i in range(n))
            keys += min(c + n, n - 1 + window)
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    return {"bytes": float(keys * nkv * (2 * hd + 2 / GROUP) + 2 * sum(new) * nq * hd * size[case["x"]]),
            "flops": 4.0 * pairs * nq * hd}


# ------------------------------------------------------------------ exact ----

def _exact_append(case, t):
    nq, nkv, hd, block, tokens = case["q_heads"], case["kv_heads"], case["head_dim"], case["block"], t["tokens"]
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
    out = {"q": heads[:, :nq].reshape(tokens, -1)}
    # the pages on the host, a group of rows at a time, from the definition
    slots = t["slots"].tolist()
    runs, last = {}, [s for s in slots if s >= 0]
    for row, s in enumerate(slots):
        if s >= 0:
            runs.setdefault(s // GROUP, []).append(row)
    assert len(set(last)) == len(last)
    for name, y in (("k", heads[:, nq:]), ("v", x[:, nq + nkv:])):
        y = y.cpu()
        codes, scale = t[name].cpu(), t[name + "_scale"].cpu()
        values = codes.double() * torch.exp2(scale.double() - 127.0).repeat_interleave(GROUP, 2)[..., None]
        for group, rows in runs.items():
            b, first = group * GROUP // block, group * GROUP % block
            offs = [slots[r] % block for r in rows]
            new = y[rows].transpose(0, 1)  # heads, rows, dims
            step = torch.exp2(torch.full((nkv,), float(LOW), dtype=torch.float64))
            if first not in offs:
                step = torch.maximum(step, torch.exp2(scale[b, :, first // GROUP].double() - 127.0))
            top = new.abs().amax((1, 2))
            for _ in range(HIGH - LOW):
                step = torch.where((top >= 127.5 * step) & (step < 2.0 ** HIGH), step * 2.0, step)
            step = step[:, None, None]
            kept = values[b, :, first:first + GROUP]
            kept = torch.round(kept / step) * step if first not in offs else torch.zeros_like(kept)
            values[b, :, first:first + GROUP] = kept
            values[b, :, offs] = torch.round(new / step) * step
        out[name] = values.cuda()
    return out


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

        def head(name, h):
            step = torch.exp2(t[name + "_scale"][pages, h].double() - 127.0)
            return (t[name][pages, h].double() * step.repeat_interleave(GROUP, 1)[..., None]).reshape(-1, hd)[:c + n]

        rows = torch.empty(n, nq, hd, dtype=torch.float64, device="cuda")
        for h in range(nq):
            k, v = head("k", h // (nq // nkv)), head("v", h // (nq // nkv))
            q = t["q"][at:at + n, h * hd:(h + 1) * hd].double()
            s = (q @ k.t().contiguous() * hd ** -0.5).masked_fill_(hidden, -math.inf)
            rows[:, h] = torch.softmax(s, 1) @ v
        out.append(rows.reshape(n, nq * hd))
        at += n
    return torch.cat(out)


def _exact_logprobs(case, t):
    logprob, entropy, tops = [], [], []
    for i in range(case["rows"]):
        x = t["logits"][i].double()
        lp = torch.log_softmax(x, 0)
        logprob.append(lp[t["tokens"][i].long()])
        entropy.append(-(lp.exp() * lp).sum())
        if case["top"]:
            tops.append(torch.topk(lp, case["top"]).values)
    out = {"logprob": torch.stack(logprob), "entropy": torch.stack(entropy)}
    if case["top"]:
        out.update(top_tokens=None, top_logprobs=torch.stack(tops))
    return out


def _exact_norm(case, t):
    d, u = t["delta"].double(), t["x"].double()
    if case["post"]:
        d = t["post"].double() * d * (d.square().sum(1, keepdim=True) / case["n"] + EPS).rsqrt()
    gate = t["gate"].double() if case["gate"] != "none" else 1.0
    u = u + d * gate * SCALE
    out = {"x": u}
    if case["pre"]:
        out["y"] = t["pre"].double() * u * (u.square().sum(1, keepdim=True) / case["n"] + EPS).rsqrt()
    return out


def exact(case, seed):
    t = _INPUTS[case["kind"]](case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs,
            "norm": _exact_norm}[case["kind"]](case, t)
