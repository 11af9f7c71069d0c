"""f64 references of the paged serving operators (include/rqmv.h), on the host.

Written from the definitions, one sequence, head or row at a time: plan() the
step's tables, qk_norm_rope() the norms, rotation and append, attention() a
sequence's new tokens over its pages, sample() the next token; store_q8() the append to
8-bit pages and values_q8() what they stand for, logprobs() what a token is reported
with, block_norm() the norms between two blocks.
"""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np


def pages(n: int, block: int) -> int:
    return -(-n // block)


def plan(cached, new, table, free_list, head, block, blocks, tokens):
    """(status, q_start, kv_len, table, positions, slots, head) of rqmv_paged_plan."""
    seqs, width = table.shape
    table = table.copy()
    status = 0
    if any(c < 0 or n < 0 or c + n > width * block for c, n in zip(cached, new)):
        status |= 1
    fits = [(c, n) for c, n in zip(cached, new) if c >= 0 and n >= 0 and c + n <= width * block]
    if sum(n for _, n in fits) > tokens:
        status |= 2
    if not 0 <= head <= len(free_list) or sum(pages(c + n, block) - pages(c, block) for c, n in fits) > \
            len(free_list) - head:
        status |= 4
    positions, slots = np.zeros(tokens, np.int32), np.full(tokens, -1, np.int32)
    q_start = np.zeros(seqs + 1, np.int32)
    kv_len = np.array(cached, np.int32)
    if status:
        return status, q_start, kv_len, table, positions, slots, head
    row = 0
    for s in range(seqs):
        for page in range(pages(cached[s], block), pages(cached[s] + new[s], block)):
            table[s, page] = free_list[head]
            head += 1
        for p in range(cached[s], cached[s] + new[s]):
            positions[row] = p
            b = int(table[s, p // block])
            slots[row] = b * block + p % block if 0 <= b < blocks else -1
            row += 1
        q_start[s + 1] = row
        kv_len[s] = cached[s] + new[s]
    return 0, q_start, kv_len, table, positions, slots, head


def qk_norm_rope(x, nq, nkv, hd, q_norm, k_norm, eps, table, rot, positions):
    """(q [tokens, nq, hd], k, v [tokens, nkv, hd]) in 64 bits; table is [rows, rot / 2, 2]."""
    x = np.asarray(x, np.float64).reshape(len(positions), nq + 2 * nkv, hd).copy()
    pos = np.clip(positions, 0, len(table) - 1)
    cos, sin = (np.asarray(table, np.float64)[pos][:, None, :, i] for i in (0, 1))

    def turn(h, w):
        if w is not None:
            h = h / np.sqrt((h ** 2).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
        out = h.copy()
        a, b = h[..., :rot // 2], h[..., rot // 2:rot]
        out[..., :rot // 2] = a * cos - b * sin
        out[..., rot // 2:rot] = b * cos + a * sin
        return out

    return turn(x[:, :nq], q_norm), turn(x[:, nq:nq + nkv], k_norm), x[:, nq + nkv:]


def attention(q, k, v, q_start, kv_len, table, max_blocks, scale, window=0):
    """[rows of q, nq, hd] in 64 bits; rows of no sequence stay NaN. k, v are
    [blocks, nkv, block, hd]."""
    blocks, nkv, block, hd = k.shape
    nq = q.shape[1]
    out = np.full((q.shape[0], nq, hd), np.nan)
    for s in range(len(kv_len)):
        n, kv = int(q_start[s + 1] - q_start[s]), int(kv_len[s])
        keep = [p for p in range(min(kv, max_blocks * block)) if 0 <= table[s, p // block] < blocks]
        at = np.array(keep, np.int64)
        if len(keep):
            b = table[s, at // block]
            keys, values = (c[b, :, at % block].astype(np.float64) for c in (k, v))  # [keys, nkv, hd]
        for i in range(n):
            row, pos = int(q_start[s]) + i, kv - n + i
            live = (at <= pos) & ((at > pos - window) if window else True) if len(keep) else np.zeros(0, bool)
            if not live.any():
                out[row] = 0.0
                continue
            for g in range(nkv):
                h = slice(g * (nq // nkv), (g + 1) * (nq // nkv))
                sc = q[row, h].astype(np.float64) @ keys[live, g].T * scale  # [the group's heads, keys]
                with np.errstate(invalid="ignore"):
                    e = np.exp(sc - sc.max(-1, keepdims=True))
                    out[row, h] = (e / e.sum(-1, keepdims=True)) @ values[live, g]
    return out


def values_q8(codes, scale):
    """[blocks, nkv, block, hd] in 64 bits; scale bytes are [blocks, nkv, block / 16]."""
    b = np.clip(scale.astype(np.int64), 103, 136)
    s = np.where(scale == 255, np.nan, 2.0 ** (b - 127.0))
    return codes.astype(np.float64) * np.repeat(s, 16, axis=2)[..., None]


def exponent_q8(a):
    """The smallest e of -24..9 with a < 127.5 * 2^e; None: there is none."""
    return next((e for e in range(-24, 10) if a < 127.5 * 2.0 ** e), None)


def store_q8(codes, scale, y, slots):
    """(codes, scale) with rows y [tokens, nkv, hd] (64 bits) stored at their slots; -1 and slots past the cache: none."""
    codes, scale = codes.copy(), scale.copy()
    blocks, nkv, block, hd = codes.shape
    groups = {}
    for t, s in enumerate(slots):
        if 0 <= s < blocks * block:
            groups.setdefault(int(s) // 16, []).append(t)
    for g, rows in groups.items():
        b, first = g * 16 // block, g * 16 % block
        at = [int(slots[t]) % block for t in rows]
        for h in range(nkv):
            new = np.asarray([y[t][h] for t in rows], np.float64)
            old = scale[b, h, first // 16]
            e = None if np.isnan(new).any() else exponent_q8(np.abs(new).max())
            part = codes[b, h, first:first + 16]
            if first in at:
                part[:] = 0
                scale[b, h, first // 16] = 255 if e is None else e + 127
            else:
                e_old = int(np.clip(int(old) - 127, -24, 9))
                e = e if e is None else max(e, e_old)
                if e is not None:
                    part[:] = np.rint(part * 2.0 ** (e_old - e))
                scale[b, h, first // 16] = 255 if e is None or old == 255 else e + 127
            if e is not None:
                codes[b, h, at] = np.rint(new * 2.0 ** -e)
    return codes, scale


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, its probability among the kept ones) of one row."""
    logits = np.asarray(logits, np.float32)
    order = [int(i) for i in np.argsort(-np.where(np.isnan(logits), -np.inf, logits).astype(np.float64), kind="stable")
             if logits[i] > -np.inf]
    if not order:
        return -1, 0.0
    if not temperature > 0:
        return order[0], 1.0
    if 0 < top_k < len(order):
        order = order[:top_k]
    best = float(logits[order[0]])
    e = [1.0 if float(logits[i]) == best else math.exp((float(logits[i]) - best) / float(temperature)) for i in order]
    if 0.0 <= top_p < 1.0:
        target, total, n = Fraction(float(top_p)) * Fraction(math.fsum(e)), Fraction(0), 0
        while n < len(e) and (n == 0 or total < target):
            total += Fraction(e[n])
            n += 1
        e = e[:n]
    if min_p > 0:
        e = [w for w in e if w >= min(float(min_p), 1.0)]
    total = math.fsum(e)
    target, end = (float(u) if u > 0 else 0.0) * total, Fraction(0)
    for i, w in enumerate(e):
        end += Fraction(w)
        if end > target:
            return order[i], w / total
    last = max(i for i, w in enumerate(e) if w > 0)
    return order[last], e[last] / total


def logprobs(logits, token=None, top=0):
    """(log p(token), entropy, top tokens, their log probabilities) of one row."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    none = np.full(len(x), -np.inf)
    if not (x > -np.inf).any():
        lp, entropy = none, 0.0
    else:
        d = np.where(x == np.inf, 0.0, -np.inf) if x.max() == np.inf else x - x.max()
        lp = d - math.log(math.fsum(np.exp(d)))
        p = np.exp(lp)
        entropy = -math.fsum(p[p > 0] * lp[p > 0])
    order = [int(i) for i in np.argsort(-x, kind="stable")[:top] if x[i] > -np.inf]
    best = [float(lp[i]) for i in order] + [-math.inf] * (top - len(order))
    given = None if token is None else float(lp[token]) if 0 <= token < len(x) else -math.inf
    return given, entropy, order + [-1] * (top - len(order)), best


def block_norm(x, delta=None, post=None, gate=None, scale=1.0, pre=None, eps=0.0):
    """(u, out) of rows [rows, n] in 64 bits; out is None without `pre`."""
    u = np.asarray(x, np.float64)
    if delta is not None:
        d = np.asarray(delta, np.float64)
        if post is not None:
            d = d / np.sqrt((d ** 2).mean(-1, keepdims=True) + eps) * np.asarray(post, np.float64)
        u = u + scale * (1.0 if gate is None else np.asarray(gate, np.float64)) * d
    return u, None if pre is None else u / np.sqrt((u ** 2).mean(-1, keepdims=True) + eps) * np.asarray(pre, np.float64)
