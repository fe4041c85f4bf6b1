"""What is measured of the operators of a serving step: the cache's write and its reading back, attention of a
few new tokens over it, and the log probabilities of given tokens.

``store``: rotary positions, and the write of keys and values into pages, in bfloat16 or in e4m3 with one power of
two a vector; the pages that were written are read back as bfloat16, as prompt attention takes them.  ``read``: reading
back alone.  ``attention``: one token a request (decoding), a chain of a few, or a tree of drafted ones, over pages of
either type.  ``logprobs``: log probability, rank and entropy of given tokens, with the best alternatives.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
E4M3 = torch.float8_e4m3fn
LOWEST, HIGHEST = -60, 119       # exponents of a vector's power of two
BIAS = 127


# ---- the cases ---------------------------------------------------------------------------------------

def _store(name, cache, requests, tokens, behind, heads, kv_heads, dim, parts, pairing="half"):
    return {"name": name, "op": "store", "cache": cache, "requests": requests, "tokens": tokens, "behind": behind, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "parts": parts, "pairing": pairing}


def _read(name, pages, kv_heads, dim):
    return {"name": name, "op": "read", "pages": pages, "kv_heads": kv_heads, "dim": dim}


def _attention(name, cache, requests, tokens, behind, heads, kv_heads, dim, tree, ragged, window=0):
    return {"name": name, "op": "attention", "cache": cache, "requests": requests, "tokens": tokens, "behind": behind, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "tree": tree, "ragged": ragged, "window": window}


def _logprobs(name, rows, vocab, top):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top}


def listed():
    return [
        # a decode step of eight requests writes its tokens to an 8-bit cache; the projection comes in partial sums
        _store("store_e4m3_decode_b8", "e4m3", 8, 1, 2047, 32, 8, 128, 4),
        # a prompt's portion into an 8-bit cache, and back for prompt attention
        _store("store_e4m3_prompt", "e4m3", 1, 2048, 0, 32, 8, 128, 0),
        # drafted tokens of four requests into a bfloat16 cache
        _store("store_bf16_drafts", "bf16", 4, 31, 1000, 32, 8, 64, 0, "adjacent"),
        # one short context for a portion's attention
        _read("read_short", 34, 8, 128),
        # contexts of a turn of many prompts
        _read("read_long", 1531, 8, 128),
        # one request decodes behind a short conversation: latency
        _attention("decode_e4m3_b1", "e4m3", 1, 1, 1000, 32, 8, 128, False, False),
        # the benchmark's own decode workload over an 8-bit cache
        _attention("decode_e4m3_b8", "e4m3", 8, 1, 2175, 32, 8, 128, False, False),
        # a busy server, contexts of many lengths
        _attention("decode_e4m3_b64", "e4m3", 64, 1, 4096, 32, 8, 128, False, True),
        # a draft tree is checked for one request, over the bfloat16 cache
        _attention("tree_bf16_b1", "bf16", 1, 27, 2176, 32, 8, 128, True, False),
        # larger trees of several requests over the 8-bit cache
        _attention("tree_e4m3_b4", "e4m3", 4, 64, 8192, 32, 8, 128, True, True),
        # the log probabilities of eight decoded tokens with five alternatives
        _logprobs("logprobs_b8", 8, 128256, 5),
        # a prompt's tokens are scored
        _logprobs("logprobs_prompt", 1021, 128256, 20),
    ]


SHAPES = [(32, 8, 128), (40, 40, 128), (32, 8, 64), (16, 4, 128), (16, 16, 64), (16, 2, 128), (8, 2, 32), (6, 2, 32), (16, 4, 80)]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    op = rng.choice(["store", "store", "read", "attention", "attention", "attention", "attention", "logprobs", "logprobs"])
    heads, kv_heads, dim = rng.choice(SHAPES)
    cache = rng.choice(["e4m3", "e4m3", "bf16"])
    if op == "store":
        few = rng.random() < 0.5
        requests, tokens = (_log(rng, 1, 64), _log(rng, 1, 16)) if few else (_log(rng, 1, 4), _log(rng, 17, 600))
        case = _store("", cache, requests, tokens, _log(rng, 1, 20000) - 1, heads, kv_heads, dim, rng.choice([0, 2, 3, 7]) if few else 0,
                      rng.choice(["half", "adjacent"]))
    elif op == "read":
        case = _read("", _log(rng, 1, min(4000, 1531 * 8 * 128 // (kv_heads * dim))), kv_heads, dim)
    elif op == "attention":
        tokens = rng.choice([1, 1, 2, 5, _log(rng, 3, 64), 64])
        requests = _log(rng, 1, 40)
        most = (64 * 4096 * 8 * 128) // (requests * kv_heads * dim) // (2 if cache == "bf16" else 1)
        most = max(64, min(30000, most, (1 << 27) // (requests * tokens * heads)))
        behind = _log(rng, 1, most) - 1
        case = _attention("", cache, requests, tokens, behind, heads, kv_heads, dim, tokens > 2 and rng.random() < 0.7, rng.random() < 0.5,
                          rng.choice([0, 0, 0, max(behind // 2, 1)]))
    else:
        vocab = rng.choice([320, 32000, 50257, 128256])
        case = _logprobs("", _log(rng, 1, max(1, min(2000, 1021 * 128256 // vocab))), vocab, rng.choice([1, 2, 5, 20, 32]))
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------

def _codes(x):
    """float32 vectors (last axis) as e4m3 codes and the exponent byte of every vector."""
    amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    e = _exponent(amax)
    codes = x * _power(-e)[..., None]
    codes = torch.where(torch.isfinite(codes), codes, torch.full_like(codes, math.nan)).to(E4M3)
    return codes, (e + BIAS).to(torch.uint8)


def _exponent(amax):
    """ceil(log2(amax / 448)) without a logarithm: 448 is 0.875 x 2^9."""
    fraction, exponent = torch.frexp(amax)
    e = torch.where(fraction <= 0.875, exponent - 9, exponent - 8)
    return torch.where(amax > 0, e, torch.full_like(e, LOWEST)).clamp(LOWEST, HIGHEST)


def _power(e):
    """2^e exactly (a power function may be a bit off, and would move values that lie halfway between two codes)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _tables(gen, contexts):
    """Block tables of requests that took their pages in any order: int32 [requests, width], and how many pages there are."""
    blocks = [-(-c // PAGE) for c in contexts]
    order = torch.randperm(sum(blocks), generator=gen, device=DEVICE).to(torch.int32).split(blocks)
    return torch.nn.utils.rnn.pad_sequence(list(order), batch_first=True, padding_value=-1).contiguous(), sum(blocks)


def _pool(gen, pages, kv_heads, dim, cache):
    """Keys (their channels of different sizes, as rotated keys have them) and values of a pool of pages."""
    spread = torch.exp(0.7 * torch.randn(kv_heads, 1, dim, generator=gen, device=DEVICE))
    sides = (torch.randn(pages, kv_heads, PAGE, dim, generator=gen, device=DEVICE).mul_(spread), torch.randn(pages, kv_heads, PAGE, dim, generator=gen, device=DEVICE))
    if cache == "bf16":
        return [sides[0].to(torch.bfloat16), sides[1].to(torch.bfloat16), None, None]
    (k, ke), (v, ve) = _codes(sides[0]), _codes(sides[1])
    return [k, v, ke, ve]


def _frequencies(dim):
    exact = torch.tensor([500000.0 ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    high = exact.float()
    return torch.stack([high, (exact - high.double()).float()]).to(DEVICE)


def _family(rng, n, tree):
    """Parents of n drafted tokens (-1: none), every token after its parent."""
    return [(rng.randrange(max(-1, i - 9), i) if tree else i - 1) for i in range(n)]


def _new_tokens(case, seed):
    """Every request's new tokens: how many, where they stand, and what each sees of the others."""
    S, n = case["requests"], case["tokens"]
    rng, ragged = random.Random(S + n), case.get("ragged", False)              # (the sizes are the case's, the trees the seed's)
    lens = [max(1, n - rng.randrange(n // 3 + 1)) if ragged else n for _ in range(S)]
    pos0 = [max(0, case["behind"] - rng.randrange(case["behind"] // 2 + 1)) if ragged else case["behind"] for _ in range(S)]
    rng = random.Random(seed * 7919 + 11)
    positions, visible = [], []
    for s in range(S):
        depth, mask = [], []
        for i, p in enumerate(_family(rng, lens[s], case.get("tree", False))):
            depth.append(0 if p < 0 else depth[p] + 1)
            mask.append((0 if p < 0 else mask[p]) | 1 << i)
            positions.append(pos0[s] + depth[i])
            visible.append(mask[i] - (1 << 64) if mask[i] >> 63 else mask[i])
    return lens, pos0, positions, visible


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    st = {"op": case["op"], "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn(rows, vocab, generator=gen, device=DEVICE).mul_(2.5)
        # a model is often sure: a few ids stand out, and the given token is mostly one of them
        best = torch.randint(0, vocab, (rows, 4), generator=gen, device=DEVICE)
        logits.scatter_add_(1, best, 12.0 * torch.rand(rows, 4, generator=gen, device=DEVICE))
        other = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
        ids = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < 0.7, best[:, 0], other).to(torch.int32)
        return {**st, "logits": logits, "ids": ids, "top": case["top"]}
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "read":
        pool = _pool(gen, case["pages"] + 7, kv_heads, dim, "e4m3")
        return {**st, "pool": pool, "pages": torch.randperm(case["pages"] + 7, generator=gen, device=DEVICE)[:case["pages"]].to(torch.int32).contiguous()}
    heads = case["heads"]
    lens, pos0, positions, visible = _new_tokens(case, seed)
    N = sum(lens)
    table, pages = _tables(gen, [p + n for p, n in zip(pos0, lens)])
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    st.update(heads=heads, kv_heads=kv_heads, dim=dim, table=table, positions=ints(positions), seq_start=ints(start), seq_pos0=ints(pos0),
              seq_of_token=ints([s for s, n in enumerate(lens) for _ in range(n)]))
    if case["op"] == "store":
        width = (heads + 2 * kv_heads) * dim
        cells = ints([p + i for p, n in zip(pos0, lens) for i in range(n)])
        taken = table.long()[st["seq_of_token"].long(), torch.div(cells.long(), PAGE, rounding_mode="floor")]
        qkv = torch.randn(N, width, generator=gen, device=DEVICE) * torch.exp(0.5 * torch.randn(width, generator=gen, device=DEVICE))
        if case["parts"]:
            rest = torch.randn(case["parts"] - 1, N, width, generator=gen, device=DEVICE)
            qkv = torch.cat([(qkv - rest.sum(0))[None], rest]).contiguous()
        else:
            qkv = qkv.to(torch.bfloat16)
        shape = (pages, kv_heads, PAGE, dim)
        pool = [torch.zeros(shape, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)] + [None, None] if case["cache"] == "bf16" else \
            [torch.zeros(shape, dtype=torch.uint8, device=DEVICE).view(E4M3) for _ in range(2)] + [torch.zeros(shape[:3], dtype=torch.uint8, device=DEVICE) for _ in range(2)]
        return {**st, "qkv": qkv, "parts": case["parts"], "pool": pool, "cells": cells, "freq": _frequencies(dim), "pairing": case["pairing"],
                "pages": torch.unique(taken).to(torch.int32).contiguous()}
    return {**st, "q": torch.randn(N, heads * dim, generator=gen, device=DEVICE).to(torch.bfloat16), "pool": _pool(gen, pages, kv_heads, dim, case["cache"]),
            "visible": torch.tensor(visible, dtype=torch.int64, device=DEVICE) if case["tree"] else None, "window": case["window"],
            "most": max(lens), "longest": max(p + n for p, n in zip(pos0, lens)), "scale": 1.0 / math.sqrt(dim)}


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    return RUN[state["op"]](state)


def _run_store(st):
    k, v, ke, ve = st["pool"]
    H, G, D = st["heads"], st["kv_heads"], st["dim"]
    if own:
        from lgml_b200 import ops
        qkv = ops.Partials(st["qkv"]) if st["parts"] else st["qkv"]
        q = torch.empty((st["cells"].numel(), H * D), dtype=torch.bfloat16, device=DEVICE)
        ops.rope_kv_store(qkv, st["positions"], st["seq_of_token"], st["table"], st["freq"], D, st["pairing"], k, v, H, G, D, st["status"],
                          cells=st["cells"], k_exps=ke, v_exps=ve, q_out=q)
        return (q, k, v) if ke is None else (q, *ops.kv_read(k, v, ke, ve, st["pages"], st["status"]))
    x = (st["qkv"].double().sum(0) if st["parts"] else st["qkv"].double()).view(-1, H + 2 * G, D)
    angle = st["positions"].double()[:, None, None] * st["freq"].double().sum(0)
    c, s = torch.cos(angle), torch.sin(angle)
    turned = x[:, :H + G]
    if st["pairing"] == "half":
        a, b = turned[..., :D // 2], turned[..., D // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    q = turned[:, :H].reshape(-1, H * D).to(torch.bfloat16)
    cells = st["cells"].long()
    page = st["table"].long()[st["seq_of_token"].long(), torch.div(cells, PAGE, rounding_mode="floor")]
    keys, values = turned[:, H:].float(), x[:, H + G:].float()
    if ke is None:
        k[page, :, cells % PAGE] = keys.to(torch.bfloat16)
        v[page, :, cells % PAGE] = values.to(torch.bfloat16)
        return q, k, v
    _write(k, ke, page, cells % PAGE, keys)
    _write(v, ve, page, cells % PAGE, values)
    return q, _values(k, ke, st["pages"]), _values(v, ve, st["pages"])


def _write(pages, exps, page, cell, x):
    codes, e = _codes(x)
    pages.view(torch.uint8)[page, :, cell] = codes.view(torch.uint8)
    exps[page, :, cell] = e


def _values(pages, exps, which):
    which = which.long()
    values = pages.view(torch.uint8)[which].view(E4M3).float()
    return (values * _power(exps[which].int() - BIAS)[..., None]).to(torch.bfloat16)


def _run_read(st):
    k, v, ke, ve = st["pool"]
    if own:
        from lgml_b200 import ops
        return ops.kv_read(k, v, ke, ve, st["pages"], st["status"])
    return _values(k, ke, st["pages"]), _values(v, ve, st["pages"])


def _run_attention(st):
    k, v, ke, ve = st["pool"]
    H, G, D = st["heads"], st["kv_heads"], st["dim"]
    if own:
        from lgml_b200 import ops
        out = torch.empty_like(st["q"])
        return ops.tree_attention(st["q"], st["positions"], st["seq_start"], st["seq_pos0"], st["table"], k, v, out, H, st["scale"], st["window"],
                                  st["status"], max_new_tokens=st["most"], max_kv_len=st["longest"], k_exps=ke, v_exps=ve, visible=st["visible"])
    S, T, dev = st["table"].shape[0], st["most"], DEVICE
    start, pos0, positions = st["seq_start"].long(), st["seq_pos0"].long(), st["positions"].long()
    count = start[1:] - start[:-1]
    place = torch.arange(T, device=dev)
    row = (start[:-1, None] + place).clamp(max=positions.numel() - 1)                              # [S, T] rows of the new tokens (and some others')
    table = st["table"].long().clamp(min=0)
    keys, vals = _context(k, ke, table), _context(v, ve, table)                                    # [S, C, G, D]
    C = keys.shape[1]
    cell = torch.arange(C, device=dev)
    node = cell - pos0[:, None]                                                                    # [S, C] which new token a cell holds
    where = torch.where(node < 0, cell, positions[(start[:-1, None] + node.clamp(min=0)).clamp(max=positions.numel() - 1)])
    at = positions[row]
    bits = st["visible"][row] if st["visible"] is not None else None
    new = node[:, None, :]
    if bits is None:
        seen = (new <= place[:, None])
    else:
        seen = (bits[:, :, None] >> new.clamp(0, 63) & 1).bool() & (new < 64) | (new < 0)
    seen = seen & (new < count[:, None, None]) & (place[None, :, None] < count[:, None, None])
    if st["window"]:
        seen = seen & (where[:, None, :] > at[:, :, None] - st["window"])
    q = st["q"][row].float().view(S, T, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(S, G, T * (H // G), D)
    score = (q @ keys.permute(0, 2, 3, 1)) * st["scale"]                                           # [S, G, T x group, C]
    seen = seen.repeat_interleave(H // G, 1)[:, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = (p @ vals.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(S, G, T, H // G, D).permute(0, 2, 1, 3, 4).reshape(S, T, H * D)
    return o[place < count[:, None]].to(torch.bfloat16)


def _context(pages, exps, table):
    """Every request's cells in order, float32 [requests, cells, KV heads, dim]."""
    if exps is None:
        x = pages[table].float()
    else:
        x = pages.view(torch.uint8)[table].view(E4M3).float() * _power(exps[table].int() - BIAS)[..., None]
    return x.transpose(2, 3).flatten(1, 2)


def _run_logprobs(st):
    x, ids, top = st["logits"], st["ids"], st["top"]
    if own:
        from lgml_b200 import ops
        return tuple(ops.token_logprobs(x, ids, top, st["status"]))
    most = x.amax(-1, keepdim=True)
    w = torch.exp(x - most)
    total = w.sum(-1, keepdim=True)
    log_z = most + torch.log(total)
    given = x.gather(1, ids.long()[:, None])
    before = torch.arange(x.shape[1], device=x.device) < ids[:, None]
    rank = ((x > given) | ((x == given) & before)).sum(-1, dtype=torch.int32)
    entropy = log_z - (w * torch.where(w > 0, x, torch.zeros_like(x))).sum(-1, keepdim=True) / total
    values, best = torch.sort(x, dim=-1, descending=True, stable=True)
    return (given - log_z)[:, 0], rank, entropy[:, 0], best[:, :top].to(torch.int32), values[:, :top] - log_z


RUN = {"store": _run_store, "read": _run_read, "attention": _run_attention, "logprobs": _run_logprobs}


# ---- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    G, D = case["kv_heads"], case["dim"]
    if case["op"] == "read":
        cells = case["pages"] * G * PAGE
        return {"bytes": 2 * cells * (3 * D + 1), "flops": 2 * cells * D}
    H, n = case["heads"], case["requests"] * case["tokens"]
    cell = 4 * D if case["cache"] == "bf16" else 2 * D + 2           # bytes of a key and a value
    if case["op"] == "store":
        entry = 4 * case["parts"] if case["parts"] else 2
        total = n * ((H + 2 * G) * D * entry + 2 * H * D + G * cell)
        if case["cache"] != "bf16":                                 # the pages that were written, read back
            at = case["behind"] // PAGE
            pages = case["requests"] * ((case["behind"] + case["tokens"] - 1) // PAGE - at + 1)
            total += 2 * pages * G * PAGE * (3 * D + 1)
        return {"bytes": total, "flops": n * (H + 2 * G) * D * max(3, case["parts"])}
    lens, pos0, _, _ = _new_tokens(case, 0)
    reach = case["window"] or 1 << 30
    cells = sum(min(p + m, reach + m) for p, m in zip(pos0, lens))
    pairs = sum(m * min(p + m / 2, reach) for p, m in zip(pos0, lens))
    return {"bytes": int(cells * G * cell + 4 * sum(lens) * H * D), "flops": int(4 * pairs * H * D)}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------

def _two_to(n):
    """2^n of whole numbers in 64 bits, exactly."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        x = st["logits"].double()
        p = torch.softmax(x, -1)
        logs = torch.log_softmax(x, -1)
        ids = st["ids"].long()
        rows = torch.arange(x.shape[0], device=DEVICE)
        order = torch.argsort(x, dim=-1, descending=True, stable=True)
        rank = (order == ids[:, None]).int().argmax(-1).to(torch.int32)
        best = order[:, :case["top"]]
        return logs[rows, ids], rank, -(p * logs).sum(-1), best.to(torch.int32), logs.gather(1, best)
    if case["op"] == "read":
        k, v, ke, ve = st["pool"]
        pick = st["pages"].long()
        return tuple(a.float()[pick].double() * _two_to(e[pick].long() - 127).unsqueeze(-1) for a, e in ((k, ke), (v, ve)))
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "store":
        x = st["qkv"].double()
        if case["parts"]:
            x = x.sum(0)
        x = x.reshape(x.shape[0], H + 2 * G, D)
        frequency = torch.tensor([500000.0 ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device=DEVICE)
        turn = torch.polar(torch.ones(x.shape[0], D // 2, dtype=torch.float64, device=DEVICE), st["positions"].double().outer(frequency))[:, None]
        if case["pairing"] == "half":
            z = torch.complex(x[:, :H + G, :D // 2].contiguous(), x[:, :H + G, D // 2:].contiguous()) * turn
            z = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_real(torch.view_as_complex(x[:, :H + G].reshape(x.shape[0], H + G, D // 2, 2).contiguous()) * turn).reshape(x.shape[0], H + G, D)
        pools = []
        owner, cells = st["seq_of_token"].long(), st["cells"].long()
        page = st["table"][owner, cells // PAGE].long()
        for side in (z[:, H:], x[:, H + G:]):
            pool = torch.zeros(st["pool"][0].shape, dtype=torch.float64, device=DEVICE)
            if case["cache"] != "bf16":
                largest = side.abs().amax(-1, keepdim=True)
                step = _two_to(torch.ceil(torch.log2(largest / 448.0)).clamp(LOWEST, HIGHEST))
                unit = side / step
                # e4m3: four significant bits, the smallest of them 2^-9
                grid = _two_to(torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6))) - 3.0)
                side = torch.round(unit / grid) * grid * step
            pool[page, :, cells % PAGE] = side
            pools.append(pool if case["cache"] == "bf16" else pool[st["pages"].long()])
        return z[:, :H].reshape(-1, H * D), *pools
    k, v, ke, ve = st["pool"]
    lens, pos0, positions, visible = _new_tokens(case, seed)
    outs, row = [], 0
    for s, n in enumerate(lens):
        c = pos0[s] + n
        blocks = st["table"][s, :-(-c // PAGE)].long()
        sides = []
        for a, e in ((k, ke), (v, ve)):
            side = (a.view(torch.uint8)[blocks].view(E4M3).float() if e is not None else a[blocks].float()).double()
            side = side if e is None else side * _two_to(e[blocks].long() - 127).unsqueeze(-1)
            sides.append(side.permute(1, 0, 2, 3).reshape(G, -1, D)[:, :c])
        at = torch.tensor(positions[row:row + n], device=DEVICE)
        sees = torch.ones(n, c, dtype=torch.bool, device=DEVICE)
        sees[:, pos0[s]:] = torch.tensor([[(visible[row + i] >> j & 1 if case["tree"] else j <= i) == 1 for j in range(n)] for i in range(n)], device=DEVICE)
        if case["window"]:
            place = torch.cat([torch.arange(pos0[s], device=DEVICE), at])
            sees &= (at[:, None] - place) < case["window"]
        q = st["q"][row:row + n].double().view(n, G, H // G, D)
        weight = torch.einsum("ngrd,gcd->grnc", q, sides[0]) / math.sqrt(D)
        weight = torch.softmax(weight.masked_fill(~sees, -math.inf), -1)
        outs.append(torch.einsum("grnc,gcd->ngrd", weight, sides[1]).reshape(n, H * D))
        row += n
    return torch.cat(outs)
