"""Performance cases of the INT8 key/value cache and the attention that reads it.

What stands behind them: a server that decodes a batch of sequences.  A prompt pass writes the keys and values of its
tokens into the cache (rotated, then quantized with one scale per head and token) and reads them back for the prompt
attention; every decode step appends one token per sequence and attends to the cache; sequences that begin with the
same tokens (a system prompt) share the cache rows of that prefix.

A cache is codes int8 [batch, kv_heads, max_seq, head_dim] and scales fp32 [batch, kv_heads, max_seq], for keys and for
values.  A row r of head_dim values is held as scale = a / 127, code = clamp(round_half_away(r * (127 / a))), with
a = max(1e-8, max |r|), every operation rounded to fp32: the package's own per-row INT8 quantizer, so that codes and
scales are whole answers, not approximations.  The rotation in front of it rounds every operation to fp32 as well.

Sizes are those of the benchmark's decoder (batch 8, 16 heads of 128, 512-token prompts, 640 positions) and generic ones
around them: grouped heads, heads of 64, one to tens of thousands of positions, ragged batches.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

MAX_ROWS = 8 * 32 * 8192            # key/value rows (sequence, kv head, position) of the largest decode batch
MAX_WRITE = 8 * 512 * 48 * 128      # values of the largest prompt written
MAX_LOAD = 8 * 16 * 512 * 128       # values of the largest cache part read back
MAX_PREFIX_WORK = 32 * 32 * 16384   # (query row, prefix position) pairs


def _package():
    return importlib.import_module("soverign-grad_b200")       # the directory name is not a Python identifier


def listed():
    return [
        # the benchmark decoder's prompt pass: eight prompts of 512 tokens, one block
        {"name": "store_b8_t512_h16", "kind": "store", "batch": 8, "tokens": 512, "heads": 16, "kv_heads": 16, "dim": 128, "max_seq": 640,
         "start": 0, "ragged": False},
        # a later chunk of three padded prompts with grouped heads of 64, into a cache of odd length
        {"name": "store_b3_t777_gqa_ragged", "kind": "store", "batch": 3, "tokens": 777, "heads": 24, "kv_heads": 8, "dim": 64, "max_seq": 2055,
         "start": 1000, "ragged": True},
        # the same decoder's prompt attention reads those rows back
        {"name": "load_b8_r512_h16", "kind": "load", "batch": 8, "kv_heads": 16, "dim": 128, "max_seq": 640, "rows": 512, "shared": False},
        # a shared prefix of odd length is read back in front of each of four sequences' own rows
        {"name": "load_prefix_b4_r1023", "kind": "load", "batch": 4, "kv_heads": 8, "dim": 64, "max_seq": 1055, "rows": 1023, "shared": True},
        # one sequence early in its answer: nothing but call, launch and latency
        {"name": "decode_b1_h16_130", "kind": "decode", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 128, "max_seq": 640, "longest": 130,
         "ragged": False, "idle": False},
        # the benchmark decoder's decode step, half way through its answer
        {"name": "decode_b8_h16_576", "kind": "decode", "batch": 8, "heads": 16, "kv_heads": 16, "dim": 128, "max_seq": 640, "longest": 576,
         "ragged": False, "idle": False},
        # a ragged batch with three heads of 64 per key/value head, one slot of it free, a cache of odd length
        {"name": "decode_b5_d64_ragged", "kind": "decode", "batch": 5, "heads": 12, "kv_heads": 4, "dim": 64, "max_seq": 1501, "longest": 1500,
         "ragged": True, "idle": True},
        # a full serving batch of long conversations with grouped heads
        {"name": "decode_b32_gqa_8192_ragged", "kind": "decode", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "max_seq": 8192,
         "longest": 8192, "ragged": True, "idle": False},
        # one sequence over a very long document
        {"name": "decode_b1_gqa_131071", "kind": "decode", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "max_seq": 131072,
         "longest": 131071, "ragged": False, "idle": False},
        # the benchmark decoder behind a shared system prompt
        {"name": "prefix_b8_h16_2048", "kind": "prefix", "batch": 8, "heads": 16, "kv_heads": 16, "dim": 128, "max_seq": 256, "longest": 128,
         "prefix": 2048, "prefix_max": 2048, "ragged": False, "idle": False},
        # a serving batch that asks about one long document, ragged answers
        {"name": "prefix_b32_gqa_16384", "kind": "prefix", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "max_seq": 512, "longest": 512,
         "prefix": 16383, "prefix_max": 16384, "ragged": True, "idle": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choices(["store", "load", "decode", "prefix"], [20, 15, 40, 25])[0]
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16])
    while kv_heads * group > 64:
        group = rng.choice([1, 2, 4])
    heads = kv_heads * group
    if kind == "store":
        width = (heads + 2 * kv_heads) * dim
        batch = rng.randint(1, 8)
        tokens = min(_log_int(rng, 1, 4096), max(1, MAX_WRITE // (batch * width)))
        start = rng.choice([0, 0, rng.randint(1, 2000)])
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "max_seq": start + tokens + rng.randint(0, 300), "start": start, "ragged": rng.random() < 0.4}
    if kind == "load":
        batch = rng.randint(1, 8)
        rows = min(_log_int(rng, 1, 8192), max(1, MAX_LOAD // (batch * kv_heads * dim)))
        return {"kind": kind, "batch": batch, "kv_heads": kv_heads, "dim": dim, "max_seq": rows + rng.randint(0, 200), "rows": rows,
                "shared": rng.random() < 0.4}
    batch = _log_int(rng, 1, 48)
    if kind == "decode":
        longest = min(_log_int(rng, 1, 131072), max(1, MAX_ROWS // (batch * kv_heads)), max(1, 4 * MAX_ROWS // (batch * heads)))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "max_seq": longest + rng.randint(0, longest // 4 + 4), "longest": longest, "ragged": rng.random() < 0.5,
                "idle": batch > 1 and rng.random() < 0.2}
    prefix = min(_log_int(rng, 16, 32768), max(1, MAX_PREFIX_WORK // (batch * heads)))
    longest = min(_log_int(rng, 1, 1024), max(1, MAX_ROWS // (16 * batch * kv_heads)))
    return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "max_seq": longest + rng.randint(0, 64),
            "longest": longest, "prefix": prefix, "prefix_max": prefix + rng.randint(0, 100), "ragged": rng.random() < 0.5,
            "idle": batch > 1 and rng.random() < 0.2}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _rope_tables(rows, dim):
    """cos and sin [rows, dim / 2] of the angles position * 10000 ^ (-2 i / dim), taken in 64 bits."""
    i = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * torch.pow(10000.0, -2.0 * i / dim)[None, :]
    return angle.cos().float(), angle.sin().float()


def _rows(gen, *shape):
    """Key-like rows: N(0, 1) with a few channels (the same for every row) several times larger, as keys of a trained
    model have."""
    x = torch.randn(*shape, device="cuda", generator=gen)
    hot = torch.randint(0, shape[-1], (2,), device="cuda", generator=gen)
    x[..., hot] *= 4.0
    return x


def _cache(gen, batch, kv_heads, max_seq, dim):
    """A cache that holds quantized rows at every position."""
    k_codes, k_scales = _quantize(_rows(gen, batch, kv_heads, max_seq, dim))
    v_codes, v_scales = _quantize(torch.randn(batch, kv_heads, max_seq, dim, device="cuda", generator=gen))
    return {"k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes, "v_scales": v_scales}


def _positions(case, gen):
    """Tokens already in the cache of each sequence: all `longest` - 1, or ragged with the longest among them; an idle
    slot has -1."""
    batch, longest = case["batch"], case["longest"]
    pos = torch.full((batch,), longest - 1, device="cuda", dtype=torch.int32)
    if case["ragged"] and batch > 1:
        pos[1:] = torch.randint(0, longest, (batch - 1,), device="cuda", generator=gen, dtype=torch.int32)
    if case["idle"]:
        pos[batch // 2] = -1
    return pos


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, kv_heads, dim, max_seq = case["batch"], case["kv_heads"], case["dim"], case["max_seq"]
    state = dict(case)
    if case["kind"] == "load":
        state["cache"] = _cache(gen, 1 if case["shared"] else batch, kv_heads, max_seq, dim)
        return state
    heads = case["heads"]
    width = (heads + 2 * kv_heads) * dim
    if case["kind"] == "store":
        tokens = case["tokens"]
        state["qkv"] = _rows(gen, batch, tokens, width // dim, dim).reshape(batch, tokens, width)
        state["cache"] = {"k_codes": torch.zeros(batch, kv_heads, max_seq, dim, dtype=torch.int8, device="cuda"),
                          "k_scales": torch.zeros(batch, kv_heads, max_seq, device="cuda"),
                          "v_codes": torch.zeros(batch, kv_heads, max_seq, dim, dtype=torch.int8, device="cuda"),
                          "v_scales": torch.zeros(batch, kv_heads, max_seq, device="cuda")}
        state["cos"], state["sin"] = _rope_tables(max_seq, dim)
        state["pos"] = torch.full((batch,), case["start"], dtype=torch.int32, device="cuda")
        state["n_new"] = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            state["pos"] = torch.randint(0, case["start"] + 1, (batch,), device="cuda", generator=gen, dtype=torch.int32)
            state["n_new"][1:] = torch.randint(1, tokens + 1, (batch - 1,), device="cuda", generator=gen, dtype=torch.int32)
        state["q_out"] = torch.zeros(batch, tokens, heads * dim, device="cuda")
        return state
    state["qkv"] = _rows(gen, batch, 1, width // dim, dim).reshape(batch, 1, width)
    state["cache"] = _cache(gen, batch, kv_heads, max_seq, dim)
    state["pos"] = _positions(case, gen)
    table = max_seq
    if case["kind"] == "prefix":
        state["prefix_cache"] = _cache(gen, 1, kv_heads, case["prefix_max"], dim)
        state["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
        table += case["prefix_max"]
    state["cos"], state["sin"] = _rope_tables(table, dim)
    return state


# ---- the plain form -------------------------------------------------------------------------------------------------

def _quantize(rows):
    """Codes and scales of the rows (the last axis): the divisions are by tensors because a division by a number is a
    product with its rounded inverse on the GPU."""
    top = rows.abs().amax(-1).clamp_min(1e-8)
    most = torch.full_like(top, 127.0)
    scaled = rows * (most / top)[..., None]
    whole = torch.trunc(scaled)
    up = torch.where((scaled - whole).abs() >= 0.5, torch.sign(scaled), torch.zeros_like(scaled))
    return (whole + up).clamp(-127.0, 127.0).to(torch.int8), top / most


def _rotate(x, cos, sin):
    """Pairs (d, d + dim / 2) of x [..., dim]; cos and sin [..., dim / 2]."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _split(state):
    """q [B, T, H, D], k and v [B, T, Hkv, D] of the rows of qkv."""
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    batch, tokens, _ = state["qkv"].shape
    rows = state["qkv"].view(batch, tokens, heads + 2 * kv_heads, dim)
    return rows[:, :, :heads], rows[:, :, heads:heads + kv_heads], rows[:, :, heads + kv_heads:]


def _store(state, offset):
    """Rotated queries [B, T, H, D]; keys and values quantized into the cache.  Tokens that are not there (behind n_new,
    or of an idle slot) leave everything as it was.  Returns the queries and which tokens are there."""
    q, k, v = _split(state)
    cache, tokens = state["cache"], q.shape[1]
    step = torch.arange(tokens, device="cuda")
    at = state["pos"].long()[:, None] + step[None, :]
    there = at >= 0
    if "n_new" in state:
        there = there & (step[None, :] < state["n_new"].long()[:, None])
    at = at.clamp_min(0)
    angle = (at + offset).clamp_max(state["cos"].shape[0] - 1)
    cos, sin = state["cos"][angle][:, :, None, :], state["sin"][angle][:, :, None, :]
    i = torch.arange(at.shape[0], device="cuda")[:, None]
    for name, rows in (("k", _rotate(k, cos, sin)), ("v", v)):
        codes, scales = _quantize(rows)
        held, held_scales = cache[name + "_codes"], cache[name + "_scales"]
        held[i, :, at] = torch.where(there[:, :, None, None], codes, held[i, :, at])
        held_scales[i, :, at] = torch.where(there[:, :, None], scales, held_scales[i, :, at])
    return _rotate(q, cos, sin), there


def _values(cache, name, rows):
    """The first `rows` positions as the values they stand for, fp32."""
    return cache[name + "_codes"][:, :, :rows].float() * cache[name + "_scales"][:, :, :rows, None]


def _attend(state, offset):
    q, there = _store(state, offset)
    batch, heads, kv_heads, dim, rows = state["batch"], state["heads"], state["kv_heads"], state["dim"], state["longest"]
    q = q.reshape(batch, kv_heads, heads // kv_heads, dim) * (1.0 / math.sqrt(dim))
    keys, values = _values(state["cache"], "k", rows), _values(state["cache"], "v", rows)
    scores = q @ keys.transpose(-1, -2)                                                   # [B, Hkv, G, rows]
    behind = torch.arange(rows, device="cuda")[None, :] > state["pos"].long()[:, None]
    scores = scores.masked_fill(behind[:, None, None, :], -math.inf)
    if "prefix_cache" in state:
        first, p = state["prefix_cache"], state["prefix"]
        shared = q.permute(1, 0, 2, 3).reshape(kv_heads, -1, dim) @ _values(first, "k", p)[0].transpose(-1, -2)
        shared = shared.view(kv_heads, batch, heads // kv_heads, p).permute(1, 0, 2, 3)
        scores = torch.cat([shared, scores], -1)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    weights = weights / weights.sum(-1, keepdim=True)
    if "prefix_cache" in state:
        out = weights[..., p:] @ values
        shared = weights[..., :p].permute(1, 0, 2, 3).reshape(kv_heads, -1, p) @ _values(first, "v", p)[0]
        out = out + shared.view(kv_heads, batch, heads // kv_heads, dim).permute(1, 0, 2, 3)
    else:
        out = weights @ values
    return torch.where(there[:, :, None, None], out, torch.zeros_like(out)).reshape(batch, heads * dim)


# ---- one pass -------------------------------------------------------------------------------------------------------

def _run_own(state):
    sgq = _package()
    kind, cache = state["kind"], sgq.KVCacheInt8(**state["cache"])
    if kind == "load":
        keys, values = sgq.kv_load_int8(cache, state["rows"], batch=state["batch"])
        return {"keys": keys, "values": values}
    if kind == "store":
        sgq.rope_kv_store_int8(state["qkv"], cache, state["cos"], state["sin"], state["pos"], state["heads"], q_out=state["q_out"],
                               n_new=state["n_new"])
        return {"q": state["q_out"], **state["cache"]}
    if kind == "decode":
        out = sgq.attn_decode_int8(state["qkv"], cache, state["cos"], state["sin"], state["pos"], state["heads"])
    else:
        out = sgq.attn_decode_prefix_int8(state["qkv"], cache, sgq.KVCacheInt8(**state["prefix_cache"]), state["prefix_len"], state["cos"],
                                          state["sin"], state["pos"], state["heads"])
    return {"out": out, **state["cache"]}


def run(state):
    """One pass.  The cache that a pass writes comes back as it is held: whole codes, which have to be the same ones, and
    their scales."""
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "load":
        rows, batch = state["rows"], state["batch"]
        keys, values = _values(state["cache"], "k", rows), _values(state["cache"], "v", rows)
        return {"keys": keys.expand(batch, -1, -1, -1).contiguous(), "values": values.expand(batch, -1, -1, -1).contiguous()}
    if kind == "store":
        q, there = _store(state, 0)
        state["q_out"].copy_(torch.where(there[:, :, None], q.reshape(state["q_out"].shape), state["q_out"]))
        return {"q": state["q_out"], **state["cache"]}
    return {"out": _attend(state, state["prefix"] if kind == "prefix" else 0), **state["cache"]}


def work(case):
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["dim"]
    row = dim + 4                                                       # a quantized row: codes and scale
    if case["kind"] == "load":
        read = (1 if case["shared"] else batch) * kv_heads * case["rows"]
        wrote = batch * kv_heads * case["rows"]
        return {"bytes": 2 * (read * row + wrote * dim * 4), "flops": 2 * wrote * dim}
    heads = case["heads"]
    width = (heads + 2 * kv_heads) * dim
    if case["kind"] == "store":
        tokens = batch * case["tokens"] * (0.5 if case["ragged"] and batch > 1 else 1.0)
        return {"bytes": tokens * (width * 4 + heads * dim * 4 + 2 * kv_heads * row + dim * 4), "flops": tokens * width * 5}
    live = batch - 1 if case["idle"] else batch
    rows = live * case["longest"]
    if case["ragged"] and live > 1:                                     # lengths are spread evenly below the longest
        rows = case["longest"] + (live - 1) * (case["longest"] + 1) / 2
    byte = 2 * kv_heads * rows * row + batch * (width + heads * dim) * 4
    flops = 4 * heads * dim * rows
    if case["kind"] == "prefix":
        byte += 2 * kv_heads * case["prefix"] * row
        flops += 4 * live * heads * dim * case["prefix"]
    return {"bytes": byte, "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _held(x):
    """What the cache holds of fp32 rows x [..., dim]: codes (as fp64) and scales.  The fp32 roundings belong to the
    definition: they decide which code a value gets."""
    a = torch.maximum(x.abs().max(-1, keepdim=True).values, x.new_full((), 1e-8))
    c = a.new_full(a.shape, 127.0)
    v = (x * torch.div(c, a)).double()
    return torch.sign(v) * torch.floor(v.abs() + 0.5), torch.div(a, c)[..., 0]


def _turned(x, cos, sin, single):
    """Rotation of x [..., dim] in 64 bits, or with every operation rounded to fp32."""
    if not single:
        x, cos, sin = x.double(), cos.double(), sin.double()
    y = torch.empty_like(x)
    h = x.shape[-1] // 2
    y[..., :h] = torch.mul(x[..., :h], cos) - torch.mul(x[..., h:], sin)
    y[..., h:] = torch.mul(x[..., h:], cos) + torch.mul(x[..., :h], sin)
    return y


def exact(case, seed):
    state = prepare(case, seed)
    cache, batch, kv_heads, dim = state["cache"], case["batch"], case["kv_heads"], case["dim"]
    if case["kind"] == "load":
        n = case["rows"]
        read = [cache[c + "_codes"][:, :, :n].double() * cache[c + "_scales"][:, :, :n].double().unsqueeze(-1) for c in "kv"]
        return {"keys": read[0].repeat(batch if case["shared"] else 1, 1, 1, 1), "values": read[1].repeat(batch if case["shared"] else 1, 1, 1, 1)}
    heads, cos, sin = case["heads"], state["cos"], state["sin"]
    if case["kind"] == "store":
        q = torch.zeros(batch, case["tokens"], heads, dim, dtype=torch.float64, device="cuda")
        scales = {"k": cache["k_scales"].double(), "v": cache["v_scales"].double()}
        for b in range(batch):
            n, p = int(state["n_new"][b]), int(state["pos"][b])
            rows = state["qkv"][b, :n].reshape(n, -1, dim)
            c, s = cos[p:p + n, None], sin[p:p + n, None]
            q[b, :n] = _turned(rows[:, :heads], c, s, False)
            scales["k"][b, :, p:p + n] = _held(_turned(rows[:, heads:heads + kv_heads], c, s, True))[1].double().t()
            scales["v"][b, :, p:p + n] = _held(rows[:, heads + kv_heads:])[1].double().t()
        return {"q": q.view(batch, case["tokens"], heads * dim), "k_codes": None, "k_scales": scales["k"], "v_codes": None, "v_scales": scales["v"]}
    out = torch.zeros(batch, kv_heads, heads // kv_heads, dim, dtype=torch.float64, device="cuda")
    before = case["prefix"] if case["kind"] == "prefix" else 0
    first = [state["prefix_cache"][c + "_codes"][0, :, :before].double() * state["prefix_cache"][c + "_scales"][0, :, :before, None].double()
             for c in "kv"] if before else None
    scales = {"k": cache["k_scales"].double(), "v": cache["v_scales"].double()}
    for b in range(batch):
        p = int(state["pos"][b])
        if p < 0:
            continue
        rows = state["qkv"][b, 0].view(-1, dim)
        c, s = cos[before + p], sin[before + p]
        q = _turned(rows[:heads], c, s, False).view(kv_heads, -1, dim)
        read = []
        for name, new in (("k", _turned(rows[heads:heads + kv_heads], c, s, True)), ("v", rows[heads + kv_heads:])):
            codes, scale = _held(new)
            scales[name][b, :, p] = scale.double()
            old = cache[name + "_codes"][b, :, :p].double() * cache[name + "_scales"][b, :, :p, None].double()
            read.append(torch.cat([old, (codes * scale.double()[:, None])[:, None]], 1))
        if before:
            read = [torch.cat([x, y], 1) for x, y in zip(first, read)]
        weights = torch.softmax(torch.bmm(q, read[0].mT) / math.sqrt(dim), -1)
        out[b] = torch.bmm(weights, read[1])
    return {"out": out.view(batch, heads * dim), "k_codes": None, "k_scales": scales["k"], "v_codes": None, "v_scales": scales["v"]}
