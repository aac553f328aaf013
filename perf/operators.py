"""The paged cache's operators as cases that can be timed one by one: writing, reading back, attention.

A paged cache keeps the K and V codes of many sequences in one pool of pages.  ``k_codes`` / ``v_codes`` are int32
``[pages, heads, page_size, head_dim * bits / 32]`` (little-endian fields of 2, 4 or 8 bits), ``k_scale`` / ``v_scale`` fp32
``[pages, heads, page_size]``: one scale per token and head.  Slot ``page * page_size + offset`` names a token's place; a block table
``[sequences, pages]`` says which pages hold a sequence.  ``op`` of a case says what a pass does:

* ``write_read``  quantise the K and V of new tokens into their slots (slot -1: a padding token, not written), and read the same
                  slots back: the values that the written cache stands for.
* ``read``        read the tokens of cached sequences back in order.
* ``attend``      a chunk of new queries per sequence, the last tokens of it, over its pages: full, causal, or causal within a
                  sliding window next to a few first tokens that stay visible.  One query per sequence is a decoding step.

Inputs are synthetic: activations ~N(0, 1) with a few large channels, queries with a common direction that the first keys of a
sequence answer to, slots and pages in random order, and scales that are NaN where nothing was written.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------ the cases
def _write(name, tokens, heads, dim, kb, vb, dtype, page=64, fused=False):
    return {"name": name, "op": "write_read", "tokens": tokens, "heads": heads, "dim": dim, "kb": kb, "vb": vb, "dtype": dtype, "page": page,
            "fused": fused}


def _read(name, batch, lo, hi, heads, dim, kb, vb, dtype, page=64):
    return {"name": name, "op": "read", "batch": batch, "kv_lo": lo, "kv_hi": hi, "heads": heads, "dim": dim, "kb": kb, "vb": vb, "dtype": dtype,
            "page": page}


def _attend(name, batch, q_lo, q_hi, lo, hi, heads, group, dim, kb, vb, dtype, page=64, causal=True, window=0, sinks=0, lse=False):
    """kv_lo, kv_hi: tokens cached before the chunk; window 0: none."""
    return {"name": name, "op": "attend", "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "kv_lo": lo, "kv_hi": hi, "heads": heads, "group": group,
            "dim": dim, "kb": kb, "vb": vb, "dtype": dtype, "page": page, "causal": causal, "window": window, "sinks": sinks, "lse": lse}


def listed():
    return [
        # one decoding step of a small batch writes a token per sequence: latency
        _write("write 8 tokens", 8, 8, 128, 8, 8, "bf16"),
        # the ragged chunks of a batch, padding tokens among them, K and V as views of a fused QKV activation
        _write("write 999 tokens, fused qkv", 999, 12, 64, 4, 2, "fp16", page=32, fused=True),
        # a long prompt
        _write("write 32768 tokens", 32768, 8, 128, 8, 8, "bf16"),
        # a few short sequences handed to a library that wants plain fp32 K and V
        _read("read 3 sequences", 3, 100, 680, 16, 64, 8, 8, "fp32", page=16),
        # long contexts read back for a program that recomputes on them
        _read("read 8 sequences", 8, 4000, 10521, 8, 128, 4, 4, "bf16"),
        # one sequence decodes over a short context: latency
        _attend("decode 1 sequence", 1, 1, 1, 1000, 1000, 8, 4, 128, 8, 8, "bf16", lse=True),
        # a serving batch decodes over long contexts
        _attend("decode 64 sequences", 64, 1, 1, 2000, 10520, 16, 1, 128, 4, 4, "bf16"),
        # few tokens per sequence (a draft being checked), sliding window and first tokens, groups of five heads
        _attend("verify 4 tokens, window", 24, 4, 4, 500, 30000, 8, 5, 128, 8, 4, "fp16", page=16, window=1024, sinks=4),
        # a chunk of a prompt behind a long context
        _attend("chunk 2048 behind 16384", 1, 2048, 2048, 16384, 16384, 8, 4, 128, 8, 8, "bf16", page=128),
        # ragged chunks of several prompts
        _attend("ragged chunks", 8, 17, 512, 0, 4000, 12, 1, 64, 4, 4, "fp16", page=16, lse=True),
        # a chunk of a prompt with a sliding window and first tokens
        _attend("chunk 4096, window", 1, 4096, 4096, 28672, 28672, 4, 4, 128, 8, 8, "bf16", window=2048, sinks=16),
        # one scale of an image schedule: every new token sees all of them
        _attend("scale 32 of 512px", 16, 1024, 1024, 1216, 1216, 30, 1, 64, 4, 4, "bf16", page=32, causal=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write_read", "read", "decode", "decode", "chunk", "chunk", "chunk"))
    dim, dtype, page = rng.choice((64, 128)), rng.choice(("bf16", "fp16")), rng.choice((16, 32, 64, 128))
    kb, vb = rng.choice(((8, 8), (8, 8), (4, 4), (4, 4), (8, 4), (4, 2), (2, 2), (4, 8)))
    if op == "write_read":
        return _unnamed(_write("", _log(rng, 8, 32768), rng.choice((1, 2, 3, 4, 6, 7, 9)), dim, kb, vb, rng.choice(("bf16", "fp16", "fp32")), page, rng.random() < 0.5))
    if op == "read":
        hi = _log(rng, 100, 10000)
        return _unnamed(_read("", _log(rng, 1, 8), max(1, hi // rng.randint(1, 5)), hi, rng.choice((1, 2, 3, 4, 7, 8)), dim, kb, vb,
                              rng.choice(("bf16", "fp16", "fp32")), page))
    while True:
        heads, group = rng.choice((1, 2, 4, 5, 8, 10, 16)), rng.choice((1, 1, 2, 4, 5, 7, 8))
        batch, hi = _log(rng, 1, 64), _log(rng, 100, 30000)
        q = rng.choice((1, 1, 1, 2, 3, 4)) if op == "decode" else _log(rng, 5, 4096)
        causal = op == "decode" or rng.random() < 0.7
        window = _log(rng, 16, 4096) if causal and rng.random() < 0.4 else 0
        c = _attend("", batch, q if op == "decode" else rng.randint(1, q), q, hi // rng.randint(1, 5) if rng.random() < 0.8 else 0, hi, heads, group, dim, kb,
                    vb, dtype, page, causal, window, rng.choice((0, 1, 4, 100)) if window else 0, rng.random() < 0.3)
        w = work(c)
        # no more than the largest listed decoding step, chunk, or score matrix of the plain form
        if w["bytes"] < 8e8 and w["flops"] < 4e11 and batch * (q + hi) * heads < 1.1e7 and batch * heads * group * q * (q + hi) < 1.3e9:
            return _unnamed(c)


def _unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """Tokens in the cache and queries of every sequence: spread over their ranges, both ends included, the same for every seed."""
    n = case["batch"]
    rng = random.Random(n * 7919 + case["kv_hi"] * 31 + case.get("q_hi", 0))
    spread = lambda lo, hi: [hi, lo][:n] + [rng.randint(lo, hi) for _ in range(n - 2)]  # noqa: E731
    before = spread(case["kv_lo"], case["kv_hi"])
    if case["op"] == "read":
        return before, [0] * n
    new = spread(case["q_lo"], case["q_hi"])
    return [a + b for a, b in zip(before, new)], new


def work(case):
    heads, dim = case["heads"], case["dim"]
    row = dim * (case["kb"] + case["vb"]) // 8 + 8                       # codes and scales of a token and head
    if case["op"] == "write_read":                                        # every input once, the cache once, every output once
        return {"bytes": case["tokens"] * (heads * (2 * 2 * dim * SIZE[case["dtype"]] + row) + 8), "flops": 0}
    kv, new = _lengths(case)
    if case["op"] == "read":
        return {"bytes": sum(kv) * (heads * (2 * dim * SIZE[case["dtype"]] + row) + 8), "flops": 0}
    seen = pairs = 0
    for n, q in zip(kv, new):
        if not case["causal"]:
            seen, pairs = seen + n, pairs + n * q
            continue
        w, s, p0 = case["window"] or n, case["sinks"], n - q                # positions p0 .. n - 1
        first = max(0, p0 - w + 1)                                           # first key of the window of the first query
        seen += n - first + min(s, first)
        grow = max(0, min(q, w - p0))                                        # queries whose window begins at token 0
        pairs += grow * p0 + grow * (grow + 1) // 2 + (q - grow) * w
        if s:                                                                # first tokens left of the window
            pairs += sum(min(s, max(0, p0 + i - w + 1)) for i in range(q))
    hq = heads * case["group"]
    return {"bytes": seen * heads * row + sum(new) * hq * (2 * dim * SIZE[case["dtype"]] + (4 if case["lse"] else 0)), "flops": 4 * dim * hq * pairs}


# ------------------------------------------------------------------------------------------------ the cache's format, in torch
def _unpack(words, bits):
    """int32 words [..., w] -> signed fields [..., w * 32 / bits]"""
    left = torch.arange(32 - bits, -1, -bits, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) << left) >> (32 - bits)).flatten(-2)


def _quantise(x, bits):
    """x [..., dim] fp32 -> int32 words and scales: abs-max over the row, codes rounded half to even, fields little-endian"""
    top = torch.tensor(float(2 ** (bits - 1) - 1), device=x.device)
    scale = (x.abs().amax(-1) / top).clamp_min(1e-12)
    codes = torch.round(x / scale.unsqueeze(-1)).to(torch.int32).clamp(-2 ** (bits - 1), 2 ** (bits - 1) - 1)
    shift = torch.arange(0, 32, bits, device=x.device, dtype=torch.int32)
    fields = (codes & (2 ** bits - 1)).unflatten(-1, (-1, 32 // bits)) << shift
    return fields.sum(-1, dtype=torch.int32), scale


def _activations(gen, tokens, heads, dim):
    x = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    x[..., ::max(8, dim // 4)] *= 5.0
    return x


def _pools(case, pages, gen):
    """Pools in which nothing is written: any codes, and no scale"""
    made = {}
    for name, bits in (("k", case["kb"]), ("v", case["vb"])):
        shape = (pages, case["heads"], case["page"])
        made[name + "_codes"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (*shape, case["dim"] * bits // 32), generator=gen, device="cuda", dtype=torch.int32)
        made[name + "_scale"] = torch.full(shape, math.nan, device="cuda")
    return made


def _put(state, name, slots, words, scale):
    page = state["page"]
    where, at = slots // page, slots % page
    state[name + "_codes"][where, :, at] = words
    state[name + "_scale"][where, :, at] = scale


def _filled(case, gen):
    """Pools that hold the cached tokens of every sequence in pages in random order, the block table (-1 behind a sequence's last page), the
    lengths, and the common direction of queries and first keys."""
    kv, new = _lengths(case)
    page, heads, dim = case["page"], case["heads"], case["dim"]
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
    state = {"page": page, **_pools(case, sum(need) + 3, gen)}
    table = torch.full((len(kv), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    toward, at, slots = torch.randn((heads, dim), generator=gen, device="cuda"), 0, []
    for b, n in enumerate(kv):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        i = torch.arange(n, device="cuda")
        s = table[b].long()[i // page] * page + i % page
        slots.append(s)
        for k in range(0, n, 65536):
            part = s[k:k + 65536]
            for name, bits in (("k", case["kb"]), ("v", case["vb"])):
                x = _activations(gen, part.numel(), heads, dim)
                if k == 0 and name == "k":
                    x[:4] += 2.0 * toward
                _put(state, name, part, *_quantise(x, bits))
    state.update(table=table, kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"), slots=torch.cat(slots))
    return state, toward, kv, new


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, heads, dim, dtype = case["op"], case["heads"], case["dim"], DTYPES[case["dtype"]]
    if op == "write_read":
        tokens, page = case["tokens"], case["page"]
        pages = -(-tokens // page) + 2
        state = {"page": page, **_pools(case, pages, gen)}
        kv = _activations(gen, tokens, 3 * heads, dim).to(dtype).view(tokens, 3, heads, dim)
        # views of a fused activation, or tensors of their own
        state["k"], state["v"] = (kv[:, 1], kv[:, 2]) if case["fused"] else (kv[:, 1].contiguous(), kv[:, 2].contiguous())
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens]
        # runs of consecutive slots, as pages give them, in random order
        run = torch.randperm(pages, generator=gen, device="cuda").unsqueeze(1) * page + torch.arange(page, device="cuda")
        slots = run.flatten()[:tokens] if tokens >= page else slots
        if case["fused"] and tokens > 16:
            slots = torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.05, -1, slots)
        state["slots"] = slots
    else:
        state, toward, kv, new = _filled(case, gen)
        if op == "attend":
            q = torch.randn((sum(new), heads, case["group"], dim), generator=gen, device="cuda") * 1.5 + 0.5 * toward.unsqueeze(1)
            state["q"] = q.reshape(sum(new), heads * case["group"], dim).to(dtype)
            state["q_starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
            state["max_q"], state["max_kv"] = max(new), max(kv)
    state["op"], state["bits"], state["dim"], state["dtype"] = op, (case["kb"], case["vb"]), dim, dtype
    if op == "attend":
        state.update(softmax_scale=1.0 / math.sqrt(dim), causal=case["causal"], window=case["window"] or None, sinks=case["sinks"], lse=case["lse"])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    cache = state.get("cache")
    if cache is None:                                     # the handle that a program makes once, with its pools
        package = os.path.abspath("var-q_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from VAR_Q.paged import PagedCache
        cache = state["cache"] = PagedCache.over(state["k_codes"], state["v_codes"], state["k_scale"], state["v_scale"], state["dim"])
    if state["op"] == "write_read":
        cache.append(state["k"], state["v"], state["slots"])
    if state["op"] != "attend":
        return cache.read(state["slots"], state["dtype"])
    return cache.attend(state["q"], state["table"], state["kv_lens"], state["q_starts"], state["max_q"], state["max_kv"], state["softmax_scale"],
                        causal=state["causal"], window=state["window"], sinks=state["sinks"], return_lse=state["lse"])


def _run_plain(state):
    if state["op"] == "write_read":
        keep = state["slots"] >= 0
        slots = state["slots"][keep]
        _put(state, "k", slots, *_quantise(state["k"][keep].float(), state["bits"][0]))
        _put(state, "v", slots, *_quantise(state["v"][keep].float(), state["bits"][1]))
    if state["op"] != "attend":
        return _plain_read(state, "k", state["bits"][0]), _plain_read(state, "v", state["bits"][1])
    return _plain_attend(state)


def _plain_read(state, name, bits):
    slots, page = state["slots"], state["page"]
    where, at = slots.clamp_min(0) // page, slots.clamp_min(0) % page
    x = _unpack(state[name + "_codes"][where, :, at], bits).float() * state[name + "_scale"][where, :, at].unsqueeze(-1)
    return torch.where((slots >= 0).view(-1, 1, 1), x, 0.0).to(state["dtype"])


def _dense(state, name, bits):
    """K or V of all sequences [B, H, L, dim] in fp32, zero behind a sequence's end"""
    table = state["table"].long().clamp_min(0)
    x = _unpack(state[name + "_codes"][table], bits).float() * state[name + "_scale"][table].unsqueeze(-1)
    x = x.permute(0, 2, 1, 3, 4).flatten(2, 3)                                          # [B, H, L, dim]
    there = torch.arange(x.shape[2], device=x.device) < state["kv_lens"].unsqueeze(1)
    return torch.where(there.view(len(table), 1, -1, 1), x, 0.0)


def _plain_attend(state):
    q, starts, kv_lens, most = state["q"], state["q_starts"].long(), state["kv_lens"].long(), state["max_q"]
    k = _dense(state, "k", state["bits"][0])
    batch, heads, length, dim = k.shape
    group, dev = q.shape[1] // heads, q.device
    counts = starts[1:] - starts[:-1]
    i = torch.arange(most, device=dev)
    rows = (starts[:-1].unsqueeze(1) + i).clamp_max(max(0, q.shape[0] - 1))              # [B, most]
    qd = q[rows].float().view(batch, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim)
    s = torch.matmul(qd, k.transpose(2, 3)).view(batch, heads, group, most, length)
    s = s.mul_(state["softmax_scale"])
    del k
    p = (kv_lens - counts).unsqueeze(1) + i                                               # position of a query
    j = torch.arange(length, device=dev)
    seen = (j < kv_lens.unsqueeze(1)).unsqueeze(1) & (i < counts.unsqueeze(1)).unsqueeze(2)
    if state["causal"]:
        seen = seen & (j <= p.unsqueeze(2))
        if state["window"]:
            seen = seen & ((p.unsqueeze(2) - j < state["window"]) | (j < state["sinks"]))
    s = s.masked_fill_(~seen.view(batch, 1, 1, most, length), -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    e = s.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(batch, heads, group * most, length), _dense(state, "v", state["bits"][1])).view(batch, heads, group, most, dim)
    o = torch.where(total > 0, o / total, 0.0)
    token = torch.arange(q.shape[0], device=dev)
    b = (token.unsqueeze(1) >= starts[1:]).sum(1)                                         # sequence of a token
    at = token - starts[b]
    out = o.permute(0, 3, 1, 2, 4)[b, at].reshape(q.shape).to(q.dtype)
    if not state["lse"]:
        return out
    lse = (m + total.log()).squeeze(-1)
    return out, lse.permute(0, 3, 1, 2)[b, at].reshape(q.shape[0], q.shape[1])


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definition
def exact(case, seed):
    state = prepare(case, seed)
    page, dim = state["page"], case["dim"]

    def rounded(x, bits):                      # the values that a row's codes stand for
        scale = (x.abs().max(-1, keepdim=True).values / (2 ** (bits - 1) - 1)).clamp(min=1e-12)
        return (x / scale).round().clamp(-2 ** (bits - 1), 2 ** (bits - 1) - 1) * scale

    def held(name, bits, slots):               # [tokens, heads, dim] of the pools
        w = state[name + "_codes"].transpose(1, 2).reshape(-1, case["heads"], dim * bits // 32)[slots].to(torch.int64) & 0xffffffff
        x = torch.stack([(w >> (bits * f)) % 2 ** bits for f in range(32 // bits)], -1).reshape(len(slots), case["heads"], dim)
        x = torch.where(x >= 2 ** (bits - 1), x - 2 ** bits, x)
        return x.double() * state[name + "_scale"].transpose(1, 2).reshape(-1, case["heads"], 1)[slots].double()

    if case["op"] == "write_read":
        gone = (state["slots"] < 0).view(-1, 1, 1)
        return tuple(rounded(state[n].double(), case[n + "b"]).masked_fill(gone, 0.0) for n in ("k", "v"))
    if case["op"] == "read":
        return held("k", case["kb"], state["slots"]), held("v", case["vb"], state["slots"])
    kv, new = _lengths(case)
    outs, sums, group = [], [], case["group"]
    for b, (n, c) in enumerate(zip(kv, new)):
        j = torch.arange(n, device="cuda")
        slots = state["table"][b].long()[j // page] * page + j % page
        k, v = held("k", case["kb"], slots), held("v", case["vb"], slots)
        q = state["q"][sum(new[:b]):sum(new[:b + 1])].double()
        out = torch.zeros((c, case["heads"] * group, dim), dtype=torch.float64, device="cuda")
        lse = torch.full((c, case["heads"] * group), -math.inf, dtype=torch.float64, device="cuda")
        pos = torch.arange(n - c, n, device="cuda").unsqueeze(1)
        blind = torch.zeros((c, n), dtype=torch.bool, device="cuda")
        if case["causal"]:
            blind |= j > pos
            if case["window"]:
                blind |= (pos - j >= case["window"]) & (j >= case["sinks"])
        for h in range(case["heads"] * group):
            s = (q[:, h] @ k[:, h // group].T / math.sqrt(dim)).masked_fill(blind, -math.inf)
            lse[:, h] = s.logsumexp(-1)
            out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
        outs.append(out)
        sums.append(lse)
    return (torch.cat(outs), torch.cat(sums)) if case["lse"] else torch.cat(outs)
