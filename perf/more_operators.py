"""Operators around a paged cache as cases that can be timed one by one: norms and rotary positions, trees of drafted tokens, copies of pages.

The cache's format is that of ``perf/operators.py``: int32 codes ``[pages, heads, page_size, head_dim * bits / 32]`` and fp32 scales
``[pages, heads, page_size]``, a slot ``page * page_size + offset`` for a token.  ``op`` of a case says what a pass does:

* ``rotate``   norms of q and k per head (L2 or root mean square, with factors, or none) and the rotation by position, one to three axes.
* ``put``      the same in front of the cache: q comes out, k is quantised into its slots after norm and rotation, v as it is; and the slots are
               read back, the values that the written cache stands for.
* ``tree``     masks and positions of drafted tokens from their parents, and the attention of these tokens over the pages of their sequences:
               each sees the context, its ancestors and itself.
* ``copy``     whole pages of all layers to other pages: forked sequences, a pool that is compacted.
* ``move``     tokens of all layers to other slots: accepted drafts to the end of their sequence, tokens that are kept to fresh pages.

Angles are products of whole positions with frequencies ``base^(-2i / rotary_dim)`` in 64 bits.  Inputs are synthetic: activations ~N(0, 1) with
a few large channels, positions from short prompts to far ones, trees as a drafting model makes them (a few children for the best nodes).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = {"l2": 1e-12, "rms": 1e-6}


# ------------------------------------------------------------------------------------------------ the cases
def _rotate(name, batch, tokens, heads, kv_heads, dim, dtype, norm, sections, interleaved, restart, far=0, rotary=0):
    """sections: pairs of every axis, joined by +; restart: every axis has the frequencies from the first on; rotary 0: all of dim."""
    return {"name": name, "op": "rotate", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "norm": norm,
            "sections": sections, "interleaved": interleaved, "restart": restart, "far": far, "rotary": rotary}


def _put(name, tokens, heads, kv_heads, dim, vb, dtype, norm, sections, interleaved, far=0, page=64, rotary=0):
    """Rotated keys have 8 bits."""
    return {"name": name, "op": "put", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "kb": 8, "vb": vb, "dtype": dtype, "norm": norm,
            "sections": sections, "interleaved": interleaved, "restart": False, "far": far, "page": page, "rotary": rotary}


def _tree(name, batch, q_lo, q_hi, lo, hi, heads, group, dim, kb, vb, dtype, page=64, window=0, sinks=0, lse=False):
    """q_lo, q_hi: drafted tokens of a sequence; kv_lo, kv_hi: its tokens before them."""
    return {"name": name, "op": "tree", "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "kv_lo": lo, "kv_hi": hi, "heads": heads, "group": group, "dim": dim,
            "kb": kb, "vb": vb, "dtype": dtype, "page": page, "window": window, "sinks": sinks, "lse": lse}


def _copy(name, layers, pages, heads, dim, kb, vb, page=64):
    return {"name": name, "op": "copy", "layers": layers, "pages": pages, "heads": heads, "dim": dim, "kb": kb, "vb": vb, "page": page}


def _move(name, layers, groups, lo, hi, draft, heads, dim, kb, vb, page=64):
    """groups: sequences, lo .. hi tokens of each move; draft: they are among so many drafted tokens of their sequence (0: from anywhere to fresh pages)."""
    return {"name": name, "op": "move", "layers": layers, "groups": groups, "lo": lo, "hi": hi, "draft": draft, "heads": heads, "dim": dim, "kb": kb, "vb": vb,
            "page": page}


def listed():
    return [
        # the last scale of a 1024px image schedule: unit queries and keys, rows and columns of the image as two axes
        _rotate("scale 64 of 1024px", 4, 4096, 16, 16, 128, "bf16", "l2", "32+32", True, True),
        # a prompt with pictures in it: time, height and width, views of a fused activation, an odd number of tokens
        _rotate("mixed prompt, three axes", 1, 1777, 28, 4, 128, "fp16", "none", "16+24+24", False, False),
        # a decoding step of a small batch far into its contexts: latency
        _put("put 16 tokens", 16, 32, 8, 128, 8, "bf16", "rms", "64", False, far=1 << 20),
        # a long prompt, values in 4 bits
        _put("put 16384 tokens", 16384, 32, 8, 128, 4, "bf16", "rms", "64", False),
        # one sequence has a small draft checked over a short context: latency
        _tree("tree of 16, 1 sequence", 1, 16, 16, 1000, 1000, 8, 4, 128, 8, 8, "bf16", lse=True),
        # drafts of different sizes, a single token among them, over short contexts, one of them empty
        _tree("ragged trees", 24, 1, 32, 0, 3000, 12, 1, 64, 4, 2, "fp16", page=16, lse=True),
        # drafts over a sliding window and first tokens, groups of five heads
        _tree("trees of 26, window", 16, 26, 26, 500, 30000, 8, 5, 128, 8, 4, "bf16", page=32, window=1024, sinks=4),
        # a serving batch has large drafts checked over long contexts
        _tree("trees of 64, 32 sequences", 32, 64, 64, 2000, 8000, 8, 4, 128, 8, 8, "bf16"),
        # a few sequences are forked: their last pages, in all layers
        _copy("fork 4 sequences", 32, 4, 8, 128, 8, 8),
        # a pool is compacted: pages in use move in front of the others
        _copy("compact 301 pages", 16, 301, 8, 128, 8, 4),
        # the accepted paths of the drafts of a batch, in all layers
        _move("accepted paths", 32, 64, 1, 6, 32, 8, 128, 8, 8),
        # tokens that are kept from long contexts, to fresh pages
        _move("keep 16000 tokens", 8, 8, 1000, 3000, 0, 8, 128, 8, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "put", "tree", "tree", "tree", "copy", "move"))
    dim, dtype = rng.choice((64, 128)), rng.choice(("bf16", "fp16"))
    kb, vb = rng.choice(((8, 8), (8, 8), (4, 4), (4, 4), (8, 4), (4, 2), (2, 2), (4, 8)))
    page = rng.choice((16, 32, 64, 128))
    rotary = rng.choice((0, 0, 0, dim // 2))
    half = (rotary or dim) // 2
    a, b = half // 4, half * 3 // 8
    sections = rng.choice((str(half), "%d+%d" % (half // 2, half // 2), "%d+%d+%d" % (a, b, half - a - b)))
    kv_heads, norm, interleaved = rng.choice((1, 2, 3, 4, 5, 8)), rng.choice(("l2", "rms", "none")), rng.random() < 0.5
    far = rng.choice((0, 0, 5000, 1 << 20))
    while True:
        if op == "rotate":
            c = _rotate("", rng.choice((1, 1, 2, 4, 7)), _log(rng, 16, 16384), kv_heads * rng.choice((1, 2, 4, 7)), kv_heads, dim, rng.choice(("bf16", "fp16", "fp32")),
                        norm, sections, interleaved, rng.random() < 0.5, far, rotary)
            if work(c)["bytes"] < 2.6e8:
                return _unnamed(c)
        elif op == "put":
            c = _put("", _log(rng, 8, 16384), kv_heads * rng.choice((1, 2, 4, 7)), kv_heads, dim, rng.choice((8, 4, 2)), dtype, norm, sections, interleaved, far, page, rotary)
            if work(c)["bytes"] < 3.8e8:
                return _unnamed(c)
        elif op == "tree":
            heads, group = rng.choice((1, 2, 4, 5, 8, 12)), rng.choice((1, 1, 2, 4, 5, 7, 8))
            batch, hi, q = _log(rng, 1, 64), _log(rng, 100, 20000), _log(rng, 4, 96)
            window = _log(rng, 128, 4096) if rng.random() < 0.3 else 0
            c = _tree("", batch, rng.randint(1, q), q, hi // rng.randint(1, 5) if rng.random() < 0.8 else 0, hi, heads, group, dim, kb, vb, dtype, page, window,
                      rng.choice((0, 1, 4, 100)) if window else 0, rng.random() < 0.3)
            if work(c)["flops"] < 1.6e11 and batch * (q + hi) * heads < 2.1e6 and batch * heads * group * q * (q + hi) < 5.3e8:
                return _unnamed(c)
        elif op == "copy":
            c = _copy("", rng.choice((1, 2, 7, 16, 32)), _log(rng, 1, 1200), kv_heads, dim, kb, vb, page)
            if work(c)["bytes"] < 9.8e8:
                return _unnamed(c)
        else:
            draft = rng.choice((0, 8, 26, 64))
            hi = _log(rng, 10, 4000) if not draft else max(1, draft // 4)
            c = _move("", rng.choice((1, 2, 7, 16, 32)), _log(rng, 1, 64), rng.randint(0, hi), hi, draft, kv_heads, dim, kb, vb, page)
            if 0 < work(c)["bytes"] < 5.3e8:
                return _unnamed(c)


def _unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ sizes
def _spread(rng, n, lo, hi):
    """Both ends of a range and numbers between, the same for every seed"""
    return [hi, lo][:n] + [rng.randint(lo, hi) for _ in range(n - 2)]


def _lengths(case):
    """Tokens in the cache, drafted ones included, and drafted tokens of every sequence"""
    n = case["batch"]
    rng = random.Random(n * 7919 + case["kv_hi"] * 31 + case["q_hi"])
    before, new = _spread(rng, n, case["kv_lo"], case["kv_hi"]), _spread(rng, n, case["q_lo"], case["q_hi"])
    rng.shuffle(before)
    return [a + b for a, b in zip(before, new)], new


def _moved(case):
    """Tokens that move, of every sequence"""
    return _spread(random.Random(case["groups"] * 31 + case["hi"]), case["groups"], case["lo"], case["hi"])


def _parents(new):
    """Parents of the drafted tokens, -1: a child of the context; the same for every seed"""
    rng = random.Random(sum(new) * 31 + len(new))
    trees = []
    for n in new:
        trees.append([-1 if i == 0 or rng.random() < 0.05 else rng.randint(max(0, i - 9), i - 1) if rng.random() < 0.7 else rng.randint(0, max(0, i // 4)) for i in range(n)])
        trees[-1] = [min(p, i - 1) for i, p in enumerate(trees[-1])]
    return trees


def _sections(case):
    return [int(s) for s in case["sections"].split("+")]


def work(case):
    heads, dim, op = case["heads"], case["dim"], case["op"]
    if op == "rotate":
        axes = len(_sections(case))
        return {"bytes": case["batch"] * case["tokens"] * (heads + case["kv_heads"]) * dim * SIZE[case["dtype"]] * 2 + case["tokens"] * 4 * axes, "flops": 0}
    row = dim * (case["kb"] + case["vb"]) // 8 + 8                       # codes and scales of a token and head
    if op == "put":                                                       # q twice, k and v once and once more read back, the cache once, slots, positions
        size, kv = dim * SIZE[case["dtype"]], case["kv_heads"]
        return {"bytes": case["tokens"] * (2 * heads * size + 4 * kv * size + kv * row + 8 + 4 * len(_sections(case))), "flops": 0}
    if op == "copy":
        return {"bytes": case["layers"] * case["pages"] * (2 * heads * case["page"] * row + 16), "flops": 0}
    if op == "move":
        return {"bytes": sum(_moved(case)) * (case["layers"] * 2 * heads * row + 16), "flops": 0}
    kv, new = _lengths(case)
    seen = pairs = 0
    for n, q, parents in zip(kv, new, _parents(new)):
        ctx, w, s = n - q, case["window"], case["sinks"]
        depth = []
        for p in parents:
            depth.append(0 if p < 0 else depth[p] + 1)
        first = [max(0, ctx + d - w + 1) if w else 0 for d in depth]     # of the window of every drafted token
        seen += q + max(0, ctx - min(first, default=ctx)) + min(s, min(first, default=0), ctx)
        pairs += sum(d + 1 + max(0, ctx - f) + min(s, f, ctx) for d, f in zip(depth, first))
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


def _activations(gen, *shape):
    x = torch.randn(shape, generator=gen, device="cuda")
    x[..., ::max(8, shape[-1] // 4)] *= 5.0
    return x


def _pools(case, pages, gen, heads, layers=None):
    """Pools in which nothing is written: any codes, and no scale (NaN); with layers, any codes and any scales"""
    made, lead = {}, () if layers is None else (layers,)
    for name, bits in (("k", case["kb"]), ("v", case["vb"])):
        shape = (*lead, pages, heads, case["page"])
        made[name + "_codes"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (*shape, case["dim"] * bits // 32), generator=gen, device="cuda", dtype=torch.int32)
        made[name + "_scale"] = torch.full(shape, math.nan, device="cuda") if layers is None else torch.rand(shape, generator=gen, device="cuda") + 0.01
    return made


def _store(state, name, slots, words, scale):
    page = state["page"]
    where, at = slots // page, slots % page
    state[name + "_codes"][where, :, at] = words
    state[name + "_scale"][where, :, at] = scale


# ------------------------------------------------------------------------------------------------ inputs
def _positions(case, gen):
    """int32 [axes, tokens]: one axis counts on from somewhere; several are a picture's rows and columns behind (a time, for three) a text"""
    n, axes = case["tokens"], len(_sections(case))
    if axes == 1:
        # prompts count on; a decoding step (few tokens) has a place of its own for every token
        if n <= 64 and case["far"]:
            return torch.randint(0, case["far"], (1, n), generator=gen, device="cuda", dtype=torch.int32)
        return (torch.arange(n, device="cuda", dtype=torch.int32) + (case["far"] and int(torch.randint(0, case["far"], (1,), generator=gen, device="cuda")))).view(1, n)
    i = torch.arange(n, device="cuda")
    side = max(1, int(math.sqrt(n)))
    rows = [i // side, i % side] if axes == 2 else [i // (side * max(1, side // 3)), i // side % max(1, side // 3), i % side]
    return torch.stack(rows).to(torch.int32) + case["far"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, heads, dim = case["op"], case["heads"], case["dim"]
    state = {"op": op, "case": case, "dim": dim}
    if op in ("rotate", "put"):
        kvh, dtype, tokens, batch = case["kv_heads"], DTYPES[case["dtype"]], case["tokens"], case.get("batch", 1)
        qkv = _activations(gen, batch * tokens, heads + 2 * kvh, dim).to(dtype)
        q, k, v = qkv.split((heads, kvh, kvh), 1)                         # views of a fused activation
        state.update(dtype=dtype, positions=_positions(case, gen), rotary=case["rotary"] or dim)
        if op == "rotate":
            lead = (batch, tokens) if batch > 1 else (tokens,)
            state.update(q=q.unflatten(0, lead), k=k.unflatten(0, lead))
        else:
            page = case["page"]
            pages = -(-tokens // page) + 2
            run = torch.randperm(pages, generator=gen, device="cuda").unsqueeze(1) * page + torch.arange(page, device="cuda")
            slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens] if tokens < page else run.flatten()[:tokens]
            state.update(q=q, k=k, v=v, page=page, slots=slots, bits=(case["kb"], case["vb"]), **_pools(case, pages, gen, kvh))
        if case["norm"] == "l2":                                          # a factor for every query head
            state.update(q_weight=(torch.rand((heads, 1), generator=gen, device="cuda") * 2 + 1), k_weight=None)
        elif case["norm"] == "rms":                                       # a factor for every dimension
            state.update(q_weight=torch.rand(dim, generator=gen, device="cuda") + 0.5, k_weight=torch.rand(dim, generator=gen, device="cuda") + 0.5)
        else:
            state.update(q_weight=None, k_weight=None)
        return state
    page = state["page"] = case["page"]
    if op == "copy":
        n = case["pages"]
        state.update(_pools(case, 2 * n + 3, gen, heads, case["layers"]))
        order = torch.randperm(2 * n + 3, generator=gen, device="cuda")
        state.update(src=order[:n].contiguous(), dst=order[n:2 * n].contiguous())
    elif op == "move":
        counts = _moved(case)
        rng, src, dst, at = random.Random(seed), [], [], 0
        room = max(counts, default=0) * 2 if not case["draft"] else case["draft"] + page       # tokens that a sequence's pages hold
        per = -(-room // page)
        pages = per * len(counts) * (1 if case["draft"] else 2) + 1
        order = list(range(pages))
        rng.shuffle(order)
        slot = lambda first, i: order[first + i // page] * page + i % page  # noqa: E731
        for g, n in enumerate(counts):
            if case["draft"]:                                             # an accepted path off the first branch: to the places of the first drafted tokens
                base = rng.randrange(page)
                path = sorted(rng.sample(range(n, case["draft"]), min(n, case["draft"] - n)))
                src += [slot(g * per, base + i) for i in path]
                dst += [slot(g * per, base + i) for i in range(len(path))]
            else:
                kept = sorted(rng.sample(range(2 * n), n))
                src += [slot(g * per, i) for i in kept]
                dst += [slot((len(counts) + g) * per, i) for i in range(n)]
        starts = [sum(counts[:g]) for g in range(len(counts) + 1)]
        state.update(_pools(case, pages, gen, heads, case["layers"]))
        state.update(src=torch.tensor(src, dtype=torch.int64, device="cuda"), dst=torch.tensor(dst, dtype=torch.int64, device="cuda"),
                     starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), most=max(counts, default=0))
    else:
        kv, new = _lengths(case)
        need = [-(-n // page) for n in kv]
        order = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
        state.update(_pools(case, sum(need) + 3, gen, heads))
        table = torch.full((len(kv), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
        toward, at, slots = torch.randn((heads, dim), generator=gen, device="cuda"), 0, []
        for b, n in enumerate(kv):
            table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            i = torch.arange(n, device="cuda")
            slots.append(table[b].long()[i // page] * page + i % page)
            for j in range(0, n, 65536):
                part = slots[-1][j:j + 65536]
                for name, bits in (("k", case["kb"]), ("v", case["vb"])):
                    x = _activations(gen, part.numel(), heads, dim)
                    if j == 0 and name == "k":
                        x[:4] += 2.0 * toward                             # the first keys answer to the queries' common direction
                    _store(state, name, part, *_quantise(x, bits))
        q = torch.randn((sum(new), heads, case["group"], dim), generator=gen, device="cuda") * 1.5 + 0.5 * toward.unsqueeze(1)
        ints = dict(dtype=torch.int32, device="cuda")
        state.update(q=q.reshape(sum(new), heads * case["group"], dim).to(DTYPES[case["dtype"]]), table=table, kv_lens=torch.tensor(kv, **ints),
                     q_starts=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], **ints), max_q=max(new), max_kv=max(kv),
                     parents=torch.tensor([p for t in _parents(new) for p in t], **ints), slots=slots, bits=(case["kb"], case["vb"]),
                     softmax_scale=1.0 / math.sqrt(dim), window=case["window"] or None, sinks=case["sinks"], lse=case["lse"])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    kept = state.get("kept")
    if kept is None:                                      # the handles that a program makes once
        package = os.path.abspath("var-q_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from VAR_Q import paged, rotary
        case, kept = state["case"], {}
        if state["op"] in ("rotate", "put"):
            kept["rotary"] = rotary.Rotary(state["dim"], base=10000.0, sections=_sections(case), interleaved=case["interleaved"], restart=case["restart"],
                                           rotary_dim=state["rotary"])
        if state["op"] != "rotate":
            names = ("k_codes", "v_codes", "k_scale", "v_scale")
            if state["op"] in ("copy", "move"):
                kept["caches"] = [paged.PagedCache.over(*(state[n][i] for n in names), state["dim"]) for i in range(case["layers"])]
            else:
                kept["cache"] = paged.PagedCache.over(*(state[n] for n in names), state["dim"])
        kept["paged"] = paged
        state["kept"] = kept
    op, paged = state["op"], kept["paged"]
    if op in ("rotate", "put"):
        norm = state["case"]["norm"]
        how = dict(norm=None if norm == "none" else norm, q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS.get(norm))
        if op == "rotate":
            return kept["rotary"].rotate(state["q"], state["k"], state["positions"], **how)
        q = kept["cache"].append_rotated(state["q"], state["k"], state["v"], state["slots"], kept["rotary"], state["positions"], **how)
        return q, *kept["cache"].read(state["slots"], state["dtype"])
    if op == "tree":
        masks, positions = paged.draft_tree(state["parents"], state["kv_lens"], state["q_starts"], state["max_q"])
        out = kept["cache"].attend(state["q"], state["table"], state["kv_lens"], state["q_starts"], state["max_q"], state["max_kv"], state["softmax_scale"],
                                   window=state["window"], sinks=state["sinks"], return_lse=state["lse"], tree=masks)
        return masks, positions, out
    if op == "copy":
        paged.copy_pages(kept["caches"], state["src"], state["dst"])
    else:
        paged.move_tokens(kept["caches"], state["src"], state["dst"], state["starts"], state["most"])
    return state["k_codes"], state["v_codes"], state["k_scale"], state["v_scale"]


def _run_plain(state):
    op = state["op"]
    if op == "rotate":
        return tuple(_plain_rotate(state, state[n], state[n + "_weight"]).to(state["dtype"]) for n in ("q", "k"))
    if op == "put":
        q, k = (_plain_rotate(state, state[n], state[n + "_weight"]) for n in ("q", "k"))
        _store(state, "k", state["slots"], *_quantise(k, state["bits"][0]))
        _store(state, "v", state["slots"], *_quantise(state["v"].float(), state["bits"][1]))
        return q.to(state["dtype"]), _plain_read(state, "k", state["bits"][0]), _plain_read(state, "v", state["bits"][1])
    if op == "tree":
        masks, positions, seen = _plain_masks(state)
        return masks, positions, _plain_attend(state, positions, seen)
    names = ("k_codes", "v_codes", "k_scale", "v_scale")
    if op == "copy":
        return tuple(state[n].index_copy_(1, state["dst"], state[n][:, state["src"]]) for n in names)
    page, src, dst = state["page"], state["src"], state["dst"]
    layer, head = (torch.arange(n, device=src.device) for n in state["k_codes"].shape[0:3:2])
    at = lambda slots: (layer.view(-1, 1, 1), (slots // page).view(1, -1, 1), head.view(1, 1, -1), (slots % page).view(1, -1, 1))  # noqa: E731
    return tuple(state[n].index_put_(at(dst), state[n][at(src)]) for n in names)       # everything is read before anything is written


def _plain_rotate(state, x, weight):
    """x [..., tokens, heads, dim] -> fp32: norm, factors, rotation"""
    case, rotary = state["case"], state["rotary"]
    x = x.float()
    if case["norm"] == "l2":
        x = x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(EPS["l2"])
    elif case["norm"] == "rms":
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS["rms"])
    if weight is not None:
        x = x * weight
    i = torch.arange(rotary // 2, device=x.device)
    sizes = torch.tensor(_sections(case), device=x.device)
    axis = torch.repeat_interleave(torch.arange(len(sizes), device=x.device), sizes)
    per = (sizes * 2)[axis] if case["restart"] else rotary                # dimensions over which the frequencies fall
    if case["restart"]:
        i = i - (sizes.cumsum(0) - sizes)[axis]
    freq = 10000.0 ** (-(2.0 * i.double()) / per)
    angle = state["positions"].double()[axis].T * freq                   # [tokens, pairs]
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    turned, rest = x[..., :rotary], x[..., rotary:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def _plain_read(state, name, bits):
    slots, page = state["slots"], state["page"]
    where, at = slots // page, slots % page
    return (_unpack(state[name + "_codes"][where, :, at], bits).float() * state[name + "_scale"][where, :, at].unsqueeze(-1)).to(state["dtype"])


def _plain_masks(state):
    """Masks [tokens, words] of 32 drafted tokens a word, positions [tokens], and what is seen [B, most, most]"""
    parents, starts, most = state["parents"].long(), state["q_starts"].long(), state["max_q"]
    batch, dev = starts.numel() - 1, parents.device
    token = torch.arange(parents.numel(), device=dev)
    b = (token.unsqueeze(1) >= starts[1:]).sum(1)
    at = token - starts[b]
    reach = torch.zeros((batch, most, most + 1), device=dev)
    reach[b, at, torch.where(parents < 0, most, parents)] = 1.0           # the last column: the context
    reach = reach[:, :, :most] + torch.eye(most, device=dev)
    for _ in range((most - 1).bit_length()):                              # ancestors twice as far away with every product
        reach = torch.matmul(reach, reach).clamp_max(1.0)
    words = -(-most // 32)
    seen = reach > 0
    bits = torch.zeros((batch, most, words * 32), dtype=torch.int64, device=dev)
    bits[:, :, :most] = seen
    packed = (bits.view(batch, most, words, 32) << torch.arange(32, device=dev)).sum(-1)
    packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
    context = state["kv_lens"].long() - (starts[1:] - starts[:-1])
    depth = seen.sum(-1) - 1
    return packed[b, at], (context[b] + depth[b, at]).to(torch.int32), seen


def _dense(state, name, bits):
    """K or V of all sequences [B, H, L, dim] in fp32, zero behind a sequence's end"""
    table = state["table"].long().clamp_min(0)
    x = _unpack(state[name + "_codes"][table], bits).float() * state[name + "_scale"][table].unsqueeze(-1)
    x = x.permute(0, 2, 1, 3, 4).flatten(2, 3)                                          # [B, H, L, dim]
    there = torch.arange(x.shape[2], device=x.device) < state["kv_lens"].unsqueeze(1)
    return torch.where(there.view(len(table), 1, -1, 1), x, 0.0)


def _plain_attend(state, positions, drafted):
    q, starts, kv_lens, most = state["q"], state["q_starts"].long(), state["kv_lens"].long(), state["max_q"]
    k = _dense(state, "k", state["bits"][0])
    batch, heads, length, dim = k.shape
    group, dev = q.shape[1] // heads, q.device
    counts = starts[1:] - starts[:-1]
    i = torch.arange(most, device=dev)
    rows = (starts[:-1].unsqueeze(1) + i).clamp_max(q.shape[0] - 1)                      # [B, most]
    qd = q[rows].float().view(batch, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim)
    s = torch.matmul(qd, k.transpose(2, 3)).view(batch, heads, group, most, length)
    s = s.mul_(state["softmax_scale"])
    del k
    j = torch.arange(length, device=dev)
    context = (kv_lens - counts).view(batch, 1, 1)
    seen = (j < context).expand(batch, most, length)
    if state["window"]:
        seen = seen & ((positions.long()[rows].unsqueeze(2) - j < state["window"]) | (j < state["sinks"]))
    at = (j - context).expand(batch, most, length)                                       # which drafted token a key is
    seen = seen | ((at >= 0) & (at < counts.view(batch, 1, 1)) & drafted.gather(2, at.clamp(0, most - 1)))
    s = s.masked_fill_(~(seen & (i < counts.unsqueeze(1)).unsqueeze(2)).view(batch, 1, 1, most, length), -math.inf)
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
    op, dim = case["op"], case["dim"]

    def turned(name):
        x, rot, sizes = state[name].double(), state["rotary"], _sections(case)
        if case["norm"] == "l2":
            x = x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp(min=EPS["l2"])
        if case["norm"] == "rms":
            x = x / ((x * x).sum(-1, keepdim=True) / dim + EPS["rms"]).sqrt()
        if state[name + "_weight"] is not None:
            x = x * state[name + "_weight"].double()
        y = x.clone()
        pair = 0
        for axis, size in enumerate(sizes):
            for i in range(size):
                f = 10000.0 ** (-2.0 * i / (2 * size)) if case["restart"] else 10000.0 ** (-2.0 * pair / rot)
                angle = (state["positions"][axis].double() * f).view(-1, 1)
                a, b = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + rot // 2)
                y[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
                y[..., b] = x[..., a] * angle.sin() + x[..., b] * angle.cos()
                pair += 1
        return y

    def rounded(x, bits):                      # the values that a row's codes stand for
        scale = (x.abs().max(-1, keepdim=True).values / (2 ** (bits - 1) - 1)).clamp(min=1e-12)
        return (x / scale).round().clamp(-2 ** (bits - 1), 2 ** (bits - 1) - 1) * scale

    def held(name, bits, slots):               # [tokens, heads, dim] of the pools
        w = state[name + "_codes"].transpose(1, 2).reshape(-1, case["heads"], dim * bits // 32)[slots].to(torch.int64) & 0xffffffff
        x = torch.stack([(w >> (bits * f)) % 2 ** bits for f in range(32 // bits)], -1).reshape(len(slots), case["heads"], dim)
        x = torch.where(x >= 2 ** (bits - 1), x - 2 ** bits, x)
        return x.double() * state[name + "_scale"].transpose(1, 2).reshape(-1, case["heads"], 1)[slots].double()

    if op == "rotate":
        return turned("q"), turned("k")
    if op == "put":
        return turned("q"), rounded(turned("k"), case["kb"]), rounded(state["v"].double(), case["vb"])
    if op == "copy":
        for n in ("k_codes", "v_codes", "k_scale", "v_scale"):
            for a, b in zip(state["src"].tolist(), state["dst"].tolist()):
                state[n][:, b] = state[n][:, a]
        return state["k_codes"], state["v_codes"], state["k_scale"].double(), state["v_scale"].double()
    if op == "move":
        page, pools = state["page"], []
        for n in ("k_codes", "v_codes", "k_scale", "v_scale"):
            flat = state[n].transpose(2, 3).flatten(1, 2)                 # [layers, slots, heads, ...]
            flat[:, state["dst"]] = flat[:, state["src"]].clone()
            pools.append(flat.unflatten(1, (-1, page)).transpose(2, 3))
        return pools[0], pools[1], pools[2].double(), pools[3].double()
    kv, new = _lengths(case)
    masks, positions, outs, sums, group = [], [], [], [], case["group"]
    words = -(-max(new) // 32)
    for b, (n, c, parents) in enumerate(zip(kv, new, _parents(new))):
        own_path = []
        for i, p in enumerate(parents):
            own_path.append((own_path[p] if p >= 0 else []) + [i])
            bits = sum(1 << a for a in own_path[-1])
            masks.append([(w - (1 << 32) if w >= 1 << 31 else w) for w in ((bits >> (32 * z)) & 0xffffffff for z in range(words))])
            positions.append(n - c + len(own_path[-1]) - 1)
        k, v = held("k", case["kb"], state["slots"][b]), held("v", case["vb"], state["slots"][b])
        q = state["q"][sum(new[:b]):sum(new[:b + 1])].double()
        blind = torch.zeros((c, n), dtype=torch.bool)
        for i, path in enumerate(own_path):
            blind[i, n - c:] = True
            blind[i, [n - c + a for a in path]] = False
            if case["window"]:
                far = positions[sum(new[:b]) + i] - case["window"] + 1
                blind[i, min(case["sinks"], n - c):max(0, min(far, n - c))] = True
        blind = blind.to("cuda")
        out, lse = torch.zeros((c, case["heads"] * group, dim), dtype=torch.float64, device="cuda"), torch.zeros((c, case["heads"] * group), dtype=torch.float64, device="cuda")
        for h in range(case["heads"] * group):
            s = (q[:, h] @ k[:, h // group].T / math.sqrt(dim)).masked_fill(blind, -math.inf)
            lse[:, h] = s.logsumexp(-1)
            out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
        outs.append(out)
        sums.append(lse)
    masks = torch.tensor(masks, dtype=torch.int32, device="cuda").view(-1, words)
    positions = torch.tensor(positions, dtype=torch.int32, device="cuda")
    return masks, positions, (torch.cat(outs), torch.cat(sums)) if case["lse"] else torch.cat(outs)
