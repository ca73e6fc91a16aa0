"""The operators of a paged key-value cache, as cases that can be timed and compared.

Several sequences share two pools of pages, keys and values, [pages, kv heads, page size, head dim]; a table names the
pages of every sequence, `lens` its length with the tokens of the call.  The operations ("op"):

  append   rows of a fused q/k/v product: queries and keys rotated to their positions, keys and values into the pages
  token    attention of one new token of every sequence over all of its pages
  prompt   causal attention of several new tokens of every sequence, packed one behind the other, over its pages: whole
           prompts, or pieces of prompts whose beginnings are in the pages already

`run` computes them with elementary torch operations in 32 bits or, with `own`, through lazyweights_b200.PagedCache.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, heads, kv_heads, head_dim, page, dtype, seqs, context, new, **more):
    """context, new: (least, most) tokens in the pages before the call, and of the call, per sequence."""
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, seqs=seqs, context_lo=context[0],
                context_hi=context[1], new_lo=new[0], new_hi=new[1], idle=0, window=0, rows="fp32", inner_heads=False, mix=1)
    case.update(more)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # batch-1 decoding, a 7B-class decoder with grouped heads: the rows of one product into the cache
        _case("append_one", "append", 32, 8, 128, 16, "fp16", 1, (2047, 2047), (1, 1)),
        # one decoding step of a batch of an odd size, some of its slots idle, bf16 products
        _case("append_batch", "append", 32, 8, 128, 64, "bf16", 131, (1, 4000), (1, 1), rows="bf16", idle=7),
        # packed prompts as the decoder runtime has them: fp32 rows of a fused product
        _case("append_prompts", "append", 32, 8, 128, 16, "fp16", 24, (0, 0), (60, 2000)),
        # batch-1 decoding at a context of 2048
        _case("token_one", "token", 32, 8, 128, 16, "fp16", 1, (2047, 2047), (1, 1)),
        # a decoding batch of sequences of very different lengths
        _case("token_batch", "token", 32, 8, 128, 16, "fp16", 64, (100, 16000), (1, 1), idle=3),
        # every query head with keys of its own, 96 dimensions, larger pages, heads inside the positions of a page
        _case("token_heads", "token", 32, 32, 96, 64, "bf16", 33, (30, 4000), (1, 1), inner_heads=True),
        # two very long contexts: few rows, the work has to be split over the length
        _case("token_long", "token", 32, 8, 128, 32, "bf16", 2, (100000, 131071), (1, 1)),
        # verification of drafted tokens, at the size of the framework's own verification passes
        _case("prompt_verify", "prompt", 32, 32, 96, 16, "fp16", 1, (1000, 1000), (8, 8)),
        # a step of a serving loop: prompts of ragged lengths, packed
        _case("prompt_packed", "prompt", 32, 8, 128, 16, "fp16", 24, (0, 0), (20, 2500)),
        # a piece of a long prompt whose beginning is in the pages
        _case("prompt_piece", "prompt", 32, 8, 128, 32, "bf16", 1, (32000, 32000), (509, 509)),
        # a sliding window over prompts of a few thousand tokens
        _case("prompt_window", "prompt", 32, 8, 128, 64, "bf16", 3, (0, 0), (5000, 8000), window=2048),
        # one long prompt
        _case("prompt_long", "prompt", 32, 8, 128, 16, "fp16", 1, (0, 0), (16384, 16384)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("append", "token", "prompt")}
    while True:
        op = rng.choices(("append", "token", "prompt"), (3, 4, 5))[0]
        kv_heads, head_dim = rng.choice((1, 2, 4, 8, 8, 16, 32)), rng.choice((64, 96, 128, 128, 128, 40, 80))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 7, 8, 16))
        page = rng.choice((8, 16, 16, 24, 32, 64, 128, 256))
        if heads > 64 or heads * head_dim > 8192:
            continue
        seqs = _log(rng, 1, 256) if op != "prompt" else _log(rng, 1, 64)
        lo = _log(rng, 1, 65536 if op == "token" else 16384)
        if op == "prompt" or (op == "append" and rng.random() < 0.4):
            new = sorted((_log(rng, 1, 8192), _log(rng, 1, 8192)))
            context = (0, 0) if rng.random() < 0.6 else sorted((lo, _log(rng, lo, 20000)))
        else:
            new, context = (1, 1), (lo, _log(rng, lo, 131071 if op == "token" else 20000))
        case = _case(None, op, heads, kv_heads, head_dim, page, rng.choice(("fp16", "bf16")), seqs, context, new,
                     idle=rng.randint(0, seqs // 8), rows=rng.choice(("fp32", "fp16", "bf16")), inner_heads=rng.random() < 0.3,
                     window=_log(rng, 64, 8192) if op != "append" and rng.random() < 0.25 else 0, mix=rng.randint(1, 1 << 30))
        if sum(n for _, n in _lengths(case)) and _cost(case) <= most[op] and max(_lengths(case))[0] <= 131072:
            return case


# ------------------------------------------------------------------------------------------------------- the sizes


def _lengths(case):
    """(length with the new tokens, new tokens) of every sequence; idle slots of the batch have neither."""
    rng = random.Random(case["mix"])
    out = []
    for i in range(case["seqs"]):
        context = _log(rng, case["context_lo"], case["context_hi"]) if case["context_hi"] else 0
        new = _log(rng, case["new_lo"], case["new_hi"])
        out.append((context + new, new))
    for i in rng.sample(range(case["seqs"]), case["idle"]):
        out[i] = (0, 0)
    return out


def _seen(case, length, new):
    """Positions that the new tokens of one sequence see, added up, and positions that any of them sees."""
    w = case["window"] or length
    first = length - new
    ramp = max(0, min(length, w) - first)         # tokens whose range still starts at 0
    total = ramp * (2 * first + ramp + 1) // 2 + (new - ramp) * w
    return total, length - max(0, first + 1 - w)


def work(case):
    size, h, hk, dh = 2, case["heads"], case["kv_heads"], case["head_dim"]
    lens = [(n, m) for n, m in _lengths(case) if m]
    tokens = sum(m for _, m in lens)
    if case["op"] == "append":
        wide = 4 if case["rows"] == "fp32" else 2
        return {"bytes": tokens * ((h + 2 * hk) * dh * (wide + size) + dh * 4), "flops": tokens * (h + hk) * dh * 3}
    total = sum(_seen(case, n, m)[0] for n, m in lens)
    read = sum(_seen(case, n, m)[1] for n, m in lens)
    return {"bytes": 2 * read * hk * dh * size + 2 * tokens * h * dh * size, "flops": 4 * total * h * dh}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15) * 1e6 + 1e-3 * case["seqs"]


# ------------------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h, hk, dh, page, dtype = case["heads"], case["kv_heads"], case["head_dim"], case["page"], TYPES[case["dtype"]]
    lens = _lengths(case)
    counts = [-(-n // page) for n, _ in lens]
    pages, width = sum(counts) + 3, max(counts) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    host = order.cpu()
    for i, c in enumerate(counts):
        table[i, :c] = host[at:at + c]
        at += c
    starts = [0]
    for _, m in lens:
        starts.append(starts[-1] + m)

    def pool():
        shape = (pages, page, hk, dh) if case["inner_heads"] else (pages, hk, page, dh)
        p = torch.randn(shape, device="cuda", generator=gen, dtype=dtype)
        return p.transpose(1, 2) if case["inner_heads"] else p

    st = dict(case=case, k=pool(), v=pool(), table=table.cuda(), lens=torch.tensor([n for n, _ in lens], dtype=torch.int32).cuda(),
              starts=torch.tensor(starts, dtype=torch.int32).cuda(), host_lens=lens, host_starts=starts, host_table=table)
    one = case["op"] == "token" or (case["op"] == "append" and case["new_hi"] == 1)
    st["one"] = one                                    # a row per slot of the batch, idle slots too
    rows = len(lens) if one else starts[-1]
    if case["op"] == "append":
        st["qkv"] = torch.randn((rows, (h + 2 * hk) * dh), device="cuda", generator=gen).to(TYPES[case["rows"]])
        top = max(n for n, _ in lens)
        inv = 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64, device="cuda") / dh)
        angle = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * inv[None]
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["q"] = torch.zeros((rows, h, dh), device="cuda", dtype=dtype)
    else:
        st["q"] = torch.randn((rows, h, dh), device="cuda", generator=gen).to(dtype)
        st["out"] = torch.zeros_like(st["q"])
    if own:
        import lazyweights_b200 as lw
        st["cache"] = lw.PagedCache(st["k"], st["v"])
    return st


# ------------------------------------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        cache = state["cache"]
        where = (state["table"], state["lens"])
        if op == "append":
            cache.append(state["qkv"], state["case"]["heads"], state["cos"], state["sin"], *where,
                         starts=None if state["one"] else state["starts"], q=state["q"])
            return [state["q"], state["k"], state["v"]]
        if op == "token":
            return cache.attend(state["q"], *where, window=state["case"]["window"], out=state["out"])
        return cache.attend_prompt(state["q"], *where, state["starts"], window=state["case"]["window"], out=state["out"])
    return _append(state) if op == "append" else _attend(state)


def _append(state):
    """Rows to positions, a rotation in 32 bits, one rounding."""
    case, lens, starts = state["case"], state["lens"].long(), state["starts"].long()
    h, hk, dh, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if state["one"]:
        seq = torch.nonzero(lens > 0)[:, 0]
        row, pos = seq, lens[seq] - 1
    else:
        row = torch.arange(state["qkv"].shape[0], device="cuda")
        seq = (row[:, None] >= starts[None, 1:]).sum(1)
        pos = lens[seq] - (starts[seq + 1] - row)
    x = state["qkv"][row].float().view(-1, h + 2 * hk, dh)
    c, s = state["cos"][pos][:, None], state["sin"][pos][:, None]
    a, b = x[:, :h + hk, :dh // 2], x[:, :h + hk, dh // 2:]
    turned = torch.cat((a * c - b * s, b * c + a * s), 2).to(state["k"].dtype)
    state["q"][row] = turned[:, :h]
    where = state["table"][seq, pos // page].long()
    state["k"][where, :, pos % page] = turned[:, h:]
    state["v"][where, :, pos % page] = x[:, h + hk:].to(state["v"].dtype)
    return [state["q"], state["k"], state["v"]]


def _spans(state):
    """Per sequence: its rows of q, its length, its keys and values in 32 bits [kv heads, length, head dim]."""
    for i, (n, m) in enumerate(state["host_lens"]):
        if m:
            first = i if state["one"] else state["host_starts"][i]
            where = state["table"][i, :-(-n // state["case"]["page"])].long()
            kv = [state[p][where].transpose(0, 1).flatten(1, 2)[:, :n].float() for p in "kv"]
            yield slice(first, first + m), n, kv[0], kv[1]


def _attend(state):
    case = state["case"]
    h, hk, dh, out = case["heads"], case["kv_heads"], case["head_dim"], state["out"]
    for rows, n, k, v in _spans(state):
        q = state["q"][rows].float()
        m = q.shape[0]
        q = q.view(m, hk, h // hk, dh).permute(1, 2, 0, 3)              # [kv heads, group, tokens, head dim]
        step = max(1, (1 << 28) // (n * h))
        parts = []
        for t in range(0, m, step):
            pos = torch.arange(n - m + t, n - m + min(t + step, m), device="cuda")[:, None]
            at = torch.arange(n, device="cuda")[None]
            hidden = at > pos
            if case["window"]:
                hidden = hidden | (at <= pos - case["window"])
            part = q[:, :, t:t + step]
            s = part.flatten(1, 2) @ k.transpose(1, 2) * dh ** -0.5
            s = s.view(hk, h // hk, part.shape[2], n).masked_fill(hidden, -math.inf)
            e = torch.exp(s - s.amax(3, keepdim=True))
            total = e.sum(3, keepdim=True)
            parts.append((e.flatten(1, 2) @ v).view(hk, h // hk, part.shape[2], dh) / total)
        out[rows] = torch.cat(parts, 2).permute(2, 0, 1, 3).reshape(m, h, dh).to(out.dtype)
    return out


# --------------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_append(state) if case["op"] == "append" else _exact_attend(state)


def _exact_append(state):
    """Complex numbers: a pair (a, b) turned by the angle of its position."""
    case = state["case"]
    h, hk, dh, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    q, k, v = state["q"].double(), state["k"].double(), state["v"].double()
    for i, (n, m) in enumerate(state["host_lens"]):
        if not m:
            continue
        first = i if state["one"] else state["host_starts"][i]
        x = state["qkv"][first:first + m].double().view(m, h + 2 * hk, 2, dh // 2)
        turn = torch.complex(state["cos"][n - m:n].double(), state["sin"][n - m:n].double())
        z = torch.view_as_real(torch.complex(x[:, :, 0], x[:, :, 1]) * turn[:, None]).movedim(3, 2).reshape(m, h + 2 * hk, dh)
        q[first:first + m] = z[:, :h]
        slots = torch.tensor([int(state["host_table"][i, p // page]) * page + p % page for p in range(n - m, n)], device="cuda")
        k[slots // page, :, slots % page] = z[:, h:h + hk]
        v[slots // page, :, slots % page] = x[:, h + hk:].reshape(m, hk, dh)
    return [q, k, v]


def _exact_attend(state):
    """Query head by query head, block of queries by block of queries, over the positions that the block sees."""
    case = state["case"]
    h, hk, dh, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    for i, (n, m) in enumerate(state["host_lens"]):
        if not m:
            continue
        first = i if state["one"] else state["host_starts"][i]
        slots = [(state["table"][i].long()[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).reshape(-1)[:n]][0]
        keys = state["k"][slots // case["page"], :, slots % case["page"]].double()      # [length, kv heads, head dim]
        values = state["v"][slots // case["page"], :, slots % case["page"]].double()
        block = 2048
        for t in range(0, m, block):
            b = min(block, m - t)
            p0 = n - m + t
            lo, hi = (max(0, p0 - w + 1) if w else 0), p0 + b
            pos = torch.arange(p0, hi, device="cuda")[:, None]
            at = torch.arange(lo, hi, device="cuda")[None]
            seen = (at <= pos) if not w else (at <= pos) & (at > pos - w)
            for j in range(hk):
                g = h // hk
                x = state["q"][first + t:first + t + b, j * g:(j + 1) * g].double().transpose(0, 1)
                logits = torch.matmul(x, keys[lo:hi, j].t()) / math.sqrt(dh)
                logits = torch.where(seen, logits, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
                p = (logits - torch.logsumexp(logits, 2, keepdim=True)).exp()
                out[first + t:first + t + b, j * g:(j + 1) * g] = torch.matmul(p, values[lo:hi, j]).transpose(0, 1)
    return out
