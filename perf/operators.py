"""Performance cases of the attention side of a serving step: queries and keys normalised and rotated into a paged cache,
the page tables and slots of that step, and the attention of the new tokens over the cache.

    own               False: the operators in plain torch, 32 bits; True: the package's own calls
    listed()          the cases
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call, from the seed
    run(state)        one pass
    work(case)        bytes and operations the pass cannot do without
    exact(case, s)    the same outputs in 64 bits

Kinds of case:
    attention  chunks of new tokens (one token each in a decode step) over a paged cache, causal, grouped queries
    rope       RMS norm of each query and key head, rotation by position, keys and values into their slots of the cache
               (without a cache: rotated queries and keys as tensors of their own)
    pages      pages for the new tokens of a batch from the list of free ones, and each token's position and slot

Layouts. Cache: [pages, KV heads, page size, head_dim], one tensor for keys and one for values. Page table: int32 [requests,
pages per request], -1 where there is none. qkv: [tokens, (heads + 2 KV heads) head_dim], a projection's output. Rotation
table: float32 [positions, head_dim], cosines then sines. Head counts are those of the models in perf/cases.py (32 / 8, 16 / 8 and 40 / 8
heads of 128) and generic ones of 64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

THETA = 1e6
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # interactive decode: one sequence, a short conversation
        {"name": "attn_decode_b1_1k", "op": "attention", "heads": 32, "kv": 8, "dim": 128, "dtype": "fp16", "page": 16,
         "batch": 1, "new": 1, "context": 1023, "ragged": False},
        # a serving batch in decode, sequences of all lengths up to 8k
        {"name": "attn_decode_b32_8k", "op": "attention", "heads": 32, "kv": 8, "dim": 128, "dtype": "fp16", "page": 16,
         "batch": 32, "new": 1, "context": 8191, "ragged": True},
        # few sequences with long contexts, an odd length
        {"name": "attn_decode_b3_40k", "op": "attention", "heads": 16, "kv": 8, "dim": 128, "dtype": "bf16", "page": 64,
         "batch": 3, "new": 1, "context": 40001, "ragged": False},
        # drafted tokens scored in one pass: five new tokens for each of a few requests
        {"name": "attn_verify_b9_5", "op": "attention", "heads": 40, "kv": 8, "dim": 128, "dtype": "fp16", "page": 32,
         "batch": 9, "new": 5, "context": 3000, "ragged": True},
        # chunked prefill: chunks of several requests at once, odd lengths
        {"name": "attn_chunk_b5_700", "op": "attention", "heads": 40, "kv": 8, "dim": 128, "dtype": "bf16", "page": 16,
         "batch": 5, "new": 700, "context": 5000, "ragged": True},
        # a whole long prompt at once
        {"name": "attn_prompt_8k", "op": "attention", "heads": 32, "kv": 8, "dim": 128, "dtype": "fp16", "page": 16,
         "batch": 1, "new": 8192, "context": 0, "ragged": False},
        # the token of one sequence in a decode step
        {"name": "rope_decode_b1", "op": "rope", "heads": 32, "kv": 8, "dim": 128, "dtype": "fp16", "page": 16, "tokens": 1,
         "norm": True, "cache": True},
        # an odd prompt of a model without head norms, heads of 64, keys kept dense
        {"name": "rope_dense_509", "op": "rope", "heads": 32, "kv": 8, "dim": 64, "dtype": "bf16", "page": 16, "tokens": 509,
         "norm": False, "cache": False},
        # a long prompt chunk into the cache
        {"name": "rope_prompt_8k", "op": "rope", "heads": 32, "kv": 8, "dim": 128, "dtype": "fp16", "page": 16, "tokens": 8192,
         "norm": True, "cache": True},
        # one sequence, one token
        {"name": "pages_b1", "op": "pages", "page": 16, "batch": 1, "new": 1, "context": 999, "ragged": False},
        # a large decode batch
        {"name": "pages_decode_b256", "op": "pages", "page": 16, "batch": 256, "new": 1, "context": 4095, "ragged": True},
        # chunks of many requests in one step
        {"name": "pages_prompts_b64", "op": "pages", "page": 16, "batch": 64, "new": 700, "context": 2000, "ragged": True},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng) -> dict:
    op = rng.choice(("attention", "attention", "attention", "rope", "pages"))
    if op == "pages":
        batch = _log(rng, 1, 512)
        return {"op": op, "page": rng.choice((16, 32, 64, 128)), "batch": batch,
                "new": 1 if rng.random() < 0.4 else _log(rng, 1, 20000 / batch), "context": _log(rng, 1, 8192),
                "ragged": rng.random() < 0.7}
    dim = rng.choice((128, 128, 64))
    heads, kv = rng.choice(((32, 8), (16, 8), (40, 8), (8, 8), (24, 2), (7, 1)))
    base = {"op": op, "heads": heads, "kv": kv, "dim": dim, "dtype": rng.choice(("fp16", "bf16")),
            "page": rng.choice((16, 32, 64, 128))}
    if op == "rope":
        return {**base, "tokens": _log(rng, 1, 6500), "norm": rng.random() < 0.7, "cache": rng.random() < 0.8}
    if rng.random() < 0.5:  # decode, or a few drafted tokens
        new, batch = rng.choice((1, 1, 1, rng.randint(2, 8))), _log(rng, 1, 64)
        context = _log(rng, 16, max(17, min(32768, 131072 // batch)))
    else:  # chunks
        new, batch = _log(rng, 9, 2048), _log(rng, 1, 6)
        context = rng.choice((0, _log(rng, 1, 8192)))
    while batch * new * (context + new) * heads > 2e9:
        batch, new = max(1, batch // 2), max(1, new * 3 // 4)
    return {**base, "batch": batch, "new": new, "context": context, "ragged": rng.random() < 0.6}


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens in the cache, new tokens) of each request: the case's largest, or spread below them with the largest among them."""
    b = case["batch"]
    if not case["ragged"]:
        return [case["context"]] * b, [case["new"]] * b
    rng = random.Random(b * 1000003 + case["new"] * 10007 + case["context"])
    context = [rng.randint(0, case["context"]) for _ in range(b)]
    new = [rng.randint(1, case["new"]) for _ in range(b)]
    context[rng.randrange(b)], new[rng.randrange(b)] = case["context"], case["new"]
    return context, new


def _pages(tokens: int, page: int) -> int:
    return -(-tokens // page)


# ---------------------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _int32(values: list[int]) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(new: list[int]) -> torch.Tensor:
    return _int32([sum(new[:i]) for i in range(len(new) + 1)])


def _table(counts: list[int], width: int, pool: torch.Tensor) -> torch.Tensor:
    """[requests, width] int32: each request's pages from `pool` in turn, -1 behind them."""
    n = _int32(counts)
    col = torch.arange(width, device="cuda")
    first = (torch.cumsum(n, 0) - n)[:, None] + col
    return torch.where(col < n[:, None], pool[first.clamp(max=pool.numel() - 1)], -1).to(torch.int32)


def _randn(g: torch.Generator, dtype: str, *shape: int) -> torch.Tensor:
    return torch.randn(shape, device="cuda", dtype=DTYPES[dtype], generator=g)


def _perm(n: int, g: torch.Generator) -> torch.Tensor:
    return torch.randperm(n, device="cuda", generator=g).to(torch.int32)


def _angles(positions: torch.Tensor, dim: int) -> torch.Tensor:
    """float64 [..., dim / 2]: position times theta^(-2 i / dim)."""
    i = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    return positions.double()[..., None] * THETA ** (-2.0 * i / dim)


def prepare(case: dict, seed: int) -> dict:
    g, op = _gen(seed), case["op"]
    if op == "rope":
        t, h, kv, d, page = case["tokens"], case["heads"], case["kv"], case["dim"], case["page"]
        state = {"op": op, "heads": h, "kv": kv, "qkv": _randn(g, case["dtype"], t, (h + 2 * kv) * d)}
        # a few sequences of the batch, somewhere in their contexts
        first = torch.randint(0, 20000, (1,), device="cuda", generator=g)
        state["positions"] = ((first + torch.arange(t, device="cuda")) % 20000).to(torch.int32)
        a = _angles(torch.arange(20000, device="cuda"), d)
        state["table"] = torch.cat([a.cos(), a.sin()], dim=-1).float()
        for name in ("q_weight", "k_weight"):
            w = (1.0 + 0.2 * (torch.rand(d, device="cuda", generator=g) - 0.5)).to(DTYPES[case["dtype"]])
            state[name] = w if case["norm"] else None
        if case["cache"]:
            n = _pages(t, page) + 3
            state["k_cache"], state["v_cache"] = (_randn(g, case["dtype"], n, kv, page, d) for _ in range(2))
            at = torch.arange(t, device="cuda")
            state["slots"] = (_perm(n, g)[at // page] * page + at % page).to(torch.int32)
        return state
    context, new = _lengths(case)
    page, total = case["page"], sum(new)
    have = [_pages(c, page) for c in context]
    need = [_pages(c + n, page) for c, n in zip(context, new)]
    state = {"op": op, "page": page, "tokens": total}
    if op == "pages":
        held = sum(have)
        pool = _perm(sum(need) + 64, g)
        state["context_lens"], state["query_lens"] = _int32(context), _int32(new)
        state["page_table"] = _table(have, max(need) + 1, pool[:max(1, held)])
        state["free_pages"] = torch.cat([pool[:5], pool[held:]])  # five taken by an earlier step
        state["taken"] = _int32([5])
        return state
    h, kv, d = case["heads"], case["kv"], case["dim"]
    pool = _perm(sum(need) + 2, g)
    state["q"] = _randn(g, case["dtype"], total, h, d)
    state["k_cache"], state["v_cache"] = (_randn(g, case["dtype"], pool.numel(), kv, page, d) for _ in range(2))
    state["page_table"] = _table(need, max(need), pool)
    state["seq_lens"] = _int32([c + n for c, n in zip(context, new)])
    state["query_start"] = None if max(new) == 1 else _starts(new)
    state["max_query_len"], state["max_seq_len"] = max(new), max(c + n for c, n in zip(context, new))
    return state


# ------------------------------------------------------------------------------------- plain forms
def _requests(starts: torch.Tensor, tokens: int) -> torch.Tensor:
    """The request of each token."""
    at = torch.arange(tokens, device="cuda")
    return torch.searchsorted(starts[1:].contiguous(), at, right=True).clamp(max=starts.numel() - 2)


def _plain_attention(s: dict) -> torch.Tensor:
    q, table, page = s["q"], s["page_table"], s["page"]
    t, h, d = q.shape
    b, kv = table.shape[0], s["k_cache"].shape[1]
    n_max, l_max, group = s["max_query_len"], s["max_seq_len"], h // s["k_cache"].shape[1]
    starts = torch.arange(b + 1, device="cuda") if s["query_start"] is None else s["query_start"].long()
    pages = table[:, :_pages(l_max, page)].long().clamp(min=0)
    keys, values = (c[pages].float().permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)[:, :, :l_max]
                    for c in (s["k_cache"], s["v_cache"]))
    token = (starts[:-1, None] + torch.arange(n_max, device="cuda")).clamp(max=t - 1)  # [b, n_max]
    rows = q.float()[token].view(b, n_max, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, group * n_max, d)
    scores = torch.matmul(rows, keys.transpose(2, 3)).view(b, kv, group, n_max, l_max) * d ** -0.5
    lens, new = s["seq_lens"].long(), starts[1:] - starts[:-1]
    last = (lens - new)[:, None] + torch.arange(n_max, device="cuda")  # the last key each new token sees
    seen = torch.arange(l_max, device="cuda") <= last[:, :, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, kv, group * n_max, l_max), values).view(b, kv, group, n_max, d)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n_max, h, d)
    r = _requests(starts, t)
    return out[r, torch.arange(t, device="cuda") - starts[r]].to(q.dtype)


def _plain_rope(s: dict):
    qkv, heads, kv = s["qkv"], s["heads"], s["kv"]
    t, d = qkv.shape[0], s["table"].shape[1]
    x = qkv.float().view(t, heads + 2 * kv, d)
    cos, sin = s["table"][s["positions"].long()][:, None].chunk(2, dim=-1)

    def rotated(y, weight):
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = y.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(qkv.dtype)

    q, k = rotated(x[:, :heads], s["q_weight"]), rotated(x[:, heads:heads + kv], s["k_weight"])
    if "slots" not in s:
        return q, k
    page = s["k_cache"].shape[2]
    slots = s["slots"].long()
    s["k_cache"][slots // page, :, slots % page] = k
    s["v_cache"][slots // page, :, slots % page] = x[:, heads + kv:].to(qkv.dtype)
    return q, s["k_cache"], s["v_cache"]


def _plain_pages(s: dict):
    context, new, table, page, tokens = s["context_lens"].long(), s["query_lens"].long(), s["page_table"], s["page"], s["tokens"]
    lens = context + new
    starts = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    have = (context + page - 1) // page
    need = (lens + page - 1) // page - have
    first = s["taken"].long() + torch.cumsum(need, 0) - need
    r = _requests(starts, tokens)
    positions = context[r] + torch.arange(tokens, device="cuda") - starts[r]
    at = positions // page
    fresh = s["free_pages"][(first[r] + at - have[r]).clamp(0, s["free_pages"].numel() - 1)]
    table[r, at] = torch.where(at >= have[r], fresh, table[r, at])
    slots = table[r, at] * page + positions % page
    taken = s["taken"] + need.sum()
    counts = torch.stack([starts[-1], need.sum(), torch.zeros_like(starts[-1]), torch.zeros_like(starts[-1])])
    return [x.to(torch.int32) for x in (table, starts, lens, positions, slots, taken, counts)]


@torch.no_grad()
def run(state: dict):
    op = state["op"]
    if not own:
        return {"attention": _plain_attention, "rope": _plain_rope, "pages": _plain_pages}[op](state)
    if op == "attention":
        from tandem_amd.layers.paged_attention import paged_attention

        return paged_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["seq_lens"],
                               state["query_start"], max_query_len=state["max_query_len"], max_seq_len=state["max_seq_len"])
    if op == "rope":
        from tandem_amd.layers import rotary

        args = (state["qkv"], state["positions"], state["table"], state["heads"], state["kv"])
        norms = {"q_weight": state["q_weight"], "k_weight": state["k_weight"], "eps": EPS}
        if "slots" not in state:
            return rotary.norm_rope(*args, **norms)
        q = rotary.norm_rope_cache(*args, state["k_cache"], state["v_cache"], state["slots"], **norms)
        return q, state["k_cache"], state["v_cache"]
    from tandem_amd.kv_cache import plan_pages

    plan = plan_pages(state["context_lens"], state["query_lens"], state["page_table"], state["free_pages"], state["taken"],
                      state["page"], state["tokens"])
    return [state["page_table"], plan.query_start, plan.seq_lens, plan.positions, plan.slots, plan.taken, plan.counts]


# ------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    op = case["op"]
    if op == "rope":
        t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
        moved = h + 2 * kv if case["cache"] else h + kv  # heads read and written once: values for the cache only
        return {"bytes": 2 * 2 * t * moved * d + t * (4 * d + 8), "flops": t * d * (h + kv) * (7.0 if case["norm"] else 3.0)}
    context, new = _lengths(case)
    if op == "pages":
        page, total = case["page"], sum(new)
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(context, new))
        # lengths in; starts and lengths out; a position and a slot for each token; each new page read from the list and put
        # into the table; each request's last page so far read
        return {"bytes": 4 * (5 * case["batch"] + 2 * total + 2 * need), "flops": 0}
    h, kv, d = case["heads"], case["kv"], case["dim"]
    keys = sum(c + n for c, n in zip(context, new))
    seen = sum(n * c + n * (n + 1) / 2 for c, n in zip(context, new))  # pairs of a new token and a key it sees
    return {"bytes": 2 * 2 * keys * kv * d + 2 * 2 * sum(new) * h * d + 4 * keys / case["page"], "flops": 4.0 * seen * h * d}


# --------------------------------------------------------------------------------- 64-bit results
def _exact_attention(case: dict, s: dict) -> torch.Tensor:
    context, new = _lengths(case)
    page, kv, d = case["page"], case["kv"], case["dim"]
    group = case["heads"] // kv
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (c, n) in enumerate(zip(context, new)):
        pages = s["page_table"][i, :_pages(c + n, page)].long()
        hidden = torch.ones(n, c + n, dtype=torch.bool, device="cuda").triu(c + 1)
        for j in range(kv):
            k, v = (x[pages, j].reshape(-1, d)[:c + n].double() for x in (s["k_cache"], s["v_cache"]))
            for head in range(j * group, (j + 1) * group):
                w = s["q"][at:at + n, head].double() @ k.t() / math.sqrt(d)
                out[at:at + n, head] = torch.softmax(w.masked_fill(hidden, -math.inf), dim=1) @ v
        at += n
    return out


def _exact_rope(case: dict, s: dict):
    t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
    a = _angles(s["positions"], d)
    turn = torch.polar(torch.ones_like(a), a)[:, None]  # a head's values i and i + d / 2 are one complex number
    x = s["qkv"].double().view(t, h + 2 * kv, d)

    def turned(y, weight):
        if weight is not None:
            y = y / ((y ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], dim=-1)

    q, k = turned(x[:, :h], s["q_weight"]), turned(x[:, h:h + kv], s["k_weight"])
    if not case["cache"]:
        return q, k
    outs = [q]
    for cache, rows in ((s["k_cache"], k), (s["v_cache"], x[:, h + kv:])):
        flat = cache.double().transpose(1, 2).reshape(-1, kv, d)
        flat[s["slots"].long()] = rows
        outs.append(flat.view(-1, case["page"], kv, d).transpose(1, 2).contiguous())
    return tuple(outs)


@torch.no_grad()
def exact(case: dict, seed: int):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    return _exact_attention(case, s) if case["op"] == "attention" else _exact_rope(case, s)
