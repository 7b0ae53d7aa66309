"""Performance cases of projections in 8-bit integers: weights with a scale for each output channel, activations with a scale for
each token, and the operators that write such activations.

    own               False: the operators in plain torch; True: the package's own calls
    listed()          the cases
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call, from the seed
    run(state)        one pass
    work(case)        bytes and operations the pass cannot do without
    exact(case, s)    the same outputs in 64 bits

Kinds of case:
    norm      RMS norm of each token (after adding the residual, which becomes the sum), its output in 8 bits
    quantize  rows of activations in 8 bits (what a projection without a norm before it reads)
    linear    a projection: codes of activations times codes of weights, both scales in the epilogue
    swiglu    the same with weight rows [gate | up]: silu(gate) * up

Codes are whole numbers, -127 .. 127, in units of their row's scale: code = round(127 t / max|t|), half to even, where t is the row before
anything common to all of it (for the norm: sum times weight, as 1 / rms cancels); scale = max|y| / 127. A value next to a border
between two codes is decided by t and max|t| alone, which 64 bits hold exactly, so that codes are the same from
everyone; they and their scales are both outputs. Widths are those of the models in perf/cases.py and generic ones.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one sequence in decode: the norm before a projection
        {"name": "norm_decode_b1", "op": "norm", "tokens": 1, "k": 4096, "dtype": "fp16", "add": True},
        # a first layer's norm (no residual yet) of an odd chunk, a width that is no power of two
        {"name": "norm_first_333", "op": "norm", "tokens": 333, "k": 2576, "dtype": "bf16", "add": False},
        # a long prompt
        {"name": "norm_prompt_8k", "op": "norm", "tokens": 8192, "k": 4096, "dtype": "fp16", "add": True},
        # a small batch in decode: what down_proj reads
        {"name": "quantize_decode_b7", "op": "quantize", "tokens": 7, "k": 12288, "dtype": "bf16"},
        # a prompt chunk: what down_proj reads
        {"name": "quantize_chunk_4k", "op": "quantize", "tokens": 4096, "k": 12288, "dtype": "fp16"},
        # one sequence in decode: qkv
        {"name": "linear_qkv_m1", "op": "linear", "m": 1, "k": 4096, "n": 6144, "dtype": "fp16"},
        # a serving batch in decode: down
        {"name": "linear_down_m32", "op": "linear", "m": 32, "k": 12288, "n": 4096, "dtype": "bf16"},
        # an odd prompt through a projection of odd width
        {"name": "linear_odd_m509", "op": "linear", "m": 509, "k": 2064, "n": 5001, "dtype": "bf16"},
        # a long prompt: o
        {"name": "linear_o_m8192", "op": "linear", "m": 8192, "k": 4096, "n": 4096, "dtype": "fp16"},
        # a few sequences in decode: gate_up
        {"name": "swiglu_m5", "op": "swiglu", "m": 5, "k": 4096, "n": 24576, "dtype": "fp16"},
        # a large decode batch, or a short chunk
        {"name": "swiglu_m200", "op": "swiglu", "m": 200, "k": 2560, "n": 19456, "dtype": "bf16"},
        # a long prompt: gate_up
        {"name": "swiglu_m8192", "op": "swiglu", "m": 8192, "k": 4096, "n": 24576, "dtype": "fp16"},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "quantize", "linear", "linear", "linear", "swiglu", "swiglu"))
    dtype = rng.choice(("fp16", "bf16"))
    if op in ("norm", "quantize"):
        k = 16 * _log(rng, 4, 1024 if op == "norm" else 1792)
        case = {"op": op, "tokens": _log(rng, 1, min(16384, 5e7 / k)), "k": k, "dtype": dtype}
        return {**case, "add": rng.random() < 0.7} if op == "norm" else case
    m, n, k = _log(rng, 1, 8192), _log(rng, 64, 32768), 16 * _log(rng, 4, 1024)
    while n * k > 1.5e8 or m * n * k > 8e11:
        n = max(1, n * 3 // 4)
    return {"op": op, "m": m, "k": k, "n": 2 * ((n + 1) // 2) if op == "swiglu" else n, "dtype": dtype}


# ---------------------------------------------------------------------------------------- inputs
def _hidden(g: torch.Generator, tokens: int, k: int) -> torch.Tensor:
    """float32 rows as hidden states are: most channels of one size, a few much larger ones."""
    size = torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    size[torch.randint(0, k, (max(1, k // 500),), device="cuda", generator=g)] *= 20
    return torch.randn(tokens, k, device="cuda", generator=g) * size


def _codes(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    top = rows.abs().amax(-1)
    return torch.round(rows * (127.0 / top)[:, None]).to(torch.int8), top / 127.0


def prepare(case: dict, seed: int) -> dict:
    g, op, k = torch.Generator(device="cuda").manual_seed(seed), case["op"], case["k"]
    dtype = DTYPES[case["dtype"]]
    state = {"op": op, "dtype": dtype}
    if op in ("norm", "quantize"):
        state["x"] = _hidden(g, case["tokens"], k).to(dtype)
        if op == "norm":
            state["residual"] = _hidden(g, case["tokens"], k).to(dtype) if case["add"] else None
            state["weight"] = (0.5 + torch.rand(k, device="cuda", generator=g)).to(dtype)
        return state
    state["x"], state["x_scale"] = _codes(_hidden(g, case["m"], k))
    w = torch.randn(case["n"], k, device="cuda", generator=g) * k ** -0.5
    state["w"], state["w_scale"] = _codes(w)
    return state


# ------------------------------------------------------------------------------------- plain forms
def _plain_codes(t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, max|t|) of float64 rows whose values and maxima are exact: so is 127 t, and the quotient is rounded in its 53rd bit,
    far from any border that it does not lie on."""
    top = t.abs().amax(-1, keepdim=True)
    return torch.round(torch.where(top > 0, 127.0 * t / top, 0.0)).to(torch.int8), top[:, 0].float()


def _plain_norm(s: dict):
    total = s["x"].float()
    if s["residual"] is not None:
        total = total + s["residual"].float()
        s["residual"].copy_(total)
    codes, top = _plain_codes(total.double() * s["weight"].double())
    scale = top * torch.rsqrt((total * total).mean(-1) + EPS) / 127.0
    return (codes, scale) if s["residual"] is None else (codes, scale, s["residual"])


def _plain_quantize(s: dict):
    codes, top = _plain_codes(s["x"].double())
    return codes, top / 127.0


def _plain_product(s: dict) -> torch.Tensor:
    y = torch.matmul(s["x"].float(), s["w"].float().t()) * s["x_scale"][:, None] * s["w_scale"]
    if s["op"] == "swiglu":
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(s["dtype"])


@torch.no_grad()
def run(state: dict):
    op = state["op"]
    if not own:
        return {"norm": _plain_norm, "quantize": _plain_quantize, "linear": _plain_product, "swiglu": _plain_product}[op](state)
    if op == "norm":
        from tandem_amd.layers import norm

        if state["residual"] is None:
            return norm.rms_norm_int8(state["x"], state["weight"], EPS)
        return norm.fused_add_rms_norm_int8(state["x"], state["residual"], state["weight"], EPS)
    from tandem_amd.layers import w8

    if op == "quantize":
        return w8.quantize_int8(state["x"])
    return w8.linear_int8(state["x"], state["x_scale"], state["w"], state["w_scale"], silu_mul=op == "swiglu", dtype=state["dtype"])


# ------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    op, k = case["op"], case["k"]
    if op == "norm":
        t = case["tokens"]
        return {"bytes": t * k * (7 if case["add"] else 3) + 2 * k + 4 * t, "flops": 6.0 * t * k}
    if op == "quantize":
        return {"bytes": 3 * case["tokens"] * k + 4 * case["tokens"], "flops": 3.0 * case["tokens"] * k}
    m, n = case["m"], case["n"]
    out = n // 2 if op == "swiglu" else n
    return {"bytes": m * k + n * k + 4 * (m + n) + 2 * m * out, "flops": 2.0 * m * n * k}


# --------------------------------------------------------------------------------- 64-bit results
@torch.no_grad()
def exact(case: dict, seed: int):
    s, op = prepare(case, seed), case["op"]
    if op in ("norm", "quantize"):  # codes are whole numbers, compared as such
        x = s["x"].double()
        if op == "quantize":
            return None, torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127
        if s["residual"] is not None:
            x = x + s["residual"].double()
        y = x / (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / case["k"] + EPS).sqrt() * s["weight"].double()
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127
        return (None, scale) if s["residual"] is None else (None, scale, x)
    x = s["x"].double() * s["x_scale"].double()[:, None]

    def product(rows: slice) -> torch.Tensor:
        return x @ (s["w"][rows].double() * s["w_scale"][rows].double()[:, None]).t()

    half = case["n"] // 2
    if op == "linear":
        return torch.cat([product(slice(0, half)), product(slice(half, None))], dim=1)
    return torch.nn.functional.silu(product(slice(0, half))) * product(slice(half, None))
