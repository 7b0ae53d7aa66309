"""SwiGLU behind the product of 8-bit integers where it leaves the usual sizes: gates from -300 to 60000, on both sides of where exp(-g) passes
2^126 (-87.3) and float32 (-88.7), results past the type, and scales of infinity; every kernel that has it.

Each token has one code and each row of w one, so that gate = x_scale w_scale c and up likewise, whatever the place.

Tolerance, relative: as in test_int8_linear.py, (13 + 5 |g|) 2^-24. Below -87 the silu is (g e) e with e = exp(g / 2): gate 3 roundings and 3 |g| through
the exponent, e is off by its argument's 2 |g / 2| and 2 of its own, twice, two products 2, up 3, the last product 1: 13 + 5 |g| too.
Absolute: the silu is subnormal in float32 from about -92 on and then rounded to a multiple of 2^-149, off by 2^-150 |u|; the result in fp16 by
2^-25, in bf16 by 2^-134, and by 2^-150 before it."""

from __future__ import annotations

import math

import pytest
import torch

from tandem_amd.layers import norm, w4_hip, w8

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
OVER = {torch.float16: 65520.0, torch.bfloat16: (2 - 2.0 ** -8) * 2.0 ** 127}  # rounds to infinity from here on
GATES = [-300.0, -200.0, -174.0, -150.0, -120.0, -104.0, -100.0, -95.0, -92.0, -90.0, -89.0, -88.8, -88.7, -88.5, -88.0, -87.5, -87.4, -87.3, -87.1, -87.001, -87.0,
         -86.999, -86.5, -60.0, -30.0, -17.0, -3.0, -0.5, 0.0, 0.5, 3.0, 17.0, 30.0, 86.0, 87.0, 88.0, 89.0, 200.0, 2000.0, 60000.0]
UPS = [1.0, -3.0, 2.0 ** 60, -2.0 ** 90, 2.0 ** 120]
K = 64


def _operands(m):
    """(x, x_scale, w, w_scale): token i has code 1 + i % 3 in one place, gate rows 100 or -100, up rows 64."""
    pairs = [(g, u) for g in GATES for u in UPS]
    out = len(pairs)
    x = torch.zeros(m, K, dtype=torch.int8)
    x[:, 5] = torch.arange(m) % 3 + 1
    w = torch.zeros(2 * out, K, dtype=torch.int8)
    w[:out, 5], w[out:, 5] = torch.tensor([-100 if g < 0 else 100 for g, _ in pairs]), 64
    ws = torch.tensor([abs(g) / 100 for g, _ in pairs] + [u / 64 for _, u in pairs])
    xs = 1.0 / x[:, 5].float()
    return [t.cuda() for t in (x, xs, w, ws)]


def _exact(x, xs, w, ws):
    y = torch.matmul(x.cpu().double(), w.cpu().double().t()) * xs.cpu().double()[:, None] * ws.cpu().double()
    return y.chunk(2, dim=1)


def _check(y, g, u, dtype):
    """Against 64 bits: values within the tolerance, infinities where a result leaves the type."""
    want, y = g * torch.sigmoid(g) * u, y.cpu().double()
    size = want.abs()
    assert not bool(((size / OVER[dtype] - 1).abs() < 0.01).any())  # none lies where either side of the border would be right
    over = size >= OVER[dtype]
    assert bool(over.any()) and torch.equal(y[over], want[over].sign() * math.inf)
    allowed = (HALF_STEP[dtype] + 1.01 * (13 + 5 * g.abs()) * 2.0 ** -24) * size + 2.0 ** -150 * (1 + u.abs()) + LEAST[dtype]
    off = (y - want).abs()[~over]
    assert bool((off <= allowed[~over]).all()), [(float(a), float(b), float(c)) for a, b, c, bad in zip(
        g.expand_as(y)[~over], want[~over], y[~over], off > allowed[~over]) if bad][:5]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kernel", range(1, 13))
def test_gates_far_out(kernel, dtype):
    lib = w4_hip.library()
    for m in (1, 5, 16, 130):
        if kernel <= 2 and m > 16:
            continue
        x, xs, w, ws = _operands(m)
        y = torch.empty(m, len(ws) // 2, dtype=dtype, device="cuda")
        w4_hip.check(lib.tw4_gemm_int8(x.data_ptr(), K, xs.data_ptr(), w.data_ptr(), K, ws.data_ptr(), y.data_ptr(), None, 0, None, 0, m, len(ws), K,
                                       1, int(dtype == torch.bfloat16), kernel, 1, w4_hip.raw_stream(0)))
        _check(y, *_exact(x, xs, w, ws), dtype)
        assert torch.equal(y, w8.linear_int8(x, xs, w, ws, silu_mul=True, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gates_far_out_of_one_token(dtype):
    """The kernel that makes the token's codes itself, alone and behind the norm."""
    _, _, w, ws = _operands(1)
    x = torch.zeros(1, K, dtype=dtype, device="cuda")
    x[0, 5] = 1.0
    layer = w8.W8Linear(K, len(ws)).cuda()
    layer.weight.copy_(w)
    layer.weight_scale.copy_(ws[:, None])
    assert layer.enable_silu_mul() and layer._one_token(x)
    codes, scales = w8.quantize_int8(x)
    y = layer(x)
    _check(y, *_exact(codes, scales, w, ws), dtype)
    assert torch.equal(y, w8.linear_int8(codes, scales, w, ws, silu_mul=True, dtype=dtype))
    weight = torch.full((K,), K ** -0.5, dtype=dtype, device="cuda")  # x's normalised value is K^(1/2)
    codes, scales = norm.rms_norm_int8(x, weight, 0.0)
    y = layer.forward_norm(x, None, weight, 0.0)[0]
    _check(y, *_exact(codes, scales, w, ws), dtype)
    assert torch.equal(y, w8.linear_int8(codes, scales, w, ws, silu_mul=True, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("silu_mul", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_infinite_scales(m, dtype, silu_mul):
    """An infinite scale of a token or a feature gives infinities by sign, NaN for a sum of 0 and for a gate of -infinity, and leaves the other rows and
    columns their bits."""
    g = torch.Generator(device="cuda").manual_seed(m)
    n = 130
    x = torch.randint(-127, 128, (m, 48), device="cuda", dtype=torch.int8, generator=g)
    w = torch.randint(-128, 128, (n, 48), device="cuda", dtype=torch.int8, generator=g)
    w[7] = 0
    xs, ws = torch.full((m,), 2.0 ** -10, device="cuda"), torch.full((n,), 2.0 ** -8, device="cuda")
    before = w8.linear_int8(x, xs, w, ws, silu_mul=silu_mul, dtype=dtype)
    for row, feature in ((m // 2, None), (None, 3), (None, n - 2)):
        xs2, ws2 = xs.clone(), ws.clone()
        if row is not None:
            xs2[row] = math.inf
        if feature is not None:
            ws2[feature] = math.inf
        y = w8.linear_int8(x, xs2, w, ws2, silu_mul=silu_mul, dtype=dtype)
        exact = torch.matmul(x.cpu().double(), w.cpu().double().t()) * xs2.cpu().double()[:, None] * ws2.cpu().double()
        if silu_mul:
            gate, up = exact.chunk(2, dim=1)
            exact = gate * torch.sigmoid(gate) * up
        inside = torch.ones_like(y, dtype=torch.bool)
        if row is not None:
            inside[row] = False
        else:
            inside[:, feature % y.shape[1]] = False
        got, want = y.cpu().double()[~inside.cpu()], exact[~inside.cpu()]
        assert bool((want.isnan() | want.isinf() | (want == 0)).all()) and torch.equal(got.nan_to_num(nan=7.0, posinf=1e300, neginf=-1e300),
                                                                                      want.nan_to_num(nan=7.0, posinf=1e300, neginf=-1e300))
        assert torch.equal(y[inside], before[inside])
