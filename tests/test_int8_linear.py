"""Products of 8-bit integers (tw4_gemm_int8 behind layers/w8.py) against the formula in 64 bits.

Tolerance. The sum of products is exact; made a float32 (2^-24 of it, nothing below 2^24), times one scale and the other: 3 roundings of 2^-24,
and one to the type, half a step of it (fp16 2^-11, bf16 2^-8, and 2^-25 absolute where fp16 is subnormal). SwiGLU: gate and up
have those 3 each; the gate's change the sigmoid by |g| 3 roundings at most; exp(-g) is off by its argument's roundings, 2 |g|, and 2
of its own, the sum by 1, its reciprocal (1 ulp) by 2, two products by 2: (3 + 3 + 2 + 1 + 2 + 2 + 5 |g|) of 2^-24."""

from __future__ import annotations

import ctypes
import json
import math
import os

import pytest
import torch
from torch import nn

from tandem_amd import model as tmodel
from tandem_amd.layers import linear, norm, w4_hip, w8
from tandem_amd.loader import QuantConfig

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
INT8 = QuantConfig("compressed-tensors", 8, 0)


# ------------------------------------------------------------------------------------------- CPU
def test_argument_errors_return_before_launch():
    lib, p, odd = w4_hip.library(), ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    #       x stride xs w stride ws y ws words locks counters M N K act bf16 kernel splits
    good = [p, 64, p, p, 64, p, p, None, 0, None, 0, 3, 5, 64, 0, 0, 3, 1]
    for at, value, needle in ((0, None, "null"), (2, None, "null"), (3, None, "null"), (5, None, "null"), (6, None, "null"),
                              (0, odd, "aligned"), (3, odd, "aligned"), (2, ctypes.c_void_p(4098), "aligned"),
                              (6, ctypes.c_void_p(4097), "aligned"), (1, 48, "apart"), (1, 72, "apart"), (4, 48, "apart"), (4, 1 << 22, "apart"),
                              (11, -1, "M"), (11, (1 << 20) + 1, "M"), (12, 0, "N"), (12, (1 << 24) + 1, "N"), (13, 72, "K"), (13, 0, "K"),
                              (13, 1 << 17, "K"), (14, 2, "act"), (14, 1, "even"), (16, -1, "kernel"), (16, 13, "kernel"), (17, 0, "splits"),
                              (17, 2, "splits")):
        args = list(good)
        args[at] = value
        assert lib.tw4_gemm_int8(*args, None) == (w4_hip.TW4_ECONFIG if at >= 16 else w4_hip.TW4_EINVAL), (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good[11] = 0
    assert lib.tw4_gemm_int8(*good, None) == w4_hip.TW4_OK
    # splits that take a workspace: none, too few words, too few counters; kernels that do not take the call
    for change, status, needle in (({13: 256, 1: 256, 4: 256, 17: 2}, w4_hip.TW4_EINVAL, "workspace"),
                                   ({13: 256, 1: 256, 4: 256, 17: 2, 7: p, 8: 2 * 32 * 64 - 1, 9: p, 10: 1}, w4_hip.TW4_ESPACE, "partial sums"),
                                   ({13: 256, 1: 256, 4: 256, 17: 2, 7: p, 8: 2 * 32 * 64, 9: p, 10: 0}, w4_hip.TW4_ESPACE, "counters"),
                                   ({11: 1 << 20, 12: 1 << 20}, w4_hip.TW4_EINVAL, "too many"), ({11: 1 << 20, 16: 0}, w4_hip.TW4_ECONFIG, "streaming"),
                                   ({12: 6, 14: 1, 16: 0}, w4_hip.TW4_ECONFIG, "SwiGLU"), ({11: 17, 16: 1}, w4_hip.TW4_ECONFIG, "16 tokens"),
                                   ({11: 17, 16: 2}, w4_hip.TW4_ECONFIG, "16 tokens")):
        args = list(good)
        args[11] = 3
        for at, value in change.items():
            args[at] = value
        assert lib.tw4_gemm_int8(*args, None) == status, change
        assert needle in lib.tw4_last_error().decode(), (change, lib.tw4_last_error())


def test_token_argument_errors_return_before_launch():
    lib, p, odd, own = w4_hip.library(), ctypes.c_void_p(4096), ctypes.c_void_p(4104), ctypes.c_void_p(8192)
    #       x residual new weight eps w stride ws y N K act bf16 cus
    good = [p, p, own, p, 1e-6, p, 64, p, p, 6, 64, 0, 0, 256]
    for at, value, needle in ((0, None, "null"), (5, None, "null"), (7, None, "null"), (8, None, "null"), (0, odd, "aligned"), (1, odd, "aligned"),
                              (2, odd, "aligned"), (3, odd, "aligned"), (5, odd, "aligned"), (7, ctypes.c_void_p(4098), "aligned"),
                              (8, ctypes.c_void_p(4097), "aligned"), (1, None, "residual"), (2, None, "residual"), (3, None, "residual"),
                              (2, p, "its own"), (0, own, "its own"), (1, own, "its own"), (6, 48, "apart"), (6, 72, "apart"), (6, 1 << 22, "apart"), (9, 0, "N"), (9, (1 << 24) + 1, "N"),
                              (10, 72, "K"), (10, 0, "K"), (10, 16400, "K"), (11, 2, "act"), (13, 0, "cus")):
        args = list(good)
        args[at] = value
        if at == 10 and value:
            args[6] = 1 << 15
        assert lib.tw4_token_int8(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, lib.tw4_last_error())
    for n, act, cus in ((32 * 7 + 1, 0, 7), (2 * (16 * 7 + 1), 1, 7), (1 << 24, 0, 256)):
        args = list(good)
        args[9], args[11], args[13] = n, act, cus
        assert lib.tw4_token_int8(*args, None) == w4_hip.TW4_ECONFIG and "CU" in lib.tw4_last_error().decode()
    args = list(good)
    args[9], args[11] = 5, 1
    assert lib.tw4_token_int8(*args, None) == w4_hip.TW4_EINVAL and "even" in lib.tw4_last_error().decode()


def _plan(m, n, k, act, cus=256):
    out = (ctypes.c_int * 4)()
    w4_hip.check(w4_hip.library().tw4_gemm_int8_plan(m, n, k, act, cus, out))
    return tuple(out)


def test_plan():
    """Every size has a kernel that takes it, within the workspace; and the choice on the sizes it was fitted to."""
    for m in (1, 16, 17, 33, 200, 201, 1100, 5000, 1 << 20):
        for n, k in ((1, 16), (2, 131056), (6144, 4096), (1 << 24, 16), (34816, 5120)):
            for act in (0, 1) if n % 2 == 0 else (0,):
                for cus in (1, 64, 256):
                    kernel, splits, words, counters = _plan(m, n, k, act, cus)
                    assert 0 <= kernel < 13 and 1 <= splits <= (max(1, k // 128) if kernel else 32) and not (kernel == 0 and act) and not (kernel in (1, 2) and m > 16)
                    assert words <= w4_hip.WORKSPACE_FLOATS and counters <= w4_hip.WORKSPACE_LOCKS and (kernel > 0 and splits > 1) == (words > 0)
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "profiles", "gemm_int8_rule_sweep.jsonl")
    ratios = []
    for line in open(path, encoding="utf-8"):
        d = json.loads(line)
        kernel, splits, _, _ = _plan(d["m"], d["n"], d["k"], d["act"])
        us = d["us"][f"{kernel},{splits if kernel else 1}"]
        ratios.append(us / min(d["us"].values()))
    assert len(ratios) > 500 and math.exp(sum(map(math.log, ratios)) / len(ratios)) < 1.015 and max(ratios) < 1.25
    with pytest.raises(RuntimeError, match="plan"):
        _plan(0, 4, 16, 0)


def test_refusals_on_the_cpu(monkeypatch):
    x, s, w = torch.zeros(2, 64, dtype=torch.int8), torch.ones(2), torch.zeros(3, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="GPU"):
        w8.linear_int8(x, s, w, torch.ones(3))

    def lay(shape, stride, dtype=torch.int8, index=0):
        return torch.Size(shape), stride, dtype, index

    def f32(*shape):
        return lay(shape, (1,) * len(shape), torch.float32)

    x, w = lay((2, 64), (64, 1)), lay((6, 64), (64, 1))
    w8._checked.cache_clear()
    monkeypatch.setattr(w8, "_cus", lambda index: 256)
    got = w8._checked(x, f32(2), w, f32(6, 1), True, torch.float16)
    assert got[:2] == (64, 64) and got[2][:5] == (2, 6, 64, 1, 0) and got[3:] == (False, 3, 0) and got[2][5:] == _plan(2, 6, 64, 1)[:2]
    got = w8._checked(lay((1, 64), (7, 1)), f32(1), w, f32(6), False, torch.bfloat16)
    assert got[:2] == (64, 64) and got[2][:5] == (1, 6, 64, 0, 1) and got[3:] == (False, 6, 0)
    for bad in ((x, f32(3), w, f32(6), False, torch.float16), (x, f32(2), w, f32(5), False, torch.float16),
                (lay((2, 48), (64, 1)), f32(2), w, f32(6), False, torch.float16), (x, f32(2), w, f32(6), False, torch.float32),
                (x, f32(2), lay((5, 64), (64, 1)), f32(5), True, torch.float16), (lay((2, 64), (72, 1)), f32(2), w, f32(6), False, torch.float16),
                (x, f32(2), lay((6, 64), (1, 6)), f32(6), False, torch.float16), (x, f32(2), lay((6, 64), (64, 1), torch.uint8), f32(6), False, torch.float16),
                (x, f32(2), lay((6, 64), (64, 1), torch.int8, 1), f32(6), False, torch.float16), (x, lay((2,), (1,), torch.float16), w, f32(6), False, torch.float16),
                (x, lay((2,), (2,), torch.float32), w, f32(6), False, torch.float16), (lay((2, 1 << 17), (1 << 17, 1)), f32(2), lay((6, 1 << 17), (1 << 17, 1)), f32(6), False, torch.float16),
                (lay((2, 64), (0, 1)), f32(2), w, f32(6), False, torch.float16), (lay((2, 64), (1 << 22, 1)), f32(2), w, f32(6), False, torch.float16)):
        with pytest.raises(RuntimeError, match="^linear_int8: "):
            w8._checked(*bad)
    w8._checked.cache_clear()


def test_layer_without_a_gpu():
    layer = linear.make_linear(64, 24, False, INT8)
    assert isinstance(layer, w8.W8Linear) and layer.weight.shape == (24, 64) and layer.weight_scale.shape == (24, 1)
    layer.weight.fill_(-128)
    layer.weight_scale.copy_(torch.arange(24)[:, None] * 1e-9 + 1e-7)  # nothing float16 could hold
    scale = layer.weight_scale.clone()
    box = nn.ModuleList([layer, nn.Linear(4, 4)]).to(dtype=torch.float16)
    assert box[1].weight.dtype == torch.float16 and layer.weight.dtype == torch.int8
    assert layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_scale, scale)
    assert linear.finalize_quantized(box) == 0 and layer.enable_silu_mul()
    with pytest.raises(NotImplementedError):
        linear.make_linear(64, 24, True, INT8)
    for bad in ((72, 8), (0, 8), (32784, 8), (64, 0)):
        with pytest.raises(ValueError):
            w8.W8Linear(*bad)
    assert not w8.W8Linear(64, 23).enable_silu_mul()


# ------------------------------------------------------------------------------------------- GPU
def _operands(m, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-127, 128, (m, k), device="cuda", dtype=torch.int8, generator=g)
    w = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8, generator=g)
    xs = (0.5 + torch.rand(m, device="cuda", generator=g)) * 0.02
    ws = (0.5 + torch.rand(n, device="cuda", generator=g)) * 0.02 * k ** -0.5
    return x, xs, w, ws


def _check(y, x, xs, w, ws, silu_mul, dtype):
    exact = torch.matmul(x.cpu().double(), w.cpu().double().t()) * xs.cpu().double()[:, None] * ws.cpu().double()
    steps = 3.0
    if silu_mul:
        g, u = exact.chunk(2, dim=1)
        exact, steps = g * torch.sigmoid(g) * u, 13 + 5 * g.abs()
    assert y.dtype == dtype and y.shape == exact.shape
    off = (y.cpu().double() - exact).abs()
    allowed = (HALF_STEP[dtype] + steps * 2.0 ** -24 * 1.01) * exact.abs() + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130)
    assert bool((off <= allowed).all()), (float((off / exact.abs().clamp(min=1e-9)).max()), int((off > allowed).sum()))


SHAPES = [(1, 1, 16), (1, 17, 48), (1, 256, 4096), (2, 6, 64), (3, 130, 2064), (4, 4096, 1024), (5, 100, 4096), (7, 33, 112), (8, 500, 1040),
          (15, 64, 128), (16, 2048, 512), (17, 34, 80), (24, 1000, 4096), (31, 48, 16), (32, 512, 12288), (33, 258, 272), (48, 4096, 1024),
          (63, 70, 336), (64, 1024, 2048), (65, 130, 528), (77, 1536, 1024), (100, 62, 4096), (127, 128, 64), (128, 256, 256), (129, 514, 640),
          (200, 2000, 512), (255, 250, 1008), (256, 256, 4096), (257, 30, 2064), (300, 5002, 272), (512, 512, 512), (513, 1026, 144),
          (700, 2, 4096), (1024, 1280, 1024), (1500, 766, 1040), (2049, 258, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("silu_mul", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, dtype, silu_mul):
    x, xs, w, ws = _operands(m, n + (n % 2 if silu_mul else 0), k, seed=m + n + k)
    kept = [t.clone() for t in (x, xs, w, ws)]
    y = w8.linear_int8(x, xs, w, ws, silu_mul=silu_mul, dtype=dtype)
    _check(y, x, xs, w, ws, silu_mul, dtype)
    assert all(torch.equal(a, b) for a, b in zip(kept, (x, xs, w, ws)))
    assert torch.equal(y, w8.linear_int8(x, xs[:, None], w, ws[:, None], silu_mul=silu_mul, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", range(13))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_kernel(kernel, dtype):
    """Each kernel with several numbers of splits (the streaming one: of rows), tiles that are full and tiles that are not, outputs of any alignment: all the same
    bits, nothing behind the output, counters back at zero."""
    lib = w4_hip.library()
    for m, n, k, act in ((1, 18, 16, 0), (5, 130, 144, 1), (16, 64, 2048, 0), (16, 515, 1040, 0), (17, 256, 400, 1), (150, 200, 640, 0), (193, 1030, 272, 1),
                         (257, 385, 1296, 0), (260, 520, 1296, 1)):
        if (kernel == 0 and act) or (kernel in (1, 2) and m > 16):
            continue
        x, xs, w, ws = _operands(m, n, k, seed=kernel + m)
        out = n // 2 if act else n
        want = None
        for splits in sorted({s for s in (1, 2, 3, 5, 11) if s <= -(-k // 128)} if kernel else {1, 5, 16, 17, 32}):
            part, locks = w4_hip.stream_workspace(x.device)
            for shift in (0, 1, 4):
                buf = torch.full((m * out + 64,), 7.0, dtype=dtype, device="cuda")
                y = buf[shift:shift + m * out].view(m, out)
                w4_hip.check(lib.tw4_gemm_int8(x.data_ptr(), k, xs.data_ptr(), w.data_ptr(), k, ws.data_ptr(), y.data_ptr(), part.data_ptr(), part.numel(),
                                               locks.data_ptr(), locks.numel(), m, n, k, act, int(dtype == torch.bfloat16), kernel, splits,
                                               w4_hip.raw_stream(0)))
                assert bool((buf[:shift] == 7).all()) and bool((buf[shift + m * out:] == 7).all())
                if want is None:
                    want = y.clone()
                    _check(want, x, xs, w, ws, bool(act), dtype)
                assert torch.equal(y, want), (m, n, k, act, splits, shift)
                assert not bool(locks.any())


@pytest.mark.gpu
@pytest.mark.parametrize("silu_mul", [False, True])
@pytest.mark.parametrize("n,k", [(514, 1040), (4096, 4096), (96, 12288)])
def test_rows_do_not_depend_on_the_batch(n, k, silu_mul):
    """Sums are exact and the epilogue is a value's own: a token's result is the same bits in every batch and kernel."""
    x, xs, w, ws = _operands(1100, n, k, seed=n)
    want = w8.linear_int8(x, xs, w, ws, silu_mul=silu_mul)
    for m in (1, 2, 5, 16, 17, 33, 64, 65, 100, 128, 200, 256, 300, 511, 600, 1025):
        assert torch.equal(w8.linear_int8(x[-m:], xs[-m:], w, ws, silu_mul=silu_mul), want[-m:]), m


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 5), (16, 40), (70, 48), (300, 130)])
def test_largest_sums(m, n):
    """K = 131056 of -128 * -128: the largest sum 32 bits hold."""
    k = (1 << 17) - 16
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[n // 2] = 127
    one = torch.full((max(m, n),), 2.0 ** -16, device="cuda")
    y = w8.linear_int8(x, one[:m], w, one[:n], dtype=torch.bfloat16)
    want = torch.full((m, n), 128 * 128 * k * 2.0 ** -32, device="cuda", dtype=torch.float64)
    want[:, n // 2] *= -127 / 128
    assert torch.equal(y, want.to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 130, 1040), (40, 254, 528), (150, 258, 784), (600, 514, 272)])
@pytest.mark.parametrize("silu_mul", [False, True])
def test_strides_scales_and_neighbours(m, n, k, silu_mul):
    """Operands inside larger buffers whose other places hold codes that would show; infinite, NaN and zero scales stay in their
    rows and columns."""
    g = torch.Generator(device="cuda").manual_seed(m)
    bx = torch.randint(-127, 128, (m + 2, k + 96), device="cuda", dtype=torch.int8, generator=g)
    bw = torch.randint(-127, 128, (n + 2, k + 48), device="cuda", dtype=torch.int8, generator=g)
    x, w = bx[1:-1, 32:32 + k], bw[1:-1, 16:16 + k]
    _, xs, _, ws = _operands(m, n, 16, seed=m)
    ws *= k ** -0.5
    for dtype in (torch.float16, torch.bfloat16):
        y = w8.linear_int8(x, xs, w, ws, silu_mul=silu_mul, dtype=dtype)
        _check(y, x, xs, w, ws, silu_mul, dtype)
        assert torch.equal(y, w8.linear_int8(x.contiguous(), xs, w.contiguous(), ws, silu_mul=silu_mul, dtype=dtype))
    xs2, ws2 = xs.clone(), ws.clone()
    xs2[m // 2], ws2[1] = float("nan"), float("nan")
    xs2[0] = 0
    y2 = w8.linear_int8(x, xs2, w, ws2, silu_mul=silu_mul, dtype=torch.bfloat16)
    assert bool(y2[m // 2].isnan().all()) and bool(y2[:, 1].isnan().all())
    keep = [i for i in range(m) if i not in (0, m // 2)]
    cols = [j for j in range(y.shape[1]) if j != 1]
    assert torch.equal(y2[keep][:, cols], y[keep][:, cols]) and (m // 2 == 0 or not bool(y2[0, cols].any()))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2, 1 << 20, 4112), (20, 1 << 20, 4112), (140, 1 << 20, 4112), (70001, 32768, 64), (300000, 16, 16384)])
def test_past_32_bits(m, n, k):
    """Weights, activations and results of more than 2^32 bytes: rows and columns at both ends and in between."""
    x, xs, w, ws = _operands(m, n, k, seed=k)
    y = w8.linear_int8(x, xs, w, ws)
    rows = torch.tensor(sorted({0, 1, m // 2, m - 2, m - 1}), device="cuda")
    for at in (0, n // 2 - 8, n - 16):
        cols = slice(at, at + 16)
        _check(y[rows, cols].contiguous(), x[rows], xs[rows], w[cols], ws[cols], False, torch.float16)


@pytest.mark.gpu
def test_refusals_and_empty():
    x, xs, w, ws = _operands(4, 32, 64, seed=0)
    assert w8.linear_int8(x[:0], xs[:0], w, ws).shape == (0, 32) and w8.linear_int8(x[:0], xs[:0], w, ws, silu_mul=True).shape == (0, 16)
    buf = torch.zeros(64 * 4 + 8, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="aligned"):
        w8.linear_int8(buf[8:].view(4, 64), xs, w, ws)
    with pytest.raises(RuntimeError, match="inference only"):
        w8.linear_int8(x, xs.clone().requires_grad_(), w, ws)


@pytest.mark.gpu
def test_streams_and_graphs():
    """Calls on two streams at once, and the whole run norm -> product -> quantise -> product captured and replayed, each against the
    eager result, with other work between the replays."""
    layers = []
    for i, (k, n) in enumerate(((1024, 4096), (2048, 1024))):
        layer = w8.W8Linear(k, n).cuda()
        _, _, w, ws = _operands(1, n, k, seed=i)
        layer.weight.copy_(w)
        layer.weight_scale.copy_(ws[:, None])
        layers.append(layer)
    layers[0].enable_silu_mul()
    weight = (0.5 + torch.rand(1024, device="cuda")).half()

    def step(x, r):
        y, r = layers[0].forward_norm(x, r, weight, 1e-6)
        return layers[1](y), r

    for m in (1, 9, 40, 300):
        xs = [torch.randn(m, 1024, device="cuda").half() for _ in range(4)]
        rs = [torch.randn(m, 1024, device="cuda").half() for _ in range(4)]
        want = [step(x, r.clone()) for x, r in zip(xs, rs)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = {}
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for i in range(4):
            with torch.cuda.stream(streams[i % 2]):
                got[i] = step(xs[i], rs[i].clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(4) for a, b in zip(got[i], want[i]))
        graphs = []
        for j in range(2):
            gx, gr = xs[0].clone(), rs[0].clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(gx, gr)
            graphs.append((graph, gx, gr, out))
        for i in (1, 3, 2, 0, 1):
            for j, (graph, gx, gr, out) in enumerate(graphs):
                at = (i + j) % 4
                gx.copy_(xs[at])
                gr.copy_(rs[at])
                graph.replay()
                step(xs[i], rs[i].clone())
                torch.cuda.synchronize()
                assert torch.equal(out[0], want[at][0]) and torch.equal(out[1], want[at][1])


@pytest.mark.gpu
def test_layer_shapes_and_norm():
    """W8Linear is its operators one behind the other, for rows and for more dimensions."""
    layer = w8.W8Linear(512, 96).cuda()
    _, _, w, ws = _operands(1, 96, 512, seed=3)
    layer.weight.copy_(w)
    layer.weight_scale.copy_(ws[:, None])
    x, r = torch.randn(6, 512, device="cuda").half(), torch.randn(6, 512, device="cuda").half()
    weight = (0.5 + torch.rand(512, device="cuda")).half()
    for silu_mul in (False, True):
        layer.silu_mul = silu_mul
        y = layer(x)
        assert torch.equal(y, w8.linear_int8(*w8.quantize_int8(x), w, ws, silu_mul=silu_mul))
        assert torch.equal(layer(x.view(2, 3, 512)), y.view(2, 3, -1)) and torch.equal(layer(x[1]), y[1])
        assert layer(x.bfloat16()).dtype == torch.bfloat16 and layer(x[:0]).shape == (0, y.shape[1])
        y, same = layer.forward_norm(x, None, weight, 1e-6)
        assert same is x and torch.equal(y, w8.linear_int8(*norm.rms_norm_int8(x, weight, 1e-6), w, ws, silu_mul=silu_mul))
        r2 = r.clone()
        codes, scales, r3 = norm.fused_add_rms_norm_int8(x, r.clone(), weight, 1e-6)
        y, out = layer.forward_norm(x, r2, weight, 1e-6)
        assert out is r2 and torch.equal(r2, r3) and torch.equal(y, w8.linear_int8(codes, scales, w, ws, silu_mul=silu_mul))
    assert tmodel.GatedMLP(512, 256, INT8).fused_act


def _pair(x, residual, weight, w, ws, silu_mul):
    """What one token's kernel does, with the operators it stands for: (y, new residual)."""
    if weight is None:
        codes, scales = w8.quantize_int8(x)
    elif residual is None:
        codes, scales = norm.rms_norm_int8(x, weight, 1e-6)
    else:
        codes, scales, residual = norm.fused_add_rms_norm_int8(x, residual.clone(), weight, 1e-6)
    return w8.linear_int8(codes, scales, w, ws, silu_mul=silu_mul, dtype=x.dtype), residual


def _same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(2, 16), (34, 48), (130, 1040), (333, 2576), (1024, 8192), (2502, 8208), (6128, 4096), (8192, 272), (96, 16384)])
def test_one_token(n, k, dtype):
    """W8Linear's one row, made in 8 bits inside the product's kernel: the bits of the operators one behind the other, rows of w any multiple
    of 16 apart, x and the residual as they were, nothing written beside y."""
    g = torch.Generator(device="cuda").manual_seed(n + k)
    step = k + 48
    w = torch.randint(-128, 128, (n, step), device="cuda", dtype=torch.int8, generator=g)[:, :k]
    ws = (0.5 + torch.rand(n, device="cuda", generator=g)) * 0.02 * k ** -0.5
    weight = (0.5 + torch.rand(k, device="cuda", generator=g)).to(dtype)
    rows = torch.randn(6, k, device="cuda", generator=g).to(dtype)
    rows[1, k // 2], rows[2, 0], rows[3] = float("inf"), float("nan"), 0
    rows[4] *= 2.0 ** -9
    residual = torch.randn(1, k, device="cuda", generator=g).to(dtype)
    for silu_mul in ((False,) if n % 2 else (False, True)):
        for i in range(6):
            x, before, r = rows[i:i + 1], rows[i].clone(), residual.clone()
            for args in ((None, None), (None, weight), (r, weight)):
                y, total = w8._token_int8(x, args[0], args[1], 1e-6, w, ws, silu_mul)
                want, want_r = _pair(x, *args, w, ws, silu_mul)
                assert y.shape == want.shape and _same_bits(y, want), (i, silu_mul)
                assert (total is None) == (args[0] is None) and (total is None or _same_bits(total, want_r))
            assert _same_bits(rows[i], before) and torch.equal(r, residual)
        out = n // 2 if silu_mul else n
        y, total = torch.full((out + 64,), 3.0, device="cuda", dtype=dtype), torch.full((k + 64,), 3.0, device="cuda", dtype=dtype)
        w4_hip.check(w4_hip.library().tw4_token_int8(
            rows[0].data_ptr(), residual.data_ptr(), total.data_ptr(), weight.data_ptr(), 1e-6, w.data_ptr(), step, ws.data_ptr(),
            y.data_ptr(), n, k, int(silu_mul), int(dtype == torch.bfloat16), 256, w4_hip.raw_stream(0)))
        want, want_r = _pair(rows[:1], residual, weight, w, ws, silu_mul)
        assert _same_bits(y[:out], want[0]) and _same_bits(total[:k], want_r[0])
        assert bool((y[out:] == 3).all()) and bool((total[k:] == 3).all())


@pytest.mark.gpu
def test_one_token_layers():
    """Which W8Linear calls take it, and that every one of them has the bits of the same row in a batch: outputs on both sides of one
    workgroup a CU, K on both sides of its longest, one row of more than two dimensions, a row of odd stride."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for n, k, silu_mul, one in ((32 * cus, 64, False, True), (32 * cus + 2, 64, False, False), (32 * cus, 64, True, True),
                                (32 * cus + 2, 64, True, False), (64, 16384, False, True), (64, 16400, False, False)):
        layer = w8.W8Linear(k, n).cuda()
        _, _, w, ws = _operands(1, n, k, seed=n + k)
        layer.weight.copy_(w)
        layer.weight_scale.copy_(ws[:, None])
        layer.silu_mul = silu_mul
        x, r = torch.randn(3, k, device="cuda").half(), torch.randn(3, k, device="cuda").half()
        weight = (0.5 + torch.rand(k, device="cuda")).half()
        assert layer._one_token(x[:1]) == one and not layer._one_token(x) and not layer._one_token(x[:0])
        y, normed = layer(x), layer.forward_norm(x, None, weight, 1e-6)[0]
        both, total = layer.forward_norm(x, r.clone(), weight, 1e-6)
        for i in range(3):
            assert torch.equal(layer(x[i:i + 1]), y[i:i + 1]) and torch.equal(layer(x[i].view(1, 1, k)), y[i].view(1, 1, -1))
            got, same = layer.forward_norm(x[i:i + 1], None, weight, 1e-6)
            assert torch.equal(got, normed[i:i + 1]) and same.data_ptr() == x[i].data_ptr()
            got, out = layer.forward_norm(x[i:i + 1], r[i:i + 1].clone(), weight, 1e-6)
            assert torch.equal(got, both[i:i + 1]) and torch.equal(out, total[i:i + 1])
        odd = x[0].as_strided((1, k), (k + 1, 1))
        assert torch.equal(layer(odd), y[:1])
    layer = w8.W8Linear(64, 32).cuda()
    x = torch.zeros(1, 64, device="cuda").half()
    for bad in (x.float(), torch.zeros(1, 80, device="cuda").half(), torch.zeros(1, 72, device="cuda").half()[:, 4:68],
                torch.zeros(64, 2, device="cuda").half().t()[:1], x.clone().requires_grad_()):
        with pytest.raises(RuntimeError):
            layer(bad)
    with pytest.raises(RuntimeError, match="residual"):
        layer.forward_norm(x, x.bfloat16(), torch.ones(64, device="cuda").half(), 1e-6)
