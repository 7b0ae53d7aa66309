"""Rows in 8 bits (tw4_quantize_int8, tw4_rms_norm_int8 behind layers/w8.py and layers/norm.py) against the formula in 64 bits.

Codes are exact. t = s * weight has 24 + 11 bits at most and 127 t 42, both exact in 64 bits; t / max|t| lies on a border between two
codes or at least 2^-43 of itself beside it, so a quotient rounded to 53 bits decides every code as the exact one would.

Scales. max|t| is rounded to float32, divided by 127: 2 roundings, 2^-24 each. With the norm: s is rounded, a chunk adds 8 squares, 4
steps add 16 chunks, a lane up to 4 of those sums and 6 steps the lanes, all positive, so that the sum is off by at most 2 + 8 + 4 +
4 + 6 = 24 roundings and its root by 12; mean, eps, reciprocal root (2) and product are 5 more: 19 of 2^-24 in all; 36 are allowed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tandem_amd.layers import norm, w4_hip, w8

EPS = 1e-6
STEP = 2.0 ** -24


# ------------------------------------------------------------------------------------------- CPU
def test_argument_errors_return_before_launch():
    lib, p, odd = w4_hip.library(), ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    good = [p, 64, p, p, 3, 64, 0]  # x stride codes scales M K bf16
    for at, value, needle in ((0, None, "null"), (2, None, "null"), (3, None, "null"), (0, odd, "aligned"), (2, odd, "aligned"),
                              (3, ctypes.c_void_p(4098), "aligned"), (1, 56, "apart"), (1, 68, "apart"), (4, -1, "M >= 0"), (5, 24, "K %"),
                              (5, 0, "K %"), (5, 32784, "K %"), (4, 1 << 26, "too many")):
        args = list(good)
        args[at] = value
        assert lib.tw4_quantize_int8(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good[4] = 0
    assert lib.tw4_quantize_int8(*good, None) == w4_hip.TW4_OK
    good = [p, 64, p, 64, p, 1e-6, p, p, 3, 64, 0]  # x stride residual stride weight eps codes scales M K bf16
    for at, value, needle in ((0, None, "null"), (4, None, "null"), (4, odd, "aligned"), (2, odd, "aligned"), (3, 56, "apart"),
                              (3, 68, "apart"), (9, 40, "K %"), (8, -1, "M >= 0"), (8, 1 << 26, "too many")):
        args = list(good)
        args[at] = value
        assert lib.tw4_rms_norm_int8(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good[8] = 0
    assert lib.tw4_rms_norm_int8(*good, None) == w4_hip.TW4_OK


def test_refusals_on_the_cpu():
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    for call in (lambda: w8.quantize_int8(x), lambda: norm.rms_norm_int8(x, w, EPS), lambda: norm.fused_add_rms_norm_int8(x, x, w, EPS)):
        with pytest.raises(RuntimeError, match="GPU rows"):
            call()


def test_rows_layouts():
    """The checks go by layouts, so GPU ones are looked at here without a GPU."""
    def lay(shape=(4, 64), stride=(64, 1), dtype=torch.float16, index=0):
        return torch.Size(shape), stride, dtype, index

    weight = lay((64,), (1,))
    assert norm.check_rows("f", lay(), lay(), weight) == (64, 64, 4, 64, 0, 0)
    assert norm.check_rows("f", lay(stride=(80, 1)), lay(stride=(72, 1), shape=(4, 64)), weight)[:2] == (80, 72)
    assert norm.check_rows("f", lay((1, 64), (0, 1)), None, None)[:3] == (64, 64, 1)
    for bad in ((lay((4, 40), (40, 1)), None, None), (lay((4, 32784), (32784, 1)), None, None), (lay((64,), (1,)), None, None),
                (lay(dtype=torch.float32), None, None), (lay(stride=(1, 4)), None, None), (lay(stride=(32, 1)), None, None),
                (lay(stride=(68, 1)), None, None), (lay(stride=(0, 1)), None, None), (lay(), lay((3, 64)), None),
                (lay(), lay(dtype=torch.bfloat16), None), (lay(), lay(index=1), None), (lay(), lay(stride=(0, 1)), None),
                (lay(), None, lay((64,), (2,))), (lay(), None, lay((64,), (1,), torch.bfloat16)), (lay(), None, lay((32,), (1,)))):
        with pytest.raises(RuntimeError, match="^f: "):
            norm.check_rows("f", *bad)


@pytest.mark.parametrize("a,step_a,b,step_b,rows,width,apart", [
    (0, 128, 512, 128, 4, 128, True), (0, 128, 384, 128, 4, 128, False), (512, 128, 0, 128, 4, 128, True), (0, 256, 128, 256, 4, 128, True),
    (128, 256, 0, 256, 4, 128, True), (0, 256, 112, 256, 4, 128, False), (0, 256, 144, 256, 4, 128, False), (0, 128, 0, 128, 4, 128, False),
    (0, 256, 128, 272, 4, 128, False), (0, 256, 256 + 128, 256, 4, 128, True), (0, 256, 128, 256, 1, 128, True)])
def test_shared_memory_is_seen(a, step_a, b, step_b, rows, width, apart):
    assert norm._apart(a, step_a, b, step_b, rows, width) is apart
    assert norm._apart(b, step_b, a, step_a, rows, width) is apart


# ------------------------------------------------------------------------------------------- GPU
def _codes(t):
    """Codes and max|t| of float64 rows."""
    top = t.abs().amax(-1, keepdim=True)
    return torch.round(torch.where(top > 0, 127.0 * t / top, 0.0)).to(torch.int8), top[:, 0]


def _rows(m, k, dtype, seed, outliers=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, device="cuda", generator=g)
    if outliers:
        x[:, k // 3] *= 30
    return x.to(dtype)


WIDTHS = [16, 32, 48, 496, 512, 528, 1024, 1040, 2048, 2064, 2560, 4096, 4112, 5120, 6160, 8192, 8208, 12288, 12304, 16384, 16400, 24576, 24592,
          28672, 30720, 30736, 32768]
ROWS = [1, 2, 3, 5, 8, 63, 64, 65, 255, 256, 333, 1023, 1024]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize(k, dtype):
    for m in ROWS if k <= 8192 else (1, 3, 40):
        x = _rows(m, k, dtype, seed=k + m, outliers=m % 2 == 0)
        before = x.clone()
        codes, scales = w8.quantize_int8(x)
        want, top = _codes(x.double())
        assert codes.dtype == torch.int8 and codes.shape == (m, k) and scales.dtype == torch.float32 and scales.shape == (m,)
        assert torch.equal(codes, want), (m, int((codes != want).sum()))
        assert bool(((scales.double() - top / 127).abs() <= 2 * STEP * top / 127).all()) and torch.equal(x, before)


@pytest.mark.gpu
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_norm(k, dtype, add):
    g = torch.Generator(device="cuda").manual_seed(k)
    w = (0.25 + 1.5 * torch.rand(k, device="cuda", generator=g)).to(dtype)
    w[k // 2] *= -1
    for m in ROWS if k <= 8192 else (1, 3, 40):
        x, r = _rows(m, k, dtype, seed=k + m), _rows(m, k, dtype, seed=k + m + 7)
        x0, r0 = x.clone(), r.clone()
        s = x.float()
        if add:
            s = s + r.float()
            codes, scales, out = norm.fused_add_rms_norm_int8(x, r, w, EPS)
            assert out is r and torch.equal(r, s.to(dtype))
        else:
            codes, scales = norm.rms_norm_int8(x, w, EPS)
            assert torch.equal(r, r0)
        want, top = _codes(s.double() * w.double())
        assert torch.equal(codes, want), (m, int((codes != want).sum()))
        full = x0.double() + r0.double() if add else x0.double()
        scale = top * torch.rsqrt((full * full).mean(-1) + EPS) / 127
        assert bool(((scales.double() - scale).abs() <= 36 * STEP * scale).all()) and torch.equal(x, x0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_rows_do_not_depend_on_the_batch(k, dtype):
    """Codes and scales of a row are the same bits whatever the batch."""
    m = 1030
    x, r = _rows(m, k, dtype, seed=k), _rows(m, k, dtype, seed=k + 1)
    w = (0.5 + torch.rand(k, device="cuda")).to(dtype)
    want = norm.rms_norm_int8(x, w, EPS), norm.fused_add_rms_norm_int8(x, r.clone(), w, EPS), w8.quantize_int8(x)
    for n in (1, 3, 255, 256, 1023):
        got = norm.rms_norm_int8(x[-n:], w, EPS), norm.fused_add_rms_norm_int8(x[-n:], r[-n:].clone(), w, EPS), w8.quantize_int8(x[-n:])
        assert all(torch.equal(a, b[-n:]) for g, v in zip(got, want) for a, b in zip(g, v)), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_borders(dtype):
    """Values that lie on borders between codes (x = max / 2 is 63.5) and one step beside them, in every place of a row."""
    for k, scale in ((64, 1.0), (1040, 0.0078125), (4096, 512.0)):
        tops = torch.tensor([254.0, 127.0, 63.5, 31.75, 2.0, 1.0], device="cuda")[:, None].expand(6, k)
        halves = (torch.arange(k, device="cuda") % 255 - 127).float() + 0.5
        x = (halves * tops / 127).clamp(-tops, tops).to(dtype)
        x = torch.cat([x, torch.nextafter(x.float(), torch.full_like(x.float(), 1e9)).to(dtype), -x], dim=0) * scale
        x[:, k // 2] = tops[:, 0].repeat(3).to(dtype) * scale
        near = x.clone().view(torch.int16)
        near[:, 1::3] += 1  # the next value of the type
        for rows in (x, near.view(dtype)):
            want, _ = _codes(rows.double())
            assert torch.equal(w8.quantize_int8(rows)[0], want)
            w = torch.full((k,), 0.75, device="cuda", dtype=dtype)
            w[::5] = 1.5
            assert torch.equal(norm.rms_norm_int8(rows, w, EPS)[0], _codes(rows.double() * w.double())[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [16, 528, 4096, 16384])
def test_special_rows(k, dtype):
    """Zeros, infinities, NaN, the type's largest and smallest values: each row by itself."""
    fin = torch.finfo(dtype)
    x = _rows(12, k, dtype, seed=k)
    x[0] = 0
    x[1, k - 1], x[2, 0], x[3, k // 2], x[4] = float("inf"), float("nan"), -float("inf"), fin.max
    x[5] = fin.smallest_normal
    x[6] = 0
    x[6, k - 2] = -fin.smallest_normal
    x[7, 3] = -fin.max
    x[8] = -0.0
    codes, scales = w8.quantize_int8(x)
    bad, small = [1, 2, 3], [0, 8] + ([5, 6] if dtype == torch.bfloat16 else [])  # bfloat16's smallest is below 2^-100
    rest = [i for i in range(12) if i not in bad + small]
    assert bool(scales[bad].isnan().all()) and bool((scales[small] == 0).all()) and not bool(codes[bad + small].any())
    want, top = _codes(x[rest].double())
    assert torch.equal(codes[rest], want) and bool(((scales[rest].double() - top / 127).abs() <= 2 * STEP * top / 127).all())

    w = torch.ones(k, device="cuda", dtype=dtype)
    codes, scales = norm.rms_norm_int8(x, w, EPS)
    assert bool(scales[bad].isnan().all()) and bool((scales[small] == 0).all()) and not bool(codes[bad + small].any())
    assert torch.equal(codes[rest], want)
    r = torch.zeros_like(x)
    assert torch.equal(norm.fused_add_rms_norm_int8(x, r, w, EPS)[0], codes)
    assert torch.equal(r.nan_to_num(nan=7.0), x.nan_to_num(nan=7.0))  # infinities: the type's largest, as in x
    for value in (float("inf"), float("nan")):
        w[k - 3] = value
        codes, scales = norm.rms_norm_int8(x, w, EPS)
        assert bool(scales.isnan().all()) and not bool(codes.any())
    w[k - 3] = 0
    w[:] = 0
    codes, scales = norm.rms_norm_int8(x[9:], w, EPS)
    assert not bool(scales.any()) and not bool(codes.any())


@pytest.mark.gpu
@pytest.mark.parametrize("k", [16, 528, 4096, 16384])
def test_squares_past_float32(k):
    """A norm whose sum of squares float32 does not hold has scale NaN, never 0; next to it, k squares of 2^(126 / 2) / sqrt(k), it is right."""
    x, w = torch.ones(5, k, device="cuda", dtype=torch.bfloat16), torch.ones(k, device="cuda", dtype=torch.bfloat16)
    x[0] *= 2.0 ** 65
    x[1, k // 2] = -2.0 ** 100
    x[2] *= 2.0 ** 63 * k ** -0.5
    x[3] *= 2.0 ** -90
    codes, scales = norm.rms_norm_int8(x, w, 0.0)
    assert bool(scales[[0, 1, 3]].isnan().all())  # row 3: its squares are 0 and so is eps
    assert bool((codes[[2, 4]] == 127).all())
    assert bool(((scales[[2, 4]].double() * 127 - 1).abs() <= 36 * STEP).all())  # equal values: the norm is 1
    codes, scales = norm.rms_norm_int8(x, w, EPS)
    want = 2.0 ** -90 * EPS ** -0.5 / 127
    assert abs(float(scales[3].double()) / want - 1) <= 36 * STEP and bool((codes[3] == 127).all())
    y, _ = w8._token_int8(x[:1], None, w, EPS, torch.ones(4, k, device="cuda", dtype=torch.int8), torch.ones(4, device="cuda"), False)
    assert bool(y.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strides_and_shared_buffers(dtype):
    """Rows inside wider ones; x and the residual beside each other in one buffer; what lies around them is left alone."""
    m, k = 37, 1040
    wide = _rows(m, 2 * k + 64, dtype, seed=1)
    before = wide.clone()
    w = (0.5 + torch.rand(k, device="cuda")).to(dtype)
    x, r = wide[:, 16:16 + k], wide[:, 48 + k:48 + 2 * k]
    s = x.float() + r.float()
    assert torch.equal(w8.quantize_int8(x)[0], _codes(x.double())[0])
    codes, _, out = norm.fused_add_rms_norm_int8(x, r, w, EPS)
    assert torch.equal(codes, _codes(s.double() * w.double())[0]) and torch.equal(out, s.to(dtype))
    before[:, 48 + k:48 + 2 * k] = s.to(dtype)
    assert torch.equal(wide, before)
    with pytest.raises(RuntimeError, match="memory of its own"):
        norm.fused_add_rms_norm_int8(x, x, w, EPS)
    with pytest.raises(RuntimeError, match="memory of its own"):
        norm.fused_add_rms_norm_int8(x, wide[:, 32:32 + k], w, EPS)
    with pytest.raises(RuntimeError, match="aligned"):
        w8.quantize_int8(wide[:, 4:4 + k])
    assert w8.quantize_int8(x[:0])[0].shape == (0, k) and norm.rms_norm_int8(x[:0], w, EPS)[1].shape == (0,)
    with pytest.raises(RuntimeError, match="inference only"):
        w8.quantize_int8(x.clone().requires_grad_())
    one = wide[3:4, 16:16 + k]
    assert torch.equal(w8.quantize_int8(one)[0], w8.quantize_int8(x)[0][3:4])


@pytest.mark.gpu
def test_past_32_bits():
    """More than 2^32 bytes of values and of codes."""
    m, k = 150001, 32768
    x = torch.empty(m, k, dtype=torch.float16, device="cuda").normal_()
    at = torch.tensor([0, 1, 65535, 65536, 131072, m - 1], device="cuda")
    kept = x[at]
    codes, scales = w8.quantize_int8(x)
    want, top = _codes(kept.double())
    assert torch.equal(codes[at], want) and bool(((scales[at].double() - top / 127).abs() <= 2 * STEP * top / 127).all())
    del codes
    w = (0.5 + torch.rand(k, device="cuda")).half()
    r = torch.ones_like(x)
    codes, _, _ = norm.fused_add_rms_norm_int8(x, r, w, EPS)
    s = kept.float() + 1
    assert torch.equal(codes[at], _codes(s.double() * w.double())[0]) and torch.equal(r[at], s.half())
