"""Projections in 8-bit integers: weights with a scale for each output feature, activations with a scale for each token, products on
the integer matrix cores.

    quantize_int8    rows of activations -> codes and scales
    linear_int8      the product, with SwiGLU if asked for
    W8Linear         the module: a projection of an int8 checkpoint, beside layers/awq.py's W4Linear

A number is code * scale, codes in -127 .. 127 (weights: -128 .. 127). layers/norm.py's rms_norm_int8 and fused_add_rms_norm_int8 write
the activations of a projection that a norm stands before. float16 and bfloat16. Inference only. No reference counterpart: the
reference's engine has 4-bit projections only (python/tandem/layers/awq.py).
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch import nn

from tandem_amd.layers import norm, w4_hip
from tandem_amd.layers.rotary import TYPES, layout


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (float16 or bfloat16, any row stride, K % 16 == 0) in 8 bits (tw4_quantize_int8): (codes int8 [M, K], scales
    float32 [M]), scale = max|x| / 127, code = 127 x / max|x| exactly, rounded to nearest, halves to even.

    A row that holds an infinity or a NaN has scale NaN and codes 0, so that its products are NaN; one with every |x| below
    2^-100 has scale 0 and codes 0."""
    step, _, m, k, code, index = norm.check_rows("quantize_int8", layout(x), None, None)
    if not w4_hip.plain(x):
        raise RuntimeError("quantize_int8: inference only, no gradient, transform or tracer can follow x")
    codes, scales = x.new_empty(m, k, dtype=torch.int8), x.new_empty(m, dtype=torch.float32)
    if m:
        xp = x.data_ptr()
        if xp % 16:
            raise RuntimeError("quantize_int8: x must be 16-byte aligned")
        with w4_hip.on_device(index):
            w4_hip.check(w4_hip.library().tw4_quantize_int8(xp, step, codes.data_ptr(), scales.data_ptr(), m, k, code,
                                                            w4_hip.raw_stream(index)))
    return codes, scales


@functools.lru_cache(maxsize=None)
def _cus(index: int) -> int:
    return torch.cuda.get_device_properties(index).multi_processor_count


# As norm.check_rows: what depends on layouts alone, once for each combination of them.
@functools.lru_cache(maxsize=1 << 14)
def _checked(x: tuple, x_scale: tuple, weight: tuple, weight_scale: tuple, silu_mul: bool, dtype: torch.dtype) -> tuple:
    """(row strides of x and of the weight, (M, N, K, act, type code, kernel, splits), whether those take a workspace,
    output features, GPU)."""
    index = x[3]
    steps = []
    for name, t in (("x", x), ("weight", weight)):
        if not (t[3] == index >= 0 and len(t[0]) == 2 and t[2] == torch.int8 and t[1][1] == 1):
            raise RuntimeError(f"linear_int8: {name} must be int8 rows on x's GPU (got {tuple(t[0])}, {t[2]})")
        steps.append(t[1][0] if t[0][0] > 1 else t[0][1])
        if steps[-1] < t[0][1] or steps[-1] % 16 or steps[-1] >= 1 << 22:
            raise RuntimeError(f"linear_int8: rows of {name} must not overlap, be 16-byte aligned and less than 2^22 apart "
                               f"(stride {steps[-1]})")
    (m, k), (n, wk) = x[0], weight[0]
    if k != wk or k % 16 or not 16 <= k < 1 << 17:
        raise RuntimeError(f"linear_int8: x [M, K] and weight [N, K] with K % 16 == 0 and K < 2^17 (got {tuple(x[0])}, {tuple(weight[0])})")
    if not (1 <= n <= 1 << 24 and m <= 1 << 20) or (silu_mul and n % 2):
        raise RuntimeError(f"linear_int8: M <= 2^20, 1 <= N <= 2^24, and an even N with silu_mul (M {m}, N {n})")
    for name, t, rows in (("x_scale", x_scale, m), ("weight_scale", weight_scale, n)):
        if t[0] not in ((rows,), (rows, 1)) or t[2:] != (torch.float32, index) or (rows > 1 and t[1][0] != 1):
            raise RuntimeError(f"linear_int8: {name} must be a contiguous float32 tensor [{rows}] or [{rows}, 1] on x's GPU")
    if dtype not in TYPES:
        raise RuntimeError(f"linear_int8: the result is float16 or bfloat16 (asked for {dtype})")
    plan = (ctypes.c_int * 4)(0, 1)
    if m:
        w4_hip.check(w4_hip.library().tw4_gemm_int8_plan(m, n, k, int(silu_mul), _cus(index), plan))
    return *steps, (m, n, k, int(silu_mul), TYPES[dtype], plan[0], plan[1]), plan[2] > 0, n // 2 if silu_mul else n, index


def linear_int8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                silu_mul: bool = False, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """x int8 [M, K], x_scale float32 [M], weight int8 [N, K], weight_scale float32 [N] (both scales also [.., 1]) -> y [M, N] of
    ``dtype``: y[m, n] = x_scale[m] * weight_scale[n] * sum_k x[m, k] weight[n, k], the sum exact, one rounding (tw4_gemm_int8).
    silu_mul: the weight's rows are [gate | up] and y [M, N / 2] = silu(gate) * up, gate and up in float32. K % 16 == 0, K < 2^17;
    any row strides of x and weight that are multiples of 16."""
    step, w_step, sizes, split, features, index = _checked(layout(x), layout(x_scale), layout(weight), layout(weight_scale),
                                                           bool(silu_mul), dtype)
    if not w4_hip.all_plain(x, x_scale, weight, weight_scale):
        raise RuntimeError("linear_int8: inference only, no gradient, transform or tracer can follow the operands")
    y = x.new_empty(sizes[0], features, dtype=dtype)
    if sizes[0]:
        xp, wp = x.data_ptr(), weight.data_ptr()
        if (xp | wp) % 16:
            raise RuntimeError("linear_int8: x and the weight must be 16-byte aligned")
        with w4_hip.on_device(index):
            wsp = locksp = words = counters = 0
            if split:
                ws, locks = w4_hip.stream_workspace(x.device)
                wsp, locksp, words, counters = ws.data_ptr(), locks.data_ptr(), ws.numel(), locks.numel()
            w4_hip.check(w4_hip.library().tw4_gemm_int8(xp, step, x_scale.data_ptr(), wp, w_step, weight_scale.data_ptr(), y.data_ptr(),
                                                        wsp, words, locksp, counters, *sizes, w4_hip.raw_stream(index)))
    return y


MAX_TOKEN_K = 16384


# As _checked. x's own stride is no matter: it is one row.
@functools.lru_cache(maxsize=1 << 14)
def _checked_token(x: tuple, residual: tuple | None, norm_weight: tuple | None, weight: tuple, weight_scale: tuple,
                   silu_mul: bool) -> tuple:
    """((N, K, act, type code, CUs), row stride of the weight, output features, GPU)."""
    _, _, _, k, code, index = norm.check_rows("token_int8", x, residual, norm_weight)
    one = ((1, k), (k, 1), torch.int8, index), ((1,), (1,), torch.float32, index)
    _, w_step, (_, n, k, act, *_), _, features, _ = _checked(*one, weight, weight_scale, silu_mul, x[2])
    return (n, k, act, code, _cus(index)), w_step, features, index


def _token_int8(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor | None, eps: float, weight: torch.Tensor,
                weight_scale: torch.Tensor, silu_mul: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    """linear_int8 of one row x [1, K] in 8 bits, K <= MAX_TOKEN_K, in one kernel: quantize_int8's codes, or with norm_weight rms_norm_int8's,
    or with residual fused_add_rms_norm_int8's -> (y, x + residual in new memory). The bits of the two calls (tw4_token_int8)."""
    sizes, w_step, features, index = _checked_token(layout(x), None if residual is None else layout(residual),
                                                    None if norm_weight is None else layout(norm_weight), layout(weight),
                                                    layout(weight_scale), silu_mul)
    operands = (x, weight, weight_scale) if norm_weight is None else (x, weight, weight_scale, norm_weight)
    if not w4_hip.all_plain(*(operands if residual is None else (*operands, residual))):
        raise RuntimeError("token_int8: inference only, no gradient, transform or tracer can follow the operands")
    y, total = x.new_empty(1, features), None if residual is None else x.new_empty(1, sizes[1])
    xp, wp = x.data_ptr(), weight.data_ptr()
    rp, tp = (0, 0) if residual is None else (residual.data_ptr(), total.data_ptr())
    gp = 0 if norm_weight is None else norm_weight.data_ptr()
    if (xp | wp | rp | gp) % 16:
        raise RuntimeError("token_int8: x, the residual and the weights must be 16-byte aligned")
    with w4_hip.on_device(index):
        w4_hip.check(w4_hip.library().tw4_token_int8(xp, rp, tp, gp, eps, wp, w_step, weight_scale.data_ptr(), y.data_ptr(), *sizes,
                                                     w4_hip.raw_stream(index)))
    return y, total


class W8Linear(nn.Module):
    """y = x @ W^T for a bias-free projection of an int8 checkpoint: ``weight`` int8 [N, K] and ``weight_scale`` float32 [N, 1], as
    such checkpoints store them (a fused qkv or gate_up holds its parts one behind the other). x is quantised token by token on
    the way in; y has x's type. Nothing is laid out anew, so a layer is ready once loaded and on the GPU. forward_norm and
    enable_silu_mul are W4Linear's (layers/awq.py)."""

    def __init__(self, in_features: int, out_features: int) -> None:
        super().__init__()
        if in_features % 16 or not 16 <= in_features <= norm.MAX_INT8_ROW or out_features < 1:
            raise ValueError(f"W8Linear({in_features}, {out_features}): K a multiple of 16 up to {norm.MAX_INT8_ROW}, N >= 1")
        self.in_features, self.out_features = in_features, out_features
        self.silu_mul = False
        self.register_buffer("weight", torch.empty(out_features, in_features, dtype=torch.int8))
        self.register_buffer("weight_scale", torch.empty(out_features, 1, dtype=torch.float32))

    def _apply(self, fn, recurse: bool = True):
        """Module.to, with the scales left in float32 where it changes floating types."""
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def enable_silu_mul(self) -> bool:
        """forward returns silu(gate) * up, [M, out_features / 2]."""
        self.silu_mul = self.out_features % 2 == 0
        return self.silu_mul

    def _one_token(self, x: torch.Tensor) -> bool:
        """Whether x's codes are made inside the product's kernel: one row, with as many outputs as one workgroup for each CU holds. Measured
        on both sides in csrc/tw4_gemm8.hip."""
        outputs, each = (self.out_features // 2, 16) if self.silu_mul else (self.out_features, 32)
        return x.shape[0] == 1 and self.in_features <= MAX_TOKEN_K and x.is_cuda and outputs <= each * _cus(x.get_device())

    def _product(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        return linear_int8(codes, scales, self.weight, self.weight_scale, silu_mul=self.silu_mul, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() != 2:
            y = self(x.reshape(-1, self.in_features))
            return y.view(*x.shape[:-1], y.shape[-1])
        if self._one_token(x):
            return _token_int8(x, None, None, 0.0, self.weight, self.weight_scale, self.silu_mul)[0]
        return self._product(*quantize_int8(x), x.dtype)

    def forward_norm(self, x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor,
                     eps: float) -> tuple[torch.Tensor, torch.Tensor]:
        """self(rms_norm(x + residual) * norm_weight), the norm's output in 8 bits as it is written, and the new residual (x itself without
        one). residual is consumed, as W4Linear's: one token gets the new one in fresh memory, more have it written in place. Rows [M, K] only. It
        does not go through forward: hooks on the layer do not see it."""
        if x.dim() == 2 and self._one_token(x):
            y, total = _token_int8(x, residual, norm_weight, eps, self.weight, self.weight_scale, self.silu_mul)
            return y, x if residual is None else total
        if residual is None:
            return self._product(*norm.rms_norm_int8(x, norm_weight, eps), x.dtype), x
        codes, scales, residual = norm.fused_add_rms_norm_int8(x, residual, norm_weight, eps)
        return self._product(codes, scales, x.dtype), residual
