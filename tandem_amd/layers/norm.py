"""RMSNorm and residual-add + RMSNorm around the W4A16 projections, on libtandem_w4.so.

The decoder layer's small per-token kernels that sit between the projections of a decode step
(python/tandem/models/llama_family.py:47-67):

    RMSNorm               the module (weight, eps)                 python/tandem/layers/norm.py:7-19
    HipOps.rms_norm       y = rms_norm(x) * w                      python/tandem/layers/ops.py:107-109
    HipOps.fused_add_rms_norm  residual <- x + residual; x <- rms_norm(residual) * w, in place
                                                                   python/tandem/layers/ops.py:111-120
    rms_norm_int8, fused_add_rms_norm_int8
                          the same with their output in 8 bits and a scale for each token, what layers/w8.py multiplies

Numerics are those of the reference's GPU path (FlashInfer's kernels and the Triton
fused_add_rmsnorm, python/tandem/layers/triton_ops.py:101-124): fp32 sum, the residual stored in
fp16, the output from the unrounded sum with one rounding. The reference's TorchOps (norm then
weight in fp16) differs from it by fp16 rounding only.
"""

from __future__ import annotations

import functools

import torch
from torch import nn

from tandem_amd.layers import w4_hip
from tandem_amd.layers.rotary import TYPES, layout


def _check(who: str, x: torch.Tensor, weight: torch.Tensor) -> tuple[int, int]:
    if x.dim() != 2 or not x.is_contiguous() or x.dtype != torch.float16 or not x.is_cuda:
        raise RuntimeError(f"{who}: contiguous float16 [M, K] GPU rows expected (got {tuple(x.shape)}, {x.dtype})")
    if (weight.shape != (x.shape[1],) or weight.dtype != torch.float16 or weight.device != x.device
            or not weight.is_contiguous()):
        raise RuntimeError(f"{who}: contiguous float16 weight [{x.shape[1]}] on x's GPU expected")
    return x.shape[0], x.shape[1]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = fp16(x * rsqrt(mean(x^2) + eps) * weight) over the last dimension (tw4_rms_norm)."""
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    m, k = _check("rms_norm", x2, weight)
    if out is None:
        y = torch.empty_like(x2)
    elif (out.shape != x.shape or out.dtype != torch.float16 or out.device != x.device or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise RuntimeError(f"rms_norm: out must be a contiguous 16-byte aligned float16 tensor shaped like x "
                           f"{tuple(shape)} on x's GPU")
    else:
        y = out.view(m, k)
    if m == 0:
        return y.view(shape)
    with w4_hip.on_device(x.get_device()):
        w4_hip.check(w4_hip.library().tw4_rms_norm(x2.data_ptr(), weight.data_ptr(), y.data_ptr(), m, k, float(eps),
                                                   w4_hip.raw_stream(x.get_device())))
    return y.view(shape)


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """In place: residual <- x + residual, x <- rms_norm(residual) * weight (tw4_add_rms_norm).
    Returns (x, residual)."""
    m, k = _check("fused_add_rms_norm", x, weight)
    if residual.shape != x.shape or residual.dtype != x.dtype or not residual.is_contiguous() \
            or residual.device != x.device:
        raise RuntimeError("fused_add_rms_norm: residual must match x")
    if m == 0:
        return x, residual
    with w4_hip.on_device(x.get_device()):
        w4_hip.check(w4_hip.library().tw4_add_rms_norm(x.data_ptr(), residual.data_ptr(), weight.data_ptr(), m, k,
                                                       float(eps), w4_hip.raw_stream(x.get_device())))
    return x, residual


MAX_INT8_ROW = 32768


# Every check of a call but those of addresses and of who follows it, once for each combination of layouts, as in layers/rotary.py.
@functools.lru_cache(maxsize=1 << 12)
def check_rows(who: str, x: tuple, residual: tuple | None, weight: tuple | None) -> tuple[int, int, int, int, int, int]:
    """(row strides of x and of the residual, M, K, type code, GPU)."""
    shape, stride, dtype, index = x
    if not (index >= 0 and len(shape) == 2 and dtype in TYPES and stride[1] == 1):
        raise RuntimeError(f"{who}: float16 or bfloat16 GPU rows [M, K] expected (got {tuple(shape)}, {dtype})")
    m, k = shape
    if k % 16 or not 16 <= k <= MAX_INT8_ROW:
        raise RuntimeError(f"{who}: K % 16 == 0 and 16 <= K <= {MAX_INT8_ROW} (K = {k})")
    steps = [k, k]
    for i, (name, t) in enumerate((("x", x), ("residual", residual))):
        if t is None:
            continue
        if t[0] != shape or t[2:] != (dtype, index) or t[1][1] != 1:
            raise RuntimeError(f"{who}: {name} must match x")
        if m > 1:
            steps[i] = t[1][0]
            if steps[i] < k or steps[i] % 8:
                raise RuntimeError(f"{who}: rows of {name} must not overlap and be 16-byte aligned (stride {steps[i]})")
    if weight is not None and weight != ((k,), (1,), dtype, index):
        raise RuntimeError(f"{who}: contiguous {dtype} weight [{k}] on x's GPU expected")
    return steps[0], steps[1], m, k, TYPES[dtype], index


def _apart(a: int, step_a: int, b: int, step_b: int, rows: int, width: int) -> bool:
    """Whether rows of ``width`` bytes from addresses a and b on, so many bytes apart, share no byte."""
    if a + (rows - 1) * step_a + width <= b or b + (rows - 1) * step_b + width <= a:
        return True
    return step_a == step_b and width <= (b - a) % step_a <= step_a - width


def _rms_norm_int8(who: str, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                   eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    step, r_step, m, k, code, index = check_rows(who, layout(x), None if residual is None else layout(residual), layout(weight))
    if not (w4_hip.all_plain(x, weight) if residual is None else w4_hip.all_plain(x, residual, weight)):
        raise RuntimeError(f"{who}: inference only, no gradient, transform or tracer can follow x, the residual or the weight")
    codes, scales = x.new_empty(m, k, dtype=torch.int8), x.new_empty(m, dtype=torch.float32)
    if m:
        xp, rp, wp = x.data_ptr(), 0 if residual is None else residual.data_ptr(), weight.data_ptr()
        if (xp | rp | wp) % 16:
            raise RuntimeError(f"{who}: x, the residual and the weight must be 16-byte aligned")
        if rp and not _apart(xp, 2 * step, rp, 2 * r_step, m, 2 * k):
            raise RuntimeError(f"{who}: the residual needs memory of its own")
        with w4_hip.on_device(index):
            w4_hip.check(w4_hip.library().tw4_rms_norm_int8(xp, step, rp, r_step, wp, eps, codes.data_ptr(), scales.data_ptr(), m,
                                                            k, code, w4_hip.raw_stream(index)))
    return codes, scales


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """rms_norm(x) * weight of rows [M, K] (float16 or bfloat16, any row stride, K % 16 == 0) in 8 bits (tw4_rms_norm_int8):
    (codes int8 [M, K], scales float32 [M]), value = code * scale, scale = max|y| / 127 of the unrounded norm y. 1 / rms is
    common to a row, so code = 127 t / max|t| with t = x * weight, and is exactly that, rounded to nearest, halves to even.

    A row that holds an infinity or a NaN (in x, the weight, or their product in float32) has scale NaN and codes 0, so that
    its products are NaN; one with every |t| below 2^-100 has scale 0 and codes 0. One whose sum of squares leaves float32 (bfloat16
    from about 10^18 on; with eps 0, all below 10^-22) has scale NaN too. Inference only: an x, residual or weight that
    a gradient, tangent or transform follows is refused."""
    return _rms_norm_int8("rms_norm_int8", x, None, weight, eps)


def fused_add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                            eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """residual <- x + residual in place, and rms_norm_int8 of the unrounded (float32) sum: (codes, scales, residual). x is left as it
    is."""
    codes, scales = _rms_norm_int8("fused_add_rms_norm_int8", x, residual, weight, eps)
    return codes, scales, residual


class HipOps:
    """The norm half of the reference's ops interface (python/tandem/layers/ops.py:62-120) on the
    HIP kernels; the attention-side ops are in ``rotary`` and ``paged_attention``."""

    name = "hip"

    @staticmethod
    def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
        return rms_norm(x, weight, eps)

    @staticmethod
    def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                           eps: float) -> tuple[torch.Tensor, torch.Tensor]:
        return fused_add_rms_norm(x, residual, weight, eps)


class RMSNorm(nn.Module):
    """RMSNorm with a learned weight (python/tandem/layers/norm.py:7-19), on tw4_rms_norm."""

    def __init__(self, dim: int, eps: float) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.weight, self.eps)
