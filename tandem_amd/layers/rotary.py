"""Query / key head norms and rotary positions in one pass, into the paged cache or into tensors of their own.

    rotary_table       cosines and sines of every position                 python/tandem/layers/rotary.py
    norm_rope          rotated queries and keys as tensors
    norm_rope_cache    rotated queries as a tensor, keys and values into their slots of the cache
                                                                           python/tandem/layers/triton_ops.py:22-99

A head x of D values becomes y = x rsqrt(mean(x^2) + eps) weight (no weight: y = x), and then, with the angle a_i of its
token's position, (y[i] cos a_i - y[i + D/2] sin a_i, y[i + D/2] cos a_i + y[i] sin a_i): the halves of a head rotate
against each other, as in the Qwen3 and Llama checkpoints of Hugging Face. fp32 arithmetic, one rounding. float16 and
bfloat16, heads of 64 or 128 values. Inference only: tensors that autograd follows are refused.
"""

from __future__ import annotations

import torch

from tandem_amd.layers import w4_hip

TYPES = {torch.float16: 0, torch.bfloat16: 1}
PAGE_SIZES = (16, 32, 64, 128, 256)


def rotary_table(positions: int, head_dim: int, theta: float, device: torch.device | str | None = None) -> torch.Tensor:
    """float32 [positions, head_dim]: cos, then sin, of position * theta^(-2 i / head_dim), i < head_dim / 2. The angles and
    their functions in 64 bits: at position 40000 an angle of 32 bits is off by 2e-3."""
    if positions < 1 or head_dim < 2 or head_dim % 2 or not theta > 0:
        raise ValueError(f"rotary_table: positions >= 1, an even head_dim and theta > 0 (got {positions}, {head_dim}, {theta})")
    i = torch.arange(head_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * theta ** (-2.0 * i / head_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def check_cache(who: str, k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, kv_heads: int | None,
                head_dim: int) -> tuple[int, int, int]:
    """The cache's checks, shared by its writer and its reader: keys and values [pages, KV heads, page size, head_dim] of one
    shape and layout. Returns (pages, KV heads, page size)."""
    if (k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[3] != head_dim
            or (kv_heads is not None and k_cache.shape[1] != kv_heads) or k_cache.shape[2] not in PAGE_SIZES):
        raise RuntimeError(f"{who}: caches [pages, {'KV heads' if kv_heads is None else kv_heads}, page size, {head_dim}] with a "
                           f"page size of {PAGE_SIZES} expected (got {tuple(k_cache.shape)} and {tuple(v_cache.shape)})")
    if k_cache.dtype != like.dtype or v_cache.dtype != like.dtype or k_cache.device != like.device or v_cache.device != like.device:
        raise RuntimeError(f"{who}: caches of {like.dtype} on {like.device} expected (got {k_cache.dtype} on {k_cache.device}, "
                           f"{v_cache.dtype} on {v_cache.device})")
    strides = k_cache.stride()
    if (v_cache.stride() != strides or strides[3] != 1 or any(s % 8 for s in strides[:3]) or k_cache.data_ptr() % 16
            or v_cache.data_ptr() % 16):
        raise RuntimeError(f"{who}: caches of one layout, heads contiguous and 16-byte aligned (strides {strides}, {v_cache.stride()})")
    return k_cache.shape[0], k_cache.shape[1], k_cache.shape[2]


def check_int32(who: str, name: str, t: torch.Tensor, shape: tuple[int, ...], like: torch.Tensor) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
        raise RuntimeError(f"{who}: {name} must be a contiguous int32 tensor {list(shape)} on {like.device} "
                           f"(got {t.dtype} {list(t.shape)} on {t.device})")


def _run(who: str, qkv, positions, table, num_heads: int, num_kv_heads: int, q_weight, k_weight, eps: float, cache, slots):
    if not (qkv.is_cuda and qkv.dim() == 2 and qkv.dtype in TYPES and qkv.stride(1) == 1):
        raise RuntimeError(f"{who}: qkv must be float16 or bfloat16 GPU rows [tokens, (heads + 2 KV heads) head_dim] "
                           f"(got {tuple(qkv.shape)}, {qkv.dtype})")
    if not w4_hip.plain(qkv):
        raise RuntimeError(f"{who}: inference only, no gradient, transform or tracer can follow qkv")
    if not (table.dim() == 2 and table.dtype == torch.float32 and table.is_contiguous() and table.device == qkv.device
            and table.shape[0] >= 1 and table.data_ptr() % 16 == 0):
        raise RuntimeError(f"{who}: table must be a contiguous float32 tensor [positions, head_dim] on {qkv.device}")
    tokens, d, dev = qkv.shape[0], table.shape[1], qkv.device
    if d not in (64, 128) or not 1 <= num_kv_heads <= num_heads or qkv.shape[1] != (num_heads + 2 * num_kv_heads) * d:
        raise RuntimeError(f"{who}: heads of 64 or 128 values and rows of {num_heads} + 2 x {num_kv_heads} of them "
                           f"(head_dim {d}, rows of {qkv.shape[1]})")
    if (tokens > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < qkv.shape[1])) or qkv.data_ptr() % 16:
        raise RuntimeError(f"{who}: rows of qkv must not overlap and be 16-byte aligned (stride {qkv.stride(0)})")
    check_int32(who, "positions", positions, (tokens,), qkv)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.dtype != qkv.dtype or w.device != dev or not w.is_contiguous()
                              or w.data_ptr() % 16):
            raise RuntimeError(f"{who}: {name} must be a contiguous 16-byte aligned {qkv.dtype} tensor [{d}] on {dev}")
    pages = size = 0
    strides = (0, 0, 0)
    if cache is not None:
        pages, _, size = check_cache(who, *cache, qkv, num_kv_heads, d)
        strides = cache[0].stride()[:3]
        check_int32(who, "slots", slots, (tokens,), qkv)
    q = torch.empty((tokens, num_heads, d), dtype=qkv.dtype, device=dev)
    k, v = cache if cache is not None else (torch.empty((tokens, num_kv_heads, d), dtype=qkv.dtype, device=dev), None)
    if tokens:
        index = qkv.get_device()
        with w4_hip.on_device(index):
            w4_hip.check(w4_hip.library().tw4_norm_rope(
                qkv.data_ptr(), max(qkv.stride(0), qkv.shape[1]), positions.data_ptr(), table.data_ptr(), table.shape[0],
                None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), float(eps),
                q.data_ptr(), k.data_ptr(), None if v is None else v.data_ptr(), None if slots is None else slots.data_ptr(),
                pages, size, *strides, tokens, num_heads, num_kv_heads, d, TYPES[qkv.dtype], w4_hip.raw_stream(index)))
    return q, k


def norm_rope(qkv: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, num_heads: int, num_kv_heads: int,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """qkv [T, (heads + 2 KV heads) head_dim] = [q | k | v], positions int32 [T], table from rotary_table -> queries
    [T, heads, head_dim] and keys [T, KV heads, head_dim], normalised where there is a weight, and rotated (tw4_norm_rope).
    A position outside of the table gives NaN."""
    return _run("norm_rope", qkv, positions, table, num_heads, num_kv_heads, q_weight, k_weight, eps, None, None)


def norm_rope_cache(qkv: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, num_heads: int, num_kv_heads: int,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, q_weight: torch.Tensor | None = None,
                    k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """norm_rope whose keys, and the values as they are, go into the caches [pages, KV heads, page size, head_dim]: token t's
    at slots[t] = page * page size + offset (int32 [T]; outside of the cache: nowhere). Slots are distinct; of two tokens
    with one slot either may win. Returns the queries [T, heads, head_dim]."""
    return _run("norm_rope_cache", qkv, positions, table, num_heads, num_kv_heads, q_weight, k_weight, eps, (k_cache, v_cache),
                slots)[0]
