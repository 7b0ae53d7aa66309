"""Query / key head norms and rotary positions in one pass, into the paged cache or into tensors of their own.

    rotary_table       cosines and sines of every position                 python/tandem/layers/rotary.py
    norm_rope          rotated queries and keys as tensors
    norm_rope_cache    rotated queries as a tensor, keys and values into their slots of the cache
                                                                           python/tandem/layers/triton_ops.py:22-99

A head x of D values becomes y = x rsqrt(mean(x^2) + eps) weight (no weight: y = x), and then, with the angle a_i of its
token's position, (y[i] cos a_i - y[i + D/2] sin a_i, y[i + D/2] cos a_i + y[i] sin a_i): the halves of a head rotate
against each other, as in the Qwen3 and Llama checkpoints of Hugging Face. fp32 arithmetic, one rounding. float16 and
bfloat16, heads of 64 or 128 values. Inference only: a projection or a cache that a gradient, tangent or transform follows is
refused, and the weights and the table are taken as values, as in layers/norm.py.
"""

from __future__ import annotations

import functools

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


def layout(t: torch.Tensor) -> tuple:
    """(shape, strides, dtype, GPU index or -1): what the checks below go by."""
    return t.shape, t.stride(), t.dtype, t.get_device()


def check_cache(who: str, k: tuple, v: tuple, dtype: torch.dtype, index: int, kv_heads: int | None,
                head_dim: int) -> tuple[int, int, int]:
    """The cache's checks, shared by its writer and its reader, on the layouts of keys and values: [pages, KV heads, page size, head_dim],
    both alike. Returns (pages, KV heads, page size)."""
    shape, strides = k[0], k[1]
    if (len(shape) != 4 or shape != v[0] or shape[3] != head_dim or (kv_heads is not None and shape[1] != kv_heads)
            or shape[2] not in PAGE_SIZES):
        raise RuntimeError(f"{who}: caches [pages, {'KV heads' if kv_heads is None else kv_heads}, page size, {head_dim}] with a "
                           f"page size of {PAGE_SIZES} expected (got {tuple(shape)} and {tuple(v[0])})")
    if k[2:] != (dtype, index) or v[2:] != (dtype, index):
        raise RuntimeError(f"{who}: caches of {dtype} on GPU {index} expected (got {k[2]} on {k[3]}, {v[2]} on {v[3]})")
    if v[1] != strides or strides[3] != 1 or any(s % 8 for s in strides[:3]):
        raise RuntimeError(f"{who}: caches of one layout, heads contiguous and 16-byte aligned (strides {strides}, {v[1]})")
    return shape[0], shape[1], shape[2]


def check_int32(who: str, name: str, t: tuple, shape: tuple[int, ...], index: int) -> None:
    if t[2] != torch.int32 or t[0] != shape or t[3] != index or (shape[0] > 1 and t[1] != (1,)):
        raise RuntimeError(f"{who}: {name} must be a contiguous int32 tensor {list(shape)} on GPU {index} "
                           f"(got {t[2]} {list(t[0])} on {t[3]})")


# Every check of a call but those of addresses and of who follows it, once for each combination of layouts: an eager call is bound by
# the host (a decode step's, 16.6 -> 13.0 us).
@functools.lru_cache(maxsize=1 << 12)
def _checked(who: str, qkv: tuple, positions: tuple, table: tuple, heads: int, kv_heads: int, q_weight: tuple | None,
             k_weight: tuple | None, k: tuple | None, v: tuple | None, slots: tuple | None) -> tuple:
    """(row stride, head_dim, cache's pages, page size and strides, type code, GPU)."""
    shape, stride, dtype, index = qkv
    if not (index >= 0 and len(shape) == 2 and dtype in TYPES and stride[1] == 1):
        raise RuntimeError(f"{who}: qkv must be float16 or bfloat16 GPU rows [tokens, (heads + 2 KV heads) head_dim] "
                           f"(got {tuple(shape)}, {dtype})")
    if not (len(table[0]) == 2 and table[2] == torch.float32 and table[1] == (table[0][1], 1) and table[3] == index and table[0][0] >= 1):
        raise RuntimeError(f"{who}: table must be a contiguous float32 tensor [positions, head_dim] on GPU {index}")
    tokens, d = shape[0], table[0][1]
    if d not in (64, 128) or not 1 <= kv_heads <= heads or shape[1] != (heads + 2 * kv_heads) * d:
        raise RuntimeError(f"{who}: heads of 64 or 128 values and rows of {heads} + 2 x {kv_heads} of them "
                           f"(head_dim {d}, rows of {shape[1]})")
    if tokens > 1 and (stride[0] % 8 or stride[0] < shape[1]):
        raise RuntimeError(f"{who}: rows of qkv must not overlap and be 16-byte aligned (stride {stride[0]})")
    check_int32(who, "positions", positions, (tokens,), index)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and w != ((d,), (1,), dtype, index):
            raise RuntimeError(f"{who}: {name} must be a contiguous {dtype} tensor [{d}] on GPU {index}")
    cache: tuple = (0, 0, 0, 0, 0)
    if k is not None:
        pages, _, size = check_cache(who, k, v, dtype, index, kv_heads, d)
        room = d
        for step, n in sorted(zip(k[1][:3], k[0][:3])):
            if n > 1 and step < room:
                raise RuntimeError(f"{who}: the caches' places must not overlap (strides {k[1]})")
            room = max(room, step * (n - 1) + room)
        check_int32(who, "slots", slots, (tokens,), index)
        cache = (pages, size, *k[1][:3])
    return stride[0] if tokens > 1 else shape[1], d, cache, TYPES[dtype], index


def _run(who: str, qkv, positions, table, num_heads: int, num_kv_heads: int, q_weight, k_weight, eps: float, k, v, slots):
    stride, d, cache, code, index = _checked(who, layout(qkv), layout(positions), layout(table), num_heads, num_kv_heads,
                                             None if q_weight is None else layout(q_weight),
                                             None if k_weight is None else layout(k_weight), None if k is None else layout(k),
                                             None if v is None else layout(v), None if slots is None else layout(slots))
    if not (w4_hip.plain(qkv) if slots is None else w4_hip.all_plain(qkv, k, v)):
        raise RuntimeError(f"{who}: inference only, no gradient, transform or tracer can follow qkv or the caches")
    tokens = qkv.shape[0]
    q = qkv.new_empty((tokens, num_heads, d))
    if slots is None:
        k = qkv.new_empty((tokens, num_kv_heads, d))
    if tokens:
        xp, tp, kp, vp = qkv.data_ptr(), table.data_ptr(), k.data_ptr(), 0 if v is None else v.data_ptr()
        qw, kw = 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr()
        if kp == vp:
            raise RuntimeError(f"{who}: keys and values need memory of their own")
        if (xp | tp | kp | vp | qw | kw) % 16:
            raise RuntimeError(f"{who}: qkv, the table, weights and caches must be 16-byte aligned")
        with w4_hip.on_device(index):
            w4_hip.check(w4_hip.library().tw4_norm_rope(
                xp, stride, positions.data_ptr(), tp, table.shape[0], qw, kw, eps, q.data_ptr(), kp, vp,
                None if slots is None else slots.data_ptr(), *cache, tokens, num_heads, num_kv_heads, d, code,
                w4_hip.raw_stream(index)))
    return q, k


def norm_rope(qkv: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, num_heads: int, num_kv_heads: int,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """qkv [T, (heads + 2 KV heads) head_dim] = [q | k | v], positions int32 [T], table from rotary_table -> queries
    [T, heads, head_dim] and keys [T, KV heads, head_dim], normalised where there is a weight, and rotated (tw4_norm_rope).
    A position outside of the table gives NaN."""
    return _run("norm_rope", qkv, positions, table, num_heads, num_kv_heads, q_weight, k_weight, eps, None, None, None)


def norm_rope_cache(qkv: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, num_heads: int, num_kv_heads: int,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, q_weight: torch.Tensor | None = None,
                    k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """norm_rope whose keys, and the values as they are, go into the caches [pages, KV heads, page size, head_dim]: token t's at
    slots[t] = page * page size + offset (int32 [T]; outside of the cache: nowhere). The two caches share no place (one tensor may
    hold both, as views). Slots are distinct; of two tokens with one slot either may win, head by head. Returns the queries [T,
    heads, head_dim]."""
    return _run("norm_rope_cache", qkv, positions, table, num_heads, num_kv_heads, q_weight, k_weight, eps, k_cache,
                v_cache, slots)[0]
