"""Causal attention of new tokens over a paged KV cache (python/tandem/layers/flashinfer_attention.py,
python/tandem/layers/triton_decode_attn.py), on tw4_paged_attention: a decode step's single tokens, a few drafted ones,
chunks of prompts, and any mix of them in one call."""

from __future__ import annotations

import functools
import math

import torch

from tandem_amd.layers import w4_hip
from tandem_amd.layers.rotary import TYPES, check_cache, check_int32, layout


# Every check of a call but those of addresses and of who follows it, once for each combination of layouts and sizes: an eager call
# is bound by the host (a decode step's, 16.9 -> 14.0 us).
@functools.lru_cache(maxsize=1 << 14)
def _checked(q: tuple, k: tuple, v: tuple, table: tuple, lens: tuple, starts: tuple | None, out: tuple | None, most: int | None,
             longest: int | None, scale: float | None) -> tuple:
    """(strides of q, rows of a tile, splits and what else tw4_paged_attention takes by value)."""
    who = "paged_attention"
    shape, stride, dtype, index = q
    if not (index >= 0 and len(shape) == 3 and dtype in TYPES and shape[2] in (64, 128) and stride[2] == 1):
        raise RuntimeError(f"{who}: q must be float16 or bfloat16 GPU rows [tokens, heads, 64 or 128] (got {tuple(shape)}, {dtype})")
    tokens, heads, d = shape
    if any(stride[i] % 8 for i in (0, 1) if shape[i] > 1):
        raise RuntimeError(f"{who}: rows and heads of q must be 16-byte aligned (strides {stride})")
    pages, kv_heads, size = check_cache(who, k, v, dtype, index, None, d)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise RuntimeError(f"{who}: heads must be a multiple of the cache's KV heads ({heads}, {kv_heads})")
    if len(table[0]) != 2 or table[2] != torch.int32 or table[3] != index or (table[0][1] > 1 and table[1][1] != 1):
        raise RuntimeError(f"{who}: page_table must be int32 [requests, pages per request] on q's GPU, rows contiguous "
                           f"(got {table[2]} {tuple(table[0])})")
    batch, width = table[0]
    check_int32(who, "seq_lens", lens, (batch,), index)
    if starts is not None:
        check_int32(who, "query_start", starts, (batch + 1,), index)
    elif tokens != batch:
        raise RuntimeError(f"{who}: without query_start there is one token per request ({tokens} tokens, {batch} requests)")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise RuntimeError(f"{who}: a positive scale (got {scale})")
    if out is not None and out != (shape, (heads * d, d, 1), dtype, index):
        raise RuntimeError(f"{who}: out must be a contiguous {dtype} tensor {list(shape)} on q's GPU")
    rows, splits = 16, 1
    if tokens and batch:
        plan = (w4_hip._I * 4)()
        w4_hip.check(w4_hip.library().tw4_paged_attention_plan(
            tokens, batch, heads, kv_heads, d, 1 if starts is None else tokens if most is None else max(min(most, tokens), 0),
            width * size if longest is None else max(min(longest, width * size), 0), int(starts is None),
            torch.cuda.get_device_properties(index).multi_processor_count, plan))
        rows, splits = plan[0], plan[1]
    return ((stride[0] if tokens > 1 else 0, stride[1] if heads > 1 else 0), (*k[1][:3], pages, size),
            (table[1][0] if batch > 1 else 0, width), (tokens, batch, heads, kv_heads, d, scale, rows, splits, TYPES[dtype]), index)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, query_start: torch.Tensor | None = None, *, max_query_len: int | None = None,
                    max_seq_len: int | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [T, heads, head_dim] (float16 or bfloat16, head_dim 64 or 128) over caches [pages, KV heads, page size,
    head_dim]. Request i of B has seq_lens[i] keys, the last of them its new tokens' own: key j lies in page
    page_table[i, j // page size]. Its new tokens are rows query_start[i] .. query_start[i + 1] - 1 of q, and the t-th of
    n = query_start[i + 1] - query_start[i] sees the keys j <= seq_lens[i] - n + t; of a request that runs past row T - 1 the tokens
    that have a row are computed. query_start None: one new token per request (T == B). Query head h reads KV head
    h // (heads / KV heads). scale: of the scores, head_dim^-0.5 by default.

    page_table int32 [B, pages per request] (any row stride), seq_lens int32 [B], query_start int32 [B + 1], ascending from 0.
    They are read on the GPU only, and nothing outside of the tensors is touched whatever they hold: keys of an entry that is no
    page, or behind the table's width, are left out, and a row that sees no key (or none with a score above -inf) is zero.
    Infinities and NaN of keys and values reach the rows that see them and no others. Rows from query_start[B] on are left as they
    were in ``out``.

    max_query_len, max_seq_len: bounds the host knows; they only choose how the work is divided (T and the table's width
    otherwise). Results do not depend on the order in which workgroups run. Inference only."""
    # the longest context in steps: a decode loop asks for a few plans only
    (q_strides, cache, (table_stride, width), sizes, index) = _checked(
        layout(q), layout(k_cache), layout(v_cache), layout(page_table), layout(seq_lens),
        None if query_start is None else layout(query_start), None if out is None else layout(out),
        max_query_len, None if max_seq_len is None else (max_seq_len + 127) // 128 * 128, scale)
    if not w4_hip.all_plain(q, k_cache, v_cache, *(() if out is None else (out,))):
        raise RuntimeError("paged_attention: inference only, no gradient, transform or tracer can follow q, the caches or out")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)  # 1 us less than torch.empty of a device
    qp, kp, vp, op = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    if (qp | kp | vp | op) % 16:
        raise RuntimeError("paged_attention: q, out and the caches must be 16-byte aligned")
    if sizes[0] == 0 or sizes[1] == 0:
        return out
    with w4_hip.on_device(index):
        wsp = locksp = floats = counters = 0
        if sizes[7] > 1:
            ws, locks = w4_hip.stream_workspace(q.device)
            wsp, locksp, floats, counters = ws.data_ptr(), locks.data_ptr(), ws.numel(), locks.numel()
        w4_hip.check(w4_hip.library().tw4_paged_attention(
            qp, *q_strides, kp, vp, *cache, page_table.data_ptr(), table_stride, width, seq_lens.data_ptr(),
            None if query_start is None else query_start.data_ptr(), op, wsp, floats, locksp, counters, *sizes,
            w4_hip.raw_stream(index)))
    return out
