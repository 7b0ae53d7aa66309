"""Causal attention of new tokens over a paged KV cache (python/tandem/layers/flashinfer_attention.py,
python/tandem/layers/triton_decode_attn.py), on tw4_paged_attention: a decode step's single tokens, a few drafted ones,
chunks of prompts, and any mix of them in one call."""

from __future__ import annotations

import functools
import math

import torch

from tandem_amd.layers import w4_hip
from tandem_amd.layers.rotary import TYPES, check_cache, check_int32


@functools.lru_cache(maxsize=1 << 14)
def _plan(index: int, tokens: int, batch: int, heads: int, kv_heads: int, head_dim: int, max_query: int, max_keys: int,
          single: bool) -> tuple[int, int, int, int]:
    """(rows of a tile, splits, workspace floats, counters) of a call of these sizes on a GPU."""
    out = (w4_hip._I * 4)()
    cus = torch.cuda.get_device_properties(index).multi_processor_count
    w4_hip.check(w4_hip.library().tw4_paged_attention_plan(tokens, batch, heads, kv_heads, head_dim, max_query, max_keys,
                                                           int(single), cus, out))
    return tuple(out)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, query_start: torch.Tensor | None = None, *, max_query_len: int | None = None,
                    max_seq_len: int | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [T, heads, head_dim] (float16 or bfloat16, head_dim 64 or 128) over caches [pages, KV heads, page size,
    head_dim]. Request i of B has seq_lens[i] keys, the last of them its new tokens' own: key j lies in page
    page_table[i, j // page size]. Its new tokens are rows query_start[i] .. query_start[i + 1] - 1 of q, and the t-th of
    n sees the keys j <= seq_lens[i] - n + t. query_start None: one new token per request (T == B). Query head h reads KV head
    h // (heads / KV heads). scale: of the scores, head_dim^-0.5 by default.

    page_table int32 [B, pages per request] (any row stride), seq_lens int32 [B], query_start int32 [B + 1], ascending from 0.
    They are read on the GPU only, and nothing outside of the tensors is touched whatever they hold: keys of an entry that is no
    page, or behind the table's width, are left out, and a row that sees no key is zero. Infinities and NaN of keys and values
    reach the rows that see them and no others. Rows from query_start[B] on are left as they were in ``out``.

    max_query_len, max_seq_len: bounds the host knows; they only choose how the work is divided (T and the table's width
    otherwise). Results do not depend on the order in which workgroups run. Inference only."""
    who = "paged_attention"
    if not (q.is_cuda and q.dim() == 3 and q.dtype in TYPES and q.shape[2] in (64, 128) and q.stride(2) == 1):
        raise RuntimeError(f"{who}: q must be float16 or bfloat16 GPU rows [tokens, heads, 64 or 128] (got {tuple(q.shape)}, "
                           f"{q.dtype} on {q.device})")
    if not w4_hip.plain(q):
        raise RuntimeError(f"{who}: inference only, no gradient, transform or tracer can follow q")
    tokens, heads, d = q.shape
    if any(q.stride(i) % 8 for i in (0, 1) if q.shape[i] > 1) or q.data_ptr() % 16:
        raise RuntimeError(f"{who}: rows and heads of q must be 16-byte aligned (strides {q.stride()})")
    pages, kv_heads, size = check_cache(who, k_cache, v_cache, q, None, d)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise RuntimeError(f"{who}: heads must be a multiple of the cache's KV heads ({heads}, {kv_heads})")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != q.device or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise RuntimeError(f"{who}: page_table must be int32 [requests, pages per request] on {q.device}, rows contiguous "
                           f"(got {page_table.dtype} {tuple(page_table.shape)} on {page_table.device})")
    batch, width = page_table.shape
    check_int32(who, "seq_lens", seq_lens, (batch,), q)
    if query_start is not None:
        check_int32(who, "query_start", query_start, (batch + 1,), q)
    elif tokens != batch:
        raise RuntimeError(f"{who}: without query_start there is one token per request ({tokens} tokens, {batch} requests)")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise RuntimeError(f"{who}: a positive scale (got {scale})")
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() or out.data_ptr() % 16:
        raise RuntimeError(f"{who}: out must be a contiguous 16-byte aligned {q.dtype} tensor {list(q.shape)} on {q.device}")
    if tokens == 0 or batch == 0:
        return out
    index = q.get_device()
    single = query_start is None
    longest = width * size if max_seq_len is None else min(int(max_seq_len), width * size)
    most = 1 if single else tokens if max_query_len is None else min(int(max_query_len), tokens)
    # the longest context in steps: a decode loop asks for a few plans only
    rows, splits, floats, counters = _plan(index, tokens, batch, heads, kv_heads, d, most, (longest + 511) // 512 * 512, single)
    with w4_hip.on_device(index):
        ws, locks = w4_hip.stream_workspace(q.device) if splits > 1 else (None, None)
        w4_hip.check(w4_hip.library().tw4_paged_attention(
            q.data_ptr(), q.stride(0) if tokens > 1 else 0, q.stride(1) if heads > 1 else 0, k_cache.data_ptr(),
            v_cache.data_ptr(), *k_cache.stride()[:3], pages, size, page_table.data_ptr(),
            page_table.stride(0) if batch > 1 else 0, width, seq_lens.data_ptr(),
            None if single else query_start.data_ptr(), out.data_ptr(), None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel(), None if locks is None else locks.data_ptr(), 0 if locks is None else locks.numel(),
            tokens, batch, heads, kv_heads, d, scale, rows, splits, TYPES[q.dtype], w4_hip.raw_stream(index)))
    return out
