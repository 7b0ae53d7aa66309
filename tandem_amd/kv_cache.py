"""The paged KV cache of a decoder and its bookkeeping on the GPU (python/tandem/cache/): pages of a fixed number of tokens, a
list of the free ones, a table of each request's pages, and the positions and slots of a step's tokens from the requests' lengths
alone. Nothing is read back: a step, with its pages, can be captured in a HIP graph and replayed.

    plan_pages         pages, positions and slots of one step (tw4_plan_pages; a PagedKVCache's own, tw4_plan_step)
    release_pages      pages of ended requests back to the list (tw4_release_pages; a PagedKVCache's own, tw4_release_lanes)
    PagedKVCache       keys and values of every layer, the table and the lists
    PagedBatch         one step over a cache, as tandem_amd.model's attention takes it
"""

from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import TYPE_CHECKING, NamedTuple, Sequence

import torch

from tandem_amd.layers import rotary, w4_hip
from tandem_amd.layers.rotary import PAGE_SIZES, check_int32, layout

if TYPE_CHECKING:
    from tandem_amd.model import DecoderConfig

MAX_REQUESTS = 4096  # of one plan_pages call


class PagePlan(NamedTuple):
    """int32 tensors of plan_pages. counts: new tokens, pages given, pages the list did not have, tokens past num_tokens."""

    query_start: torch.Tensor  # [B + 1]
    seq_lens: torch.Tensor     # [B]
    positions: torch.Tensor    # [num_tokens]
    slots: torch.Tensor        # [num_tokens]
    taken: torch.Tensor        # [1]
    counts: torch.Tensor       # [4]


@functools.lru_cache(maxsize=1 << 12)
def _checked(who: str, table: tuple, free_pages: tuple, page_size: int, num_tokens: int,
             *vectors: tuple[str, tuple, int | None]) -> tuple:
    """(requests, pages per request, row stride, free pages, GPU); vectors: (name, layout, length, None for the number of requests).
    Once for each combination of layouts: an eager call is bound by the host."""
    shape, stride, dtype, index = table
    if not (index >= 0 and len(shape) == 2 and dtype == torch.int32) or (shape[1] > 1 and stride[1] != 1) or (
            shape[0] > 1 and stride[0] < shape[1]):
        raise RuntimeError(f"{who}: page_table must be an int32 GPU tensor [requests, pages per request] of separate contiguous rows "
                           f"(got {dtype} {tuple(shape)} on {index}, strides {stride})")
    batch, width = shape
    if page_size not in PAGE_SIZES:
        raise RuntimeError(f"{who}: a page size of {PAGE_SIZES} (got {page_size})")
    if not 1 <= batch <= MAX_REQUESTS:
        raise RuntimeError(f"{who}: 1 to {MAX_REQUESTS} requests (got {batch})")
    if not 0 <= num_tokens < 1 << 30:
        raise RuntimeError(f"{who}: 0 <= num_tokens < 2^30 (got {num_tokens})")
    if len(free_pages[0]) != 1:
        raise RuntimeError(f"{who}: free_pages must be one list (got {list(free_pages[0])})")
    check_int32(who, "free_pages", free_pages, tuple(free_pages[0]), index)
    for name, vector, length in vectors:
        check_int32(who, name, vector, (batch if length is None else length,), index)
    return batch, width, max(stride[0], width), free_pages[0][0], index


def plan_pages(context_lens: torch.Tensor, query_lens: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
               taken: torch.Tensor, page_size: int, num_tokens: int, *, seq_lens_out: torch.Tensor | None = None,
               taken_out: torch.Tensor | None = None) -> PagePlan:
    """Room in the cache for the new tokens of a step. Request i of B has context_lens[i] tokens in its pages page_table[i] and
    brings query_lens[i] more (0: it sits this step out); free_pages [F] lists free pages, of which the first taken[0] are
    in use. New pages are entered into page_table, in order of request; num_tokens rows get their positions and slots, those
    behind the last request's position 0 and slot -1. Where the list has no page left, or a request outgrows its row of the
    table, the entry and the slots there are -1.

    int32 GPU tensors; lengths below zero count as zero, and each new length and all new tokens together are below 2^31. seq_lens_out (context_lens
    itself, to advance it) and taken_out (taken itself) are written instead of new tensors. Nothing is read back; the caller that
    wants to know whether the pages sufficed reads counts[2]. Tokens past num_tokens (counts[3]) have pages, and count in seq_lens and
    query_start, but no position or slot."""
    outs = () if seq_lens_out is None else (("seq_lens_out", layout(seq_lens_out), None),)
    if taken_out is not None:
        outs += (("taken_out", layout(taken_out), 1),)
    batch, width, stride, n_free, index = _checked(
        "plan_pages", layout(page_table), layout(free_pages), page_size, num_tokens, ("context_lens", layout(context_lens), None),
        ("query_lens", layout(query_lens), None), ("taken", layout(taken), 1), *outs)
    # one allocation for what is new
    sizes = (batch + 1, num_tokens, num_tokens, 4, 1 if taken_out is None else 0, batch if seq_lens_out is None else 0)
    flat = page_table.new_empty(sum(sizes))
    query_start, positions, slots, counts, left, lens = flat.split_with_sizes(sizes)
    if seq_lens_out is not None:
        lens = seq_lens_out
    if taken_out is not None:
        left = taken_out
    base = flat.data_ptr()
    with w4_hip.on_device(index):
        w4_hip.check(w4_hip.library().tw4_plan_pages(
            context_lens.data_ptr(), query_lens.data_ptr(), page_table.data_ptr(), stride, width, free_pages.data_ptr(), n_free,
            taken.data_ptr(), left.data_ptr(), page_size, base, lens.data_ptr(), base + 4 * (batch + 1),
            base + 4 * (batch + 1 + num_tokens), base + 4 * (batch + 1 + 2 * num_tokens), batch, num_tokens, w4_hip.raw_stream(index)))
    return PagePlan(query_start, lens, positions, slots, left, counts)


def release_pages(ended: torch.Tensor, context_lens: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
                  taken: torch.Tensor, page_size: int) -> None:
    """The pages of the requests ``ended`` (int32 [n], indices into page_table's rows; others are passed over) go back to the
    list: taken[0] falls by their number and they are the next to be given. Their rows become -1 and their lengths 0, all in place. A
    request's pages are those of its length: entries behind it are not looked at."""
    _release("release_pages", w4_hip.library().tw4_release_pages, ended, context_lens, page_table, free_pages, taken, page_size)


def _release(who: str, entry, ended: torch.Tensor, context_lens: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
             taken: torch.Tensor, page_size: int) -> None:
    if ended.dim() != 1:
        raise RuntimeError(f"{who}: ended must be one list (got {list(ended.shape)})")
    batch, width, stride, n_free, index = _checked(
        who, layout(page_table), layout(free_pages), page_size, 0, ("ended", layout(ended), ended.shape[0]),
        ("context_lens", layout(context_lens), None), ("taken", layout(taken), 1))
    if ended.shape[0] == 0:
        return
    with w4_hip.on_device(index):
        w4_hip.check(entry(ended.data_ptr(), ended.shape[0], page_table.data_ptr(), stride, width, context_lens.data_ptr(), batch,
                           free_pages.data_ptr(), n_free, taken.data_ptr(), page_size, w4_hip.raw_stream(index)))


@dataclass(frozen=True)
class PagedBatch:
    """One step over a PagedKVCache: which tokens, where they go, and what they may see. Its tensors but page_table, the cache's, are its
    own, so the next steps may be planned before it has run. Its lanes are released after it has run: released pages go to others."""

    cache: "PagedKVCache"
    page_table: torch.Tensor
    seq_lens: torch.Tensor
    query_start: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    counts: torch.Tensor
    max_query_len: int
    max_seq_len: int


class PagedKVCache:
    """Keys and values [layers, pages, KV heads, page size, head_dim] for up to max_requests requests of up to max_seq_len tokens.
    A request has a lane (a row of the table) from its first token until release. Lanes 0 .. B - 1 take part in a step of B;
    those with no new token sit it out. One stream at a time works on a cache, as on any tensor it writes.

    context_lens [max_requests] may be lowered in place between steps (drafted tokens that were not accepted; tokens of a step that the list
    had too few pages for, down to the last whole page that is there): the lane keeps the pages behind its length for the
    tokens to come."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int, max_requests: int, max_seq_len: int,
                 page_size: int = 16, rope_theta: float = 1e6, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda") -> None:
        if page_size not in PAGE_SIZES or head_dim not in (64, 128) or dtype not in rotary.TYPES:
            raise ValueError(f"PagedKVCache: page size of {PAGE_SIZES}, head_dim 64 or 128, float16 or bfloat16 (got {page_size}, "
                             f"{head_dim}, {dtype})")
        if min(layers, kv_heads, num_pages, max_seq_len) < 1 or not 1 <= max_requests <= MAX_REQUESTS:
            raise ValueError(f"PagedKVCache: at least one layer, head, page and token, 1 to {MAX_REQUESTS} requests (got {layers}, "
                             f"{kv_heads}, {num_pages}, {max_seq_len}, {max_requests})")
        if num_pages * page_size >= 1 << 31:
            raise ValueError(f"PagedKVCache: fewer than 2^31 slots (got {num_pages} pages of {page_size})")
        self.page_size, self.max_seq_len, self.max_requests = page_size, max_seq_len, max_requests
        width = -(-max_seq_len // page_size)
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.keys, self.values = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        dev = self.keys.device
        self.page_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=dev)
        self.context_lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=dev)
        self.taken = torch.zeros(1, dtype=torch.int32, device=dev)
        self.rotary = rotary.rotary_table(width * page_size, head_dim, rope_theta, dev)

    @classmethod
    def for_model(cls, config: "DecoderConfig", num_pages: int, max_requests: int, max_seq_len: int, page_size: int = 16,
                  device: torch.device | str = "cuda") -> "PagedKVCache":
        """A cache of float16 for a DecoderModel of this configuration. NotImplementedError where it asks for attention that the model
        does not compute."""
        if config.rope_type != "default":
            raise NotImplementedError(f"rope_scaling of type {config.rope_type!r}: only plain rotary positions are supported")
        if config.sliding_window is not None and config.sliding_window < max_seq_len:
            raise NotImplementedError(f"sliding_window {config.sliding_window}: only attention over all keys is supported (a cache of no "
                                      f"more than that per request is; got max_seq_len {max_seq_len})")
        if config.other_attention:
            raise NotImplementedError(f"attention with {', '.join(config.other_attention)} is not supported")
        return cls(config.num_layers, config.num_kv_heads, config.head_dim, num_pages, max_requests, max_seq_len, page_size,
                   config.rope_theta, torch.float16, device)

    def plan(self, query_lens: torch.Tensor, num_tokens: int, max_query_len: int | None = None,
             max_seq_len: int | None = None) -> PagedBatch:
        """Takes pages for query_lens[i] new tokens of lane i (int32 [B], B <= max_requests) and advances the lanes' lengths; the
        step's tokens are num_tokens rows, lane by lane (rows behind the last are computed for nothing). Tokens that have no row, past
        num_tokens, are not in the step: query_start and the lengths stop at those that are, counts[3] says how many are left, and they
        are to come again. max_query_len,
        max_seq_len: bounds the host knows, for the division of the work."""
        if query_lens.dim() != 1 or not 1 <= query_lens.numel() <= self.max_requests:
            raise RuntimeError(f"PagedKVCache.plan: query_lens [1 .. {self.max_requests}] expected (got {tuple(query_lens.shape)})")
        b = query_lens.numel()
        table = self.page_table[:b]
        _, width, stride, n_free, index = _checked(
            "PagedKVCache.plan", layout(table), layout(self.free_pages), self.page_size, num_tokens,
            ("query_lens", layout(query_lens), None), ("context_lens", layout(self.context_lens), self.max_requests),
            ("taken", layout(self.taken), 1))
        sizes = (b + 1, num_tokens, num_tokens, 4, b)
        flat = self.page_table.new_empty(sum(sizes))
        query_start, positions, slots, counts, lens = flat.split_with_sizes(sizes)
        base = flat.data_ptr()
        with w4_hip.on_device(index):
            w4_hip.check(w4_hip.library().tw4_plan_step(
                self.context_lens.data_ptr(), query_lens.data_ptr(), table.data_ptr(), stride, width, self.free_pages.data_ptr(), n_free,
                self.taken.data_ptr(), self.page_size, base, lens.data_ptr(), base + 4 * (b + 1), base + 4 * (b + 1 + num_tokens),
                base + 4 * (b + 1 + 2 * num_tokens), b, num_tokens, w4_hip.raw_stream(index)))
        return PagedBatch(self, table, lens, query_start, positions, slots, counts,
                          num_tokens if max_query_len is None else max_query_len,
                          self.max_seq_len if max_seq_len is None else max_seq_len)

    def release(self, lanes: Sequence[int] | torch.Tensor) -> None:
        """The lanes' requests have ended: their pages are free again."""
        ended = torch.as_tensor(lanes, dtype=torch.int32).to(self.page_table.device)
        _release("PagedKVCache.release", w4_hip.library().tw4_release_lanes, ended, self.context_lens, self.page_table, self.free_pages,
                 self.taken, self.page_size)
