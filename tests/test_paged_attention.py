"""Attention over a paged cache (tw4_paged_attention behind layers/paged_attention.py) against softmax in 64 bits.

Tolerance, per output value, with u half a step of the type (fp16 2^-11, bf16 2^-8), w_j the weights, n the keys a row sees and
A = sum_j w_j |v_j|:
    u |o|                  the result's rounding
    u A                    each probability's rounding (the sum of probabilities is of the unrounded ones)
    2 d A                  the scores' error d, which the exponential makes relative: fp32 products of D terms, (D + 4) 2^-24 scale
                           sum_i |q_i k_i| (largest over the keys), once for the probability and once for their sum; the
                           exponential itself is good to 2^-22
    n 2^-23 A              the fp32 sums over the keys, numerator and denominator
    n 2^-31 max |v|        (fp16) probabilities are held times 2^6 at least, so below 2^-20 they are subnormal: half a step is 2^-31 of
                           the largest"""

from __future__ import annotations

import ctypes
import json
import os
import random

import pytest
import torch

from tandem_amd.layers import w4_hip
from tandem_amd.layers.paged_attention import paged_attention

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ------------------------------------------------------------------------------------------- CPU
def _good():
    p = ctypes.c_void_p(4096)
    #     q qt qh k v ps hs ts pages size table tstride width lens starts out ws wsn locks ln tokens batch heads kv dim scale rows splits bf16
    return [p, 4096, 128, p, p, 16384, 2048, 128, 50, 16, p, 10, 10, p, p, p, p, 1 << 23, p, 1 << 15, 7, 3, 32, 8, 128, 0.1, 16, 1, 0]


def test_argument_errors_return_before_launch():
    lib, odd = w4_hip.library(), ctypes.c_void_p(4104)
    for at, value, needle in ((0, None, "null"), (0, odd, "aligned"), (3, odd, "aligned"), (15, odd, "aligned"), (1, 4, "multiples"),
                              (7, 12, "multiples"), (8, 1 << 28, "2^31"), (12, 1 << 28, "2^31"), (8, 0, "without pages"),
                              (9, 48, "page_size"), (22, 30, "multiple"), (23, 0, "multiple"), (24, 96, "head_dim"), (25, 0.0, "scale"),
                              (25, float("nan"), "scale"), (25, -1.0, "scale"), (20, 1 << 28, "too many"), (14, None, "one token"),
                              (12, (1 << 26) + 1, "2^30"), (21, 1 << 22, "grid"), (27, 0, "splits"), (10, None, "null"), (13, None, "null")):
        args = _good()
        args[at] = value
        assert lib.tw4_paged_attention(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    args = _good()
    args[26] = 48
    assert lib.tw4_paged_attention(*args, None) == w4_hip.TW4_ECONFIG
    for at, value in ((16, None), (17, 100), (18, None), (19, 3)):
        args = _good()
        args[27], args[at] = 4, value
        assert lib.tw4_paged_attention(*args, None) == w4_hip.TW4_ESPACE and "splits" in lib.tw4_last_error().decode()
    for at in (20, 21):
        args = _good()
        args[at] = 0
        assert lib.tw4_paged_attention(*args, None) == w4_hip.TW4_OK


def _plan(*args, cus=256):
    out = (ctypes.c_int * 4)()
    w4_hip.check(w4_hip.library().tw4_paged_attention_plan(*args, cus, out))
    return tuple(out)


def test_plan_fits_the_workspace():
    """Over the range of sizes the plan never asks for more than the workspace has, and what it says is enough for the call."""
    rng = random.Random(0)
    for _ in range(3000):
        kv = rng.choice((1, 2, 8, 16))
        heads, dim = kv * rng.choice((1, 2, 4, 5, 7, 8, 12, 40)), rng.choice((64, 128))
        batch = round(2 ** rng.uniform(0, 12))
        single = rng.random() < 0.5
        tokens = batch if single else round(2 ** rng.uniform(0, 15))
        most = 1 if single else rng.randint(1, tokens)
        rows, splits, floats, counters = _plan(tokens, batch, heads, kv, dim, most, round(2 ** rng.uniform(0, 18)), int(single))
        assert splits >= 1 and floats <= w4_hip.WORKSPACE_FLOATS and counters <= w4_hip.WORKSPACE_LOCKS
        assert (splits == 1) == (floats == 0) == (counters == 0)
    assert _plan(1, 1, 32, 8, 128, 1, 100, 1)[1] == 1  # too few keys to split
    assert _plan(1, 1, 32, 8, 128, 1, 40000, 1)[1] > 8
    # a tile is no larger than a request's rows need
    for keys in (100, 2000, 40000):
        for batch in (1, 5, 60):
            assert _plan(batch * 3, batch, 32, 8, 128, 3, keys, 0)[0] == 16
            assert _plan(batch * 8, batch, 32, 8, 128, 8, keys, 0)[0] <= 32


def test_refusals_on_the_cpu():
    with pytest.raises(RuntimeError, match="GPU rows"):
        paged_attention(torch.zeros(1, 2, 64, dtype=torch.float16), *[torch.zeros(1, 1, 16, 64, dtype=torch.float16)] * 2,
                        torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


# ------------------------------------------------------------------------------------------- GPU
def build(context, new, heads, kv, d, dtype, page, seed=0, spread=1.0, spare=3):
    """(q, k_cache, v_cache, page_table, seq_lens, query_start) of requests with `context` old and `new` new tokens: pages in
    random order, what lies behind a request's last key NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [c + n for c, n in zip(context, new)]
    count = [-(-x // page) for x in lens]
    pool = torch.randperm(sum(count) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    caches = [torch.full((len(pool), kv, page, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    width = max(count + [1]) + 1
    table, at = [], 0
    for x, n in zip(lens, count):
        ids = pool[at:at + n]
        at += n
        for c, size in zip(caches, (1.0, 1.0)):
            rows = torch.randn((n * page, kv, d), generator=g, device="cuda") * size
            rows[x:] = float("nan")
            if n:
                c[ids] = rows.to(dtype).view(n, page, kv, d).transpose(1, 2)
        table.append(ids + [-1] * (width - n))
    q = (torch.randn((sum(new), heads, d), generator=g, device="cuda") * spread).to(dtype)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, *caches, as_int(table), as_int(lens), as_int(starts)


def exact(q, k_cache, v_cache, table, lens, starts, scale=None, absent=()):
    """(o, allowance) in 64 bits, request by request. absent: pages that count as not there."""
    t, heads, d = q.shape
    pages, kv, page, _ = k_cache.shape
    group = heads // kv
    scale = d ** -0.5 if scale is None else scale
    u, tiny = HALF_STEP[q.dtype], 2.0 ** -31 if q.dtype == torch.float16 else 0.0
    out = torch.zeros(t, heads, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for i, (n_keys, a, b) in enumerate(zip(lens.tolist(), starts.tolist(), starts.tolist()[1:])):
        n = b - a
        if n == 0 or n_keys <= 0:
            continue
        ids = table[i, :-(-n_keys // page)]
        there = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:n_keys]
        ids = ids.long().clamp(0, pages - 1)
        k, v = (c[ids].transpose(1, 2).reshape(-1, kv, d)[:n_keys].double() for c in (k_cache, v_cache))
        last = n_keys - n + torch.arange(n, device=q.device)
        seen = (torch.arange(n_keys, device=q.device) <= last[:, None]) & there
        for h in range(heads):
            kk, vv = k[:, h // group], v[:, h // group]
            qq = q[a:b, h].double()
            s = (qq @ kk.nan_to_num().t() * scale).masked_fill(~seen, -float("inf"))
            w = torch.softmax(s, dim=1).nan_to_num()
            vz = vv.masked_fill(~seen.any(0)[:, None], 0.0)  # NaN behind every row's keys
            out[a:b, h] = w @ vz
            size = w @ vz.abs()
            err = (d + 4) * 2.0 ** -24 * scale * (qq.abs() @ kk.nan_to_num().abs().t()).amax(1, keepdim=True) + 2.0 ** -22
            tol[a:b, h] = (u * out[a:b, h].abs() + (1.01 * u + 2 * err + n_keys * 2.0 ** -23) * size + n_keys * tiny * vz.abs().max()
                           + 1e-7)
    return out, tol


def check(args, scale=None, **kw):
    got = paged_attention(*args, scale=scale, **kw)
    want, tol = exact(*args, scale=scale)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), float((err / tol).max())
    return got


CASES = [
    # context, new, heads, kv, d, dtype, page
    ([0], [1], 4, 1, 128, torch.float16, 16),                       # one key
    ([16], [1], 8, 8, 64, torch.bfloat16, 16),
    ([31, 0, 127, 128, 700], [1] * 5, 32, 8, 128, torch.float16, 16),
    ([4000, 3, 33], [1] * 3, 40, 8, 128, torch.bfloat16, 64),
    ([9000], [1], 16, 8, 128, torch.float16, 256),                  # split
    ([5003, 17], [1, 1], 7, 1, 64, torch.float16, 32),
    ([100, 2000], [1, 1], 48, 2, 128, torch.bfloat16, 128),         # 24 rows: a tile and a half
    ([63, 500, 0], [5, 2, 7], 40, 8, 128, torch.float16, 16),       # drafted tokens
    ([0], [33], 4, 4, 64, torch.bfloat16, 16),
    ([0, 50, 1111], [129, 1, 64], 8, 2, 128, torch.float16, 32),    # chunks beside a decoding request
    ([0], [300], 16, 8, 128, torch.bfloat16, 16),
    ([777, 0, 5], [131, 257, 0], 12, 4, 64, torch.float16, 64),     # a request that sits out
    ([6000], [70], 8, 1, 128, torch.float16, 16),                   # a chunk behind a long context
    ([0, 1500], [515, 640], 32, 8, 128, torch.bfloat16, 128),
    ([3000], [16], 64, 8, 128, torch.bfloat16, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("context,new,heads,kv,d,dtype,page", CASES)
def test_against_64_bits(context, new, heads, kv, d, dtype, page):
    args = build(context, new, heads, kv, d, dtype, page, seed=len(new) + heads)
    got = check(args)
    bounds = dict(max_query_len=max(new), max_seq_len=max(c + n for c, n in zip(context, new)))
    check(args, **bounds)
    assert torch.equal(got, paged_attention(*args))  # the same bits again
    if all(n == 1 for n in new):
        check((*args[:5], args[5]))
        one = paged_attention(*args[:5], max_seq_len=bounds["max_seq_len"])
        want, tol = exact(*args)
        assert ((one.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("rows", [16, 32, 128])
def test_every_split_and_tile(splits, rows):
    """Every tile and any number of splits is right for any call."""
    args = build([1000, 40, 0, 129], [3, 1, 20, 1], 8, 2, 128, torch.float16, 16, seed=2)
    q, k, v, table, lens, starts = args
    out = torch.full_like(q, float("nan"))
    ws = torch.empty(1 << 25, device="cuda")
    locks = torch.zeros(1 << 12, dtype=torch.int32, device="cuda")
    for _ in range(2):
        w4_hip.check(w4_hip.library().tw4_paged_attention(
            q.data_ptr(), *q.stride()[:2], k.data_ptr(), v.data_ptr(), *k.stride()[:3], k.shape[0], k.shape[2], table.data_ptr(),
            table.stride(0), table.shape[1], lens.data_ptr(), starts.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
            locks.data_ptr(), locks.numel(), q.shape[0], 4, 8, 2, 128, 128 ** -0.5, rows, splits, 0,
            torch.cuda.current_stream().cuda_stream))
        want, tol = exact(*args)
        assert ((out.double() - want).abs() <= tol).all()
        assert not locks.any()


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", [16, 32, 128])
@pytest.mark.parametrize("heads,kv,d", [(40, 1, 128), (24, 2, 64), (8, 8, 128)])
def test_single_tokens_in_every_tile(heads, kv, d, rows, splits):
    args = build([1000, 40, 0, 300], [1] * 4, heads, kv, d, torch.float16, 16, seed=4)
    q, k, v, table, lens, starts = args
    out = torch.full_like(q, float("nan"))
    ws = torch.empty(1 << 23, device="cuda")
    locks = torch.zeros(1 << 12, dtype=torch.int32, device="cuda")
    w4_hip.check(w4_hip.library().tw4_paged_attention(
        q.data_ptr(), *q.stride()[:2], k.data_ptr(), v.data_ptr(), *k.stride()[:3], k.shape[0], k.shape[2], table.data_ptr(),
        table.stride(0), table.shape[1], lens.data_ptr(), None, out.data_ptr(), ws.data_ptr(), ws.numel(),
        locks.data_ptr(), locks.numel(), q.shape[0], 4, heads, kv, d, d ** -0.5, rows, splits, 0,
        torch.cuda.current_stream().cuda_stream))
    want, tol = exact(*args)
    assert ((out.double() - want).abs() <= tol).all() and not locks.any()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,most", [(65, 40), (300, 70), (4200, 3)])
def test_many_requests(batch, most):
    """More requests than a wavefront looks at in one step, or in two, of no token, one, and several tiles."""
    rng = random.Random(batch)
    new = [rng.choice((0, 1, 1, 2, rng.randint(0, most))) for _ in range(batch)]
    context = [rng.randint(0, 40) for _ in range(batch)]
    args = build(context, new, 2, 1, 64, torch.float16, 16, seed=12)
    check(args)
    check(args, max_query_len=most, max_seq_len=40 + most)


@pytest.mark.gpu
def test_bounds_and_starts_that_do_not_hold_and_rows_of_nan():
    """max_query_len and max_seq_len only divide the work; a query of NaN stays alone."""
    args = build([3000, 10, 100], [1, 150, 9], 8, 2, 128, torch.float16, 16, seed=14)
    for bounds in ((1, 1), (0, 0), (-3, -3), (10 ** 9, 10 ** 9), (2, 10 ** 5), (200, 16)):
        check(args, max_query_len=bounds[0], max_seq_len=bounds[1])
    # starts that are none: the rows are anything, and the calls after it right (no counter stays up)
    for wrong in ([5, 0, 900, -7], [0, 160, 3, 160], [160, 160, 0, 0], [-2 ** 31, 2 ** 31 - 1, 0, 70]):
        assert paged_attention(*args[:5], torch.tensor(wrong, dtype=torch.int32, device="cuda")).shape == args[0].shape
        check(args)
    want, tol = exact(*args)
    q = args[0].clone()
    q[77, 3], q[0, 0], q[155, 7] = float("nan"), float("inf"), float("nan")
    got = paged_attention(q, *args[1:])
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    hit[77, 3] = hit[0, 0] = hit[155, 7] = True
    assert ((got.double() - want).abs() <= tol)[~hit].all() and not torch.isfinite(got[hit]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_and_small_scores(dtype):
    """Scores far apart (one key takes all), all alike, and a scale of the caller's."""
    for spread, scale in ((40.0, None), (0.0, None), (1.0, 1.0), (1.0, 1e-3)):
        check(build([900, 20], [1, 40], 8, 2, 128, dtype, 16, seed=3, spread=spread), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 20, 129])
def test_many_small_probabilities(dtype, new):
    """30000 keys of 2^-25 of the largest each: less than fp16 has steps for, more than its rounding together."""
    q, k, v, table, lens, starts = build([30000], [new], 1, 1, 64, dtype, 16, seed=11)
    q.zero_()[..., 0] = 4.0
    first = table[0, 0]
    k.zero_()[first, 0, 0, 0] = 4.4
    v.fill_(1.0)[first, 0, 0] = 0.0
    got = check((q, k, v, table, lens, starts), scale=1.0)
    assert (got > 5e-4).all()
    if new == 1:
        assert (check((q, k, v, table, lens, starts), scale=1.0, max_seq_len=30001) > 5e-4).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 3, 200]])
def test_odd_values_reach_the_rows_that_see_them_only(new):
    """Infinities and NaN in keys and values of the chunk's later tokens leave its earlier ones as they are; behind the last key
    everything is NaN in every test here."""
    args = build([40, 200, 7], new, 8, 2, 128, torch.float16, 16, seed=5)
    q, k, v, table, lens, starts = args
    want, tol = exact(*args)
    for name, cache, value in (("v", v, float("inf")), ("v", v, float("nan")), ("k", k, float("nan"))):
        for i, n in enumerate(new):
            j = int(lens[i]) - 1 - n // 2  # seen by the request's tokens from n - 1 - n // 2 on
            old = cache[table[i, j // 16], 1, j % 16, 77].clone()
            cache[table[i, j // 16], 1, j % 16, 77] = value
            got = paged_attention(*args)
            cache[table[i, j // 16], 1, j % 16, 77] = old
            hit = torch.zeros(q.shape[0], 8, 128, dtype=torch.bool, device="cuda")
            rows = slice(int(starts[i]) + n - 1 - n // 2, int(starts[i + 1]))
            hit[rows, 4:, 77 if name == "v" else slice(None)] = True
            ok = (got.double() - want).abs() <= tol
            assert ok[~hit].all(), (name, value, i)
            assert not torch.isfinite(got[hit]).any(), (name, value, i)
            if value == float("inf"):
                assert (got[hit] == value).all()


@pytest.mark.gpu
def test_rows_without_a_key_and_rows_behind_the_last_request():
    """A row that sees nothing is zero (no keys, lengths below the new tokens' number, pages that are none); rows from
    query_start[B] on, and those of out there, stay as they are."""
    q, k, v, table, lens, starts = build([50, 10, 20], [2, 3, 4], 8, 2, 64, torch.float16, 16, seed=6)
    want, tol = exact(q, k, v, table, lens, starts)
    out = torch.full_like(q, 7.0)
    paged_attention(q, k, v, table, lens, starts, out=out)
    assert ((out.double() - want).abs() <= tol).all()
    wide = torch.cat([q, q])
    out = torch.full_like(wide, 7.0)
    got = paged_attention(wide, k, v, table, lens, starts, out=out)
    assert got is out and (out[9:] == 7).all() and ((out[:9].double() - want).abs() <= tol).all()
    lens2 = torch.tensor([0, 2, -5], dtype=torch.int32, device="cuda")  # second request: its first token sees nothing
    table2 = table.clone()
    got = paged_attention(q, k, v, table2, lens2, starts)
    assert (got[:3] == 0).all() and (got[5:] == 0).all() and not (got[3:5] == 0).all(-1).any()
    assert (paged_attention(q, k, v, table2, lens2 * 0 - 2 ** 31, starts) == 0).all()
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):  # entries that are no page
        table2 = table.clone()
        table2[0, 1], table2[1, 0], table2[2, 0] = bad, bad, bad
        got = paged_attention(q, k, v, table2, lens, starts)
        want2, tol2 = exact(q, k, v, table2, lens, starts)
        assert (got[2:5] == 0).all() and ((got.double() - want2).abs() <= tol2).all()
        one = torch.arange(4, dtype=torch.int32, device="cuda")
        got = paged_attention(q[:3], k, v, table2, lens, one)
        want2, tol2 = exact(q[:3], k, v, table2, lens, one)
        assert ((got.double() - want2).abs() <= tol2).all()
    # more keys than the table has room for: what is there counts
    got = paged_attention(q[:2], k, v, table[:1, :1], lens[:1] + 5000, starts[:2])
    short = torch.tensor([[int(table[0, 0]), -1]], dtype=torch.int32, device="cuda")
    want2, tol2 = exact(q[:2], k, v, short, torch.tensor([17]), starts[:2])
    assert ((got.double() - want2).abs() <= tol2).all()


@pytest.mark.gpu
def test_strides_layouts_and_refusals():
    args = build([333, 40], [3, 17], 8, 4, 128, torch.bfloat16, 32, seed=8)
    q, k, v, table, lens, starts = args
    want = paged_attention(*args)
    qkv = torch.randn(q.shape[0], 8 + 9, 128, device="cuda").bfloat16()
    qkv[:, 3:11] = q
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    both = torch.stack([k, v], dim=1)                                                  # pages hold keys and values
    by_token = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v)]         # [pages, page size, heads, D]
    big = torch.full((2, table.shape[1] + 5), 99, dtype=torch.int32, device="cuda")
    big[:, 2:2 + table.shape[1]] = table
    for other in ((qkv[:, 3:11], k, v, table), (heads_first, k, v, table), (q, both[:, 0], both[:, 1], table), (q, *by_token, table),
                  (q, k, v, big[:, 2:2 + table.shape[1]])):
        assert torch.equal(paged_attention(*other, lens, starts), want)
    ok = dict(q=q, k_cache=k, v_cache=v, page_table=table, seq_lens=lens, query_start=starts)
    for change, needle in ((dict(q=q.float()), "float16 or bfloat16"), (dict(q=q[..., :64]), "caches"), (dict(q=q[:, :6]), "multiple"),
                           (dict(q=q.clone().requires_grad_()), "inference"), (dict(v_cache=v.clone().requires_grad_()), "inference"), (dict(q=qkv.view(20, -1)[:, 4:1028].view(20, 8, 128)), "aligned"),
                           (dict(k_cache=k.half()), "caches of"), (dict(k_cache=k[:, :, :24], v_cache=v[:, :, :24]), "page size"),
                           (dict(v_cache=by_token[1]), "layout"), (dict(page_table=table.long()), "page_table"),
                           (dict(page_table=table.t()), "page_table"), (dict(seq_lens=lens[:1]), "seq_lens"),
                           (dict(query_start=starts[:2]), "query_start"), (dict(query_start=None), "one token"),
                           (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(out=torch.empty_like(q)[:1]), "out"),
                           (dict(out=torch.empty_like(q).half()), "out"), (dict(seq_lens=lens.cpu()), "seq_lens")):
        with pytest.raises(RuntimeError, match=needle):
            paged_attention(**{**ok, **change})
    assert paged_attention(q[:0], k, v, table, lens, starts * 0).shape == (0, 8, 128)
    assert paged_attention(q[:0], k, v, table[:0], lens[:0], starts[:1]).shape == (0, 8, 128)


@pytest.mark.gpu
def test_far_pages():
    """Pages whose offset in values passes 2^31 (a cache of 6 GB a side)."""
    pages, kv, page, d = 13000, 8, 256, 128
    k = torch.zeros(pages, kv, page, d, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    q, sk, sv, table, lens, starts = build([700, 300], [1, 6], 16, kv, d, torch.float16, page, seed=9)
    far = torch.arange(sk.shape[0], device="cuda") * 3 + pages - 3 * sk.shape[0]
    k[far], v[far] = sk, sv
    moved = torch.where(table >= 0, far[table.clamp(min=0).long()].int(), table)
    assert int(moved.max()) * k.stride(0) > 2 ** 31
    assert torch.equal(paged_attention(q, k, v, moved, lens, starts), paged_attention(q, sk, sv, table, lens, starts))
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_streams_and_graphs():
    """Calls on two streams at once, and captured graphs replayed with eager work between them, give what one eager call gives."""
    sets = [build([3000 + 500 * i, 10], [1, 1], 16, 8, 128, torch.float16, 16, seed=20 + i) for i in range(2)]
    want = [paged_attention(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(paged_attention(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(*s))
        graphs.append(graph)
    for rep in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), rep
        assert torch.equal(paged_attention(*sets[rep % 2]), want[rep % 2])
    # a graph whose lengths move between replays
    lens = sets[0][4]
    for cut in (1000, 17, 1):
        lens[0] = cut
        graphs[0].replay()
        assert torch.equal(outs[0], paged_attention(*sets[0])), cut
        w, tol = exact(*sets[0])
        assert ((outs[0].double() - w).abs() <= tol).all()


def _direct(args, rows, splits):
    """paged_attention with a tile and a number of splits of the caller's."""
    q, k, v, table, lens, starts = args
    out = torch.full_like(q, float("nan"))
    ws = torch.empty(1 << 25, device="cuda")
    locks = torch.zeros(1 << 12, dtype=torch.int32, device="cuda")
    w4_hip.check(w4_hip.library().tw4_paged_attention(
        q.data_ptr(), *q.stride()[:2], k.data_ptr(), v.data_ptr(), *k.stride()[:3], k.shape[0], k.shape[2], table.data_ptr(),
        table.stride(0), table.shape[1], lens.data_ptr(), starts.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
        locks.data_ptr(), locks.numel(), q.shape[0], lens.shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[2] ** -0.5, rows, splits,
        int(q.dtype == torch.bfloat16), torch.cuda.current_stream().cuda_stream))
    assert not locks.any()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", [16, 32, 128])
def test_rows_of_a_step_cut_short_see_no_later_key(rows, splits):
    """q has fewer rows than query_start says (plan_pages counts such tokens): those it has see what they see in the whole step."""
    q, k, v, table, lens, starts = args = build([40, 1000, 7], [5, 150, 9], 8, 2, 128, torch.float16, 16, seed=31)
    want, tol = exact(*args)
    for cut in (1, 3, 5, 6, 100, 154, 155, 160):
        got = _direct((q[:cut], k, v, table, lens, starts), rows, splits)
        assert ((got.double() - want[:cut]).abs() <= tol[:cut]).all(), cut
        got = paged_attention(q[:cut], k, v, table, lens, starts)
        assert ((got.double() - want[:cut]).abs() <= tol[:cut]).all(), cut


@pytest.mark.gpu
def test_caches_and_out_that_a_gradient_or_tangent_follows_are_refused():
    q, k, v, table, lens, starts = args = build([33], [2], 4, 2, 64, torch.float16, 16, seed=33)
    want = paged_attention(*args)
    with torch.autograd.forward_ad.dual_level():
        for name, x in (("q", q), ("k_cache", k), ("v_cache", v), ("out", torch.empty_like(q))):
            dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="inference only"):
                paged_attention(**{**dict(q=q, k_cache=k, v_cache=v, page_table=table, seq_lens=lens, query_start=starts), name: dual})
        assert torch.equal(paged_attention(*args), want)
    out = torch.empty_like(q).requires_grad_()
    with pytest.raises(RuntimeError, match="inference only"):
        paged_attention(*args, out=out)
    with torch.no_grad():
        assert torch.equal(paged_attention(q, k.requires_grad_(), v, table, lens, starts, out=out), want)
    k.requires_grad_(False)
    assert torch.equal(paged_attention(q, torch.nn.Parameter(k, requires_grad=False), v, table, lens, starts), want)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 3, 7])
@pytest.mark.parametrize("rows", [16, 32, 128])
@pytest.mark.parametrize("dtype,page,d", [(torch.float16, 16, 128), (torch.bfloat16, 64, 64), (torch.bfloat16, 16, 128), (torch.float16, 64, 64)])
def test_entries_that_are_no_page_in_every_tile_and_split(dtype, page, d, rows, splits):
    """Holes at the start, in the middle and at the end of long contexts, whole tiles of keys and parts of them; page 0, which is read in
    their place, is NaN."""
    q, k, v, table, lens, starts = build([1500, 700, 0, 900], [140, 3, 70, 1], 8, 2, d, dtype, page, seed=41)
    pages = k.shape[0]
    k, v = (torch.cat([torch.full_like(c[:1], float("nan")), c]) for c in (k, v))
    table = torch.where(table >= 0, table + 1, table)
    whole = (q, k, v, table, lens, starts)
    bad = (-1, pages + 1, 2 ** 31 - 1, -2 ** 31)
    last = [-(-int(x) // page) - 1 for x in lens]
    for holes in ([(0, 0)], [(0, last[0])], [(0, last[0] // 2), (0, last[0] // 2 + 1), (1, 2), (2, 0), (3, last[3])],
                  [(0, 3), (0, last[0] - 1), (1, last[1]), (1, 0), (3, 1), (3, 4)], [(1, i) for i in range(last[1] + 1)]):
        cut = table.clone()
        for n, (i, j) in enumerate(holes):
            cut[i, j] = bad[n % 4]
        args = (q, k, v, cut, lens, starts)
        want, tol = exact(*args)
        got = _direct(args, rows, splits)
        assert torch.isfinite(got).all() and ((got.double() - want).abs() <= tol).all(), holes
    want, tol = exact(*whole)
    assert ((_direct(whole, rows, splits).double() - want).abs() <= tol).all()


def test_plan_against_the_timed_choices():
    """The choice of tile and splits beside every one that was timed (profiles/paged_attention_rule_sweep.jsonl: us of a call in a graph for
    each "rows,splits", MI355X): the fitted calls and those left out of the fit."""
    with open(os.path.join(os.path.dirname(__file__), "..", "profiles", "paged_attention_rule_sweep.jsonl"), encoding="utf-8") as f:
        calls = [json.loads(line) for line in f]
    for fitted, least in ((True, 290), (False, 70)):
        ratios = []
        for c in calls:
            rows, splits, _, _ = _plan(c["tokens"], c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["max_query"],
                                       (c["max_keys"] + 127) // 128 * 128, int(c["single"]))
            chosen = c["us"].get(f"{rows},{splits}")  # a number of splits that fills the CUs exactly was not timed everywhere
            if c["fitted"] == fitted and chosen is not None:
                ratios.append(chosen / min(c["us"].values()))
        assert len(ratios) >= least and sum(ratios) / len(ratios) < 1.02 and max(ratios) < 1.25, (fitted, len(ratios))
