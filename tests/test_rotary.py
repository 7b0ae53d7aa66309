"""Head norms and rotary positions (tw4_norm_rope behind layers/rotary.py) against the formula in 64 bits.

Tolerance. With u half a step of the type (fp16 2^-11, bf16 2^-8): the result is rounded once, u |out|. Before that everything is
fp32, each operation off by 2^-24 of its result: the sum of up to 128 squares takes 8 additions in a lane and 4 over
lanes, halved by the root (6), the mean, eps and reciprocal root at most 4, two products 2, the table's rounding 1, two products
and a sum of the rotation 3: 16 of the rotated values' size, |y_i| + |y_partner|; twice that is allowed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tandem_amd.layers import rotary, w4_hip

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ------------------------------------------------------------------------------------------- CPU
def test_table():
    t = rotary.rotary_table(40, 64, 1e4)
    assert t.shape == (40, 64) and t.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (39, 31), (17, 5)):
        a = torch.tensor(p * 1e4 ** (-2 * i / 64), dtype=torch.float64)
        assert abs(float(t[p, i]) - float(a.cos())) <= 2.0 ** -24 and abs(float(t[p, 32 + i]) - float(a.sin())) <= 2.0 ** -24
    for bad in ((0, 64, 1e4), (4, 63, 1e4), (4, 64, 0.0)):
        with pytest.raises(ValueError):
            rotary.rotary_table(*bad)


def test_argument_errors_return_before_launch():
    lib, p, odd = w4_hip.library(), ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    #       qkv stride pos table rows qw kw eps q k v slots pages size ps hs ts tokens heads kv dim bf16
    good = [p, 6144, p, p, 100, p, p, 1e-6, p, p, p, p, 10, 16, 16384, 2048, 128, 3, 32, 8, 128, 0]
    for at, value, needle in ((0, None, "null"), (0, odd, "aligned"), (5, odd, "aligned"), (10, None, "null"), (4, 0, "table"),
                              (1, 6136, "rows of"), (1, 6148, "rows of"), (13, 24, "page_size"), (13, 8, "page_size"),
                              (12, 1 << 28, "2^31"), (14, 4, "multiples"), (19, 0, "kv_heads"), (20, 96, "head_dim"),
                              (17, -1, "tokens"), (17, 1 << 30, "too many")):
        args = list(good)
        args[at] = value
        assert lib.tw4_norm_rope(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good[17] = 0
    assert lib.tw4_norm_rope(*good, None) == w4_hip.TW4_OK


def test_refusals_on_the_cpu():
    table = rotary.rotary_table(8, 64, 1e4)
    with pytest.raises(RuntimeError, match="GPU rows"):
        rotary.norm_rope(torch.zeros(2, 6 * 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32), table, 4, 1)


# ------------------------------------------------------------------------------------------- GPU
def _exact(qkv, positions, table_positions, d, heads, kv, qw, kw, eps, theta):
    """(q, k, v, allowance of q, of k) in 64 bits on the CPU."""
    x = qkv.double().cpu().view(qkv.shape[0], heads + 2 * kv, d)
    i = torch.arange(d // 2, dtype=torch.float64)
    a = positions.cpu().double()[:, None, None] * theta ** (-2.0 * i / d)

    def turn(y, w):
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w.double().cpu()
        lo, hi = y[..., :d // 2], y[..., d // 2:]
        size = (lo.abs() + hi.abs()).repeat(1, 1, 2)
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], dim=-1), size

    (q, qs), (k, ks) = turn(x[:, :heads], qw), turn(x[:, heads:heads + kv], kw)
    u = HALF_STEP[qkv.dtype]
    return q, k, x[:, heads + kv:], u * q.abs() + 32 * 2.0 ** -24 * qs + 1e-7, u * k.abs() + 32 * 2.0 ** -24 * ks + 1e-7


def _inputs(tokens, heads, kv, d, dtype, norm, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, (heads + 2 * kv) * d, generator=g) * 3).to(dtype).cuda()
    positions = torch.randint(0, 5000, (tokens,), generator=g).int().cuda()
    w = [(0.5 + torch.rand(d, generator=g)).to(dtype).cuda() if norm else None for _ in range(2)]
    return qkv, positions, w


CASES = [(1, 32, 8, 128, torch.float16, True), (1, 1, 1, 64, torch.bfloat16, True), (3, 7, 1, 128, torch.bfloat16, False),
         (5, 5, 5, 64, torch.float16, False), (77, 40, 8, 128, torch.float16, True), (300, 24, 2, 64, torch.bfloat16, True),
         (2100, 16, 8, 128, torch.bfloat16, True), (6000, 32, 8, 128, torch.float16, True), (9001, 15, 7, 128, torch.bfloat16, False),
         (1031, 3, 3, 64, torch.float16, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,d,dtype,norm", CASES)
def test_dense(tokens, heads, kv, d, dtype, norm):
    qkv, positions, (qw, kw) = _inputs(tokens, heads, kv, d, dtype, norm, seed=tokens)
    table = rotary.rotary_table(5000, d, 1e6, "cuda")
    before = qkv.clone()
    q, k = rotary.norm_rope(qkv, positions, table, heads, kv, qw, kw, 1e-6)
    assert q.shape == (tokens, heads, d) and k.shape == (tokens, kv, d) and q.dtype == k.dtype == dtype
    eq, ek, _, tq, tk = _exact(qkv, positions, 5000, d, heads, kv, qw, kw, 1e-6, 1e6)
    assert ((q.double().cpu() - eq).abs() <= tq).all() and ((k.double().cpu() - ek).abs() <= tk).all()
    assert torch.equal(qkv, before)
    wide = torch.cat([qkv, qkv], dim=1)  # rows with something behind them
    q2, k2 = rotary.norm_rope(wide[:, :qkv.shape[1]], positions, table, heads, kv, qw, kw, 1e-6)
    assert torch.equal(q, q2) and torch.equal(k, k2)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,d,dtype,norm", CASES)
@pytest.mark.parametrize("page,tokens_first", [(16, False), (64, True)])
def test_cache(tokens, heads, kv, d, dtype, norm, page, tokens_first):
    """Keys and values land in their slots, and nothing else of the cache changes; tokens without a slot go nowhere.
    tokens_first: a cache laid out [pages, page size, KV heads, head_dim] seen through its transpose."""
    qkv, positions, (qw, kw) = _inputs(tokens, heads, kv, d, dtype, norm, seed=tokens + 1)
    table = rotary.rotary_table(5000, d, 1e4, "cuda")
    pages = (tokens + page - 1) // page + 2
    shape = (pages, page, kv, d) if tokens_first else (pages, kv, page, d)
    caches = [torch.randn(shape, device="cuda").to(dtype) for _ in range(2)]
    views = [c.transpose(1, 2) if tokens_first else c for c in caches]
    old = [v.clone() for v in views]
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=g)[:tokens].int().cuda()
    lost = torch.arange(tokens) % 5 == 4
    slots[lost.cuda()] = torch.tensor([-1, pages * page, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32).repeat(tokens)[:int(lost.sum())].cuda()
    q = rotary.norm_rope_cache(qkv, positions, table, heads, kv, *views, slots, qw, kw, 1e-6)
    eq, ek, ev, tq, tk = _exact(qkv, positions, 5000, d, heads, kv, qw, kw, 1e-6, 1e4)
    assert ((q.double().cpu() - eq).abs() <= tq).all()
    kept = (~lost).nonzero().flatten()
    at = slots.long().cpu()[kept]
    got_k, got_v = (v.transpose(1, 2).reshape(-1, kv, d).cpu() for v in views)
    assert ((got_k[at].double() - ek[kept]).abs() <= tk[kept]).all()
    assert torch.equal(got_v[at].double(), ev[kept])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[at] = False
    for got, o in ((got_k, old[0]), (got_v, old[1])):
        assert torch.equal(got[rest], o.transpose(1, 2).reshape(-1, kv, d).cpu()[rest])


@pytest.mark.gpu
def test_far_positions_nan_and_values_as_they_are():
    d, heads, kv = 128, 4, 2
    table = rotary.rotary_table(60000, d, 1e6, "cuda")
    qkv = torch.randn(6, (heads + 2 * kv) * d, device="cuda").half()
    qkv[:, -2] = torch.tensor([float("inf"), float("nan"), -0.0, 65504, 6e-8, -float("inf")]).half()
    positions = torch.tensor([0, 59999, 60000, -1, 2 ** 31 - 1, 40961], dtype=torch.int32, device="cuda")
    cache = [torch.zeros(1, kv, 16, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    q = rotary.norm_rope_cache(qkv, positions, table, heads, kv, *cache, torch.arange(6, dtype=torch.int32, device="cuda"))
    out_of_table = torch.tensor([False, False, True, True, True, False])
    assert torch.equal(q.isnan().all(-1).all(-1).cpu(), out_of_table) and torch.equal(q.isnan().any(-1).any(-1).cpu(), out_of_table)
    eq, _, _, tq, _ = _exact(qkv, positions, 60000, d, heads, kv, None, None, 1e-6, 1e6)
    assert ((q.double().cpu() - eq).abs() <= tq)[~out_of_table].all()
    values = qkv.view(6, -1, d)[:, heads + kv:]
    assert torch.equal(cache[1][0].transpose(0, 1)[:6].view(torch.int16), values.view(torch.int16))


@pytest.mark.gpu
def test_refusals():
    d, heads, kv = 64, 4, 2
    table = rotary.rotary_table(8, d, 1e4, "cuda")
    qkv = torch.zeros(2, 8 * d, dtype=torch.float16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = torch.zeros(2, kv, 16, d, dtype=torch.float16, device="cuda")
    ok = (qkv, pos, table, heads, kv)
    for args, needle in (((qkv.float(), *ok[1:]), "float16 or bfloat16"), ((qkv[0], *ok[1:]), "float16 or bfloat16"),
                         ((qkv, pos.long(), *ok[2:]), "positions"), ((qkv, pos[:1], *ok[2:]), "positions"),
                         ((qkv, pos, table.half(), heads, kv), "table"), ((qkv, pos, table[:, :32], heads, kv), "table"),
                         ((qkv, pos, table, 5, kv), "rows of"), ((qkv, pos, table, heads, 0), "rows of"),
                         ((qkv.clone().requires_grad_(), *ok[1:]), "inference"),
                         ((qkv.expand(2, -1)[:, 4:], *ok[1:]), "rows of")):
        with pytest.raises(RuntimeError, match=needle):
            rotary.norm_rope(*args)
    with pytest.raises(RuntimeError, match="q_weight"):
        rotary.norm_rope(*ok, q_weight=torch.ones(d, device="cuda"))
    slots = pos
    for k, v, s, needle in ((cache[..., :32], cache[..., :32], slots, "caches"), (cache.bfloat16(), cache.bfloat16(), slots, "float16"),
                            (cache[:, :1], cache[:, :1], slots, "caches"), (cache[:, :, :8], cache[:, :, :8], slots, "caches"),
                            (cache, cache[:1], slots, "caches"), (cache, cache, slots.long(), "slots"),
                            (cache, cache.transpose(0, 1).contiguous().transpose(0, 1), slots, "layout"),
                            (cache[:1].expand(2, -1, -1, -1), cache[1:].expand(2, -1, -1, -1), slots, "overlap"),
                            (cache.view(-1).as_strided(cache.shape, (2048, 1024, 56, 1)),) * 2 + (slots, "overlap"),
                            (cache, cache.clone().requires_grad_(), slots, "inference")):
        with pytest.raises(RuntimeError, match=needle):
            rotary.norm_rope_cache(*ok, k, v, s)
    # one row has no stride
    one = torch.zeros(3, 8 * d + 1, dtype=torch.float16, device="cuda")[:1, :8 * d]
    assert (rotary.norm_rope(one, pos[:1], table, heads, kv)[0] == 0).all()
    q, k = rotary.norm_rope(qkv[:0], pos[:0], table, heads, kv)
    assert q.shape == (0, heads, d) and k.shape == (0, kv, d)


@pytest.mark.gpu
def test_caches_that_a_tangent_follows_are_refused():
    d, heads, kv = 64, 4, 2
    table = rotary.rotary_table(8, d, 1e4, "cuda")
    qkv = torch.zeros(2, 8 * d, dtype=torch.float16, device="cuda")
    pos = torch.arange(2, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(2, kv, 16, d, dtype=torch.float16, device="cuda") for _ in range(2))
    with torch.autograd.forward_ad.dual_level():
        for at in range(2):
            caches = [k, v]
            caches[at] = torch.autograd.forward_ad.make_dual(caches[at], torch.ones_like(k))
            with pytest.raises(RuntimeError, match="inference only"):
                rotary.norm_rope_cache(qkv, pos, table, heads, kv, *caches, pos)
        rotary.norm_rope_cache(qkv, pos, table, heads, kv, k, v, pos)


@pytest.mark.gpu
def test_one_cache_for_keys_and_values_is_refused():
    d, heads, kv = 64, 4, 2
    table = rotary.rotary_table(8, d, 1e4, "cuda")
    qkv = torch.zeros(2, 8 * d, dtype=torch.float16, device="cuda")
    pos = torch.arange(2, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, kv, 16, d, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="memory of their own"):
        rotary.norm_rope_cache(qkv, pos, table, heads, kv, k, k, pos)
    both = torch.zeros(2, 2, kv, 16, d, dtype=torch.float16, device="cuda")  # keys and values in one tensor: two places each
    rotary.norm_rope_cache(qkv, pos, table, heads, kv, both[:, 0], both[:, 1], pos)


def test_all_plain_is_plain_of_each():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    from torch.func import vmap

    class Own(torch.Tensor):
        pass

    x, y, p, own = torch.zeros(3), torch.ones(3, requires_grad=True), torch.nn.Parameter(torch.zeros(3), requires_grad=False), Own([1.0])

    def agree(*extra):
        pool = [x, y, p, own, *extra]
        for a in pool:
            for b in pool:
                assert w4_hip.all_plain(x, a, b) == all(map(w4_hip.plain, (x, a, b)))
        assert w4_hip.all_plain(x, p) == (w4_hip.plain(x) and w4_hip.plain(p))

    agree()
    assert w4_hip.all_plain(x, p) and not w4_hip.all_plain(x, y) and not w4_hip.all_plain(own, x)
    for mode in (torch.no_grad(), torch.inference_mode(), FakeTensorMode()):
        with mode:
            agree()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(3), torch.ones(3))
        agree(dual)
        assert w4_hip.all_plain(x, p) and not w4_hip.all_plain(x, dual)

    def wrapped(t):
        agree(t)
        assert w4_hip.all_plain(x, p) and not w4_hip.all_plain(x, t)
        return t

    vmap(wrapped)(torch.zeros(2, 3))
