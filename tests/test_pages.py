"""The bookkeeping of a paged cache on the GPU (tw4_plan_pages, tw4_release_pages behind kv_cache.py) against the same in Python
loops. Whole numbers: they have to be equal."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from tandem_amd import kv_cache
from tandem_amd.layers import w4_hip


def loops(context, new, table, free, taken, page, rows):
    """plan_pages in plain Python: (starts, lens, positions, slots, taken, counts, table)."""
    table = [list(r) for r in table]
    starts, lens, positions, slots, lacked, given = [0], [], [], [], 0, 0
    at = min(max(taken, 0), len(free))
    for i, (c, n) in enumerate(zip(context, new)):
        c, n = max(c, 0), max(n, 0)
        width = len(table[i])
        for p in range(min(-(-c // page), width), min(-(-(c + n) // page), width)):
            if at < len(free):
                table[i][p] = free[at]
                at, given = at + 1, given + 1
            else:
                table[i][p] = -1
                lacked += 1
        for j in range(c, c + n):
            positions.append(j)
            known = j // page < width and table[i][j // page] >= 0
            slots.append(table[i][j // page] * page + j % page if known else -1)
        starts.append(starts[-1] + n)
        lens.append(c + n)
    past = max(starts[-1] - rows, 0)
    positions = (positions + [0] * rows)[:rows]
    slots = (slots + [-1] * max(rows - starts[-1], 0))[:rows]
    return starts, lens, positions, slots, [at], [starts[-1], given, lacked, past], table


# ------------------------------------------------------------------------------------------- CPU
def test_argument_errors_return_before_launch():
    lib, p = w4_hip.library(), ctypes.c_void_p(4096)
    #       context fresh table stride width free n_free taken out size starts lens pos slots counts batch tokens
    good = [p, p, p, 10, 10, p, 5, p, p, 16, p, p, p, p, p, 4, 4]
    for at, value, needle in ((9, 12, "page_size"), (9, 512, "page_size"), (15, 0, "requests"), (15, 4097, "requests"), (16, -1, "tokens"),
                              (4, 11, "overlap"), (4, -1, "overlap"), (0, None, "null"), (2, None, "null"), (13, None, "null"),
                              (6, -1, "overlap")):
        args = list(good)
        args[at] = value
        assert lib.tw4_plan_pages(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good = [p, 2, p, 10, 10, p, 4, p, 5, p, 16]
    for at, value, needle in ((10, 17, "page_size"), (1, -1, "sizes"), (6, 0, "sizes"), (4, 12, "sizes"), (0, None, "null")):
        args = list(good)
        args[at] = value
        assert lib.tw4_release_pages(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode(), (at, value, lib.tw4_last_error())
    good[1] = 0
    assert lib.tw4_release_pages(*good, None) == w4_hip.TW4_OK


def test_refusals_on_the_cpu():
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kv_cache.plan_pages(z, z, torch.zeros(2, 3, dtype=torch.int32), z, z[:1], 16, 2)
    for bad in (dict(page_size=8), dict(head_dim=96), dict(dtype=torch.float32), dict(max_requests=0), dict(max_requests=5000),
                dict(num_pages=1 << 27), dict(layers=0)):
        args = dict(layers=1, kv_heads=1, head_dim=64, num_pages=4, max_requests=2, max_seq_len=32, device="cpu")
        with pytest.raises(ValueError):
            kv_cache.PagedKVCache(**{**args, **bad})


# ------------------------------------------------------------------------------------------- GPU
def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _case(rng, batch, page, longest, most, width=None, spare=8, idle=0.2):
    context = [rng.randint(0, longest) for _ in range(batch)]
    new = [0 if rng.random() < idle else rng.randint(1, most) for _ in range(batch)]
    width = width or -(-(longest + most) // page)
    held = [min(-(-c // page), width) for c in context]
    need = sum(min(-(-(c + n) // page), width) for c, n in zip(context, new)) - sum(held)
    pool = list(range(sum(held) + max(need + spare, 1)))
    rng.shuffle(pool)
    table, at = [], 0
    for h in held:
        table.append(pool[at:at + h] + [-1] * (width - h))
        at += h
    return context, new, table, pool[at:]


def _check(context, new, table, free, taken, page, rows, in_place=False):
    want = loops(context, new, table, free, taken, page, rows)
    t, c, k = _int(table), _int(context), _int([taken])
    if in_place:
        plan = kv_cache.plan_pages(c, _int(new), t, _int(free), k, page, rows, seq_lens_out=c, taken_out=k)
        assert plan.seq_lens is c and plan.taken is k
    else:
        plan = kv_cache.plan_pages(c, _int(new), t, _int(free), k, page, rows)
        assert c.tolist() == context and k.tolist() == [taken]
    for name, g, w in zip(("starts", "lens", "positions", "slots", "taken", "counts", "table"), (*plan, t), want):
        assert g.tolist() == w, name


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,longest,most,extra", [
    (1, 16, 0, 1, 0), (1, 16, 15, 1, 0), (1, 16, 16, 1, 3), (1, 64, 1000, 1, 0), (5, 16, 40, 7, 4), (64, 32, 500, 90, 0),
    (63, 256, 3000, 1, 1), (65, 16, 100, 1, 63), (257, 128, 4000, 1, 0), (4096, 16, 60, 3, 17), (1000, 16, 300, 40, 5),
    (3, 16, 9000, 9000, 100)])
def test_plan_equals_loops(batch, page, longest, most, extra, in_place):
    rng = random.Random(batch * 31 + most)
    context, new, table, free = _case(rng, batch, page, longest, most)
    _check(context, new, table, free, 0, page, sum(new) + extra, in_place)


@pytest.mark.gpu
def test_all_idle_no_rows_and_negative_lengths():
    _check([5, 0, 31], [0, 0, 0], [[3, -1], [-1, -1], [1, 2]], [7, 8], 1, 16, 4)
    _check([5, 0, 31], [0, 0, 0], [[3, -1], [-1, -1], [1, 2]], [7, 8], 1, 16, 0)
    _check([-3, 10, 4], [2, -5, 1], [[-1, -1], [4, -1], [5, -1]], [7, 8], 0, 16, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 128])
def test_shortage_and_narrow_table(page):
    """A list that runs out gives -1 entries and slots from there on; a request that outgrows its row keeps what fits."""
    rng = random.Random(page)
    context, new, table, free = _case(rng, 40, page, 6 * page, 3 * page)
    for short in (0, 1, len(free) // 2):
        _check(context, new, table, free[:short], 0, page, sum(new) + 2)
    _check(context, new, table, free, len(free), page, sum(new))       # all taken
    _check(context, new, table, free, len(free) + 50, page, sum(new))  # a count past the list is the list's end
    _check(context, new, table, free, -4, page, sum(new))
    context, new, table, free = _case(rng, 40, page, 6 * page, 3 * page, width=5)
    _check(context, new, table, free, 3, page, sum(new) + 1)
    _check(context, new, table, free, 0, page, max(sum(new) - 30, 0))  # more tokens than rows: counted


@pytest.mark.gpu
def test_strided_table_and_refusals():
    wide = torch.full((3, 12), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = _int([[4, -1, -1, -1], [5, 6, -1, -1], [-1, -1, -1, -1]])
    context, new = _int([16, 20, 0]), _int([1, 30, 5])
    plan = kv_cache.plan_pages(context, new, wide[:, 2:6], _int([9, 8, 7, 3]), _int([0]), 16, 36)
    assert wide[:, 2:6].tolist() == [[4, 9, -1, -1], [5, 6, 8, 7], [3, -1, -1, -1]]
    assert (wide[:, :2] == -7).all() and (wide[:, 6:] == -7).all() and plan.counts.tolist() == [36, 4, 0, 0]
    ok = dict(context_lens=context, query_lens=new, page_table=wide[:, 2:6], free_pages=_int([1]), taken=_int([0]), page_size=16,
              num_tokens=4)
    for key, value, needle in (("context_lens", context.long(), "context_lens"), ("query_lens", new[:2], "query_lens"),
                               ("page_table", wide[:1].expand(3, -1), "separate"), ("page_table", wide.t(), "separate"),
                               ("page_table", wide[:0], "requests"), ("free_pages", _int([1]).float(), "free_pages"),
                               ("taken", _int([0, 1]), "taken"), ("page_size", 20, "page size"), ("num_tokens", -1, "num_tokens"),
                               ("context_lens", context.cpu(), "context_lens")):
        with pytest.raises(RuntimeError, match=needle):
            kv_cache.plan_pages(**{**ok, key: value})


@pytest.mark.gpu
def test_release_gives_pages_back_in_order():
    table = _int([[3, 1, -1], [0, -1, -1], [5, 9, 7], [2, -1, -1]])
    lens, free, taken = _int([20, 16, 48, 3]), _int([3, 1, 0, 5, 9, 7, 2, 4, 6, 8]), _int([7])
    kv_cache.release_pages(_int([2, 9, 0, -1, 0]), lens, table, free, taken, 16)
    assert taken.tolist() == [2] and lens.tolist() == [0, 16, 0, 3]
    assert table.tolist() == [[-1, -1, -1], [0, -1, -1], [-1, -1, -1], [2, -1, -1]]
    assert free.tolist()[2:7] == [3, 1, 5, 9, 7] and free.tolist()[7:] == [4, 6, 8]
    # a request that was short of pages has entries that are none
    table, lens, free, taken = _int([[3, -1, 4]]), _int([40]), _int([3, 4, 6]), _int([2])
    kv_cache.release_pages(_int([0]), lens, table, free, taken, 16)
    assert taken.tolist() == [0] and free.tolist() == [3, 4, 6]


@pytest.mark.gpu
def test_cache_lives_through_many_steps():
    """Random steps, idle lanes and releases: no page is ever held twice, none is lost, and slots follow the table."""
    rng = random.Random(4)
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=64, max_requests=9, max_seq_len=200, page_size=16)
    lens = [0] * 9
    for step in range(60):
        b = rng.randint(1, 9)
        new = [rng.choice((0, 1, 1, rng.randint(1, 20))) for _ in range(b)]
        new = [n if lens[i] + n <= 100 else 0 for i, n in enumerate(new)]
        rows = sum(new) + rng.randint(0, 3)
        batch = cache.plan(_int(new), rows, max_query_len=max(new))
        lens[:b] = [x + n for x, n in zip(lens, new)]
        assert batch.seq_lens.tolist() == lens[:b] and batch.counts[2:].tolist() == [0, 0]
        slots = batch.slots.tolist()
        at = 0
        table = cache.page_table.tolist()
        for i, n in enumerate(new):
            for j in range(lens[i] - n, lens[i]):
                assert slots[at] == table[i][j // 16] * 16 + j % 16
                at += 1
        assert slots[at:] == [-1] * (rows - at)
        if rng.random() < 0.3:
            gone = rng.sample(range(9), rng.randint(1, 3))
            cache.release(gone)
            for i in gone:
                lens[i] = 0
        held = [p for i, r in enumerate(cache.page_table.tolist()) for p in r[:-(-lens[i] // 16)]]
        left = cache.free_pages.tolist()[int(cache.taken):]
        assert sorted(held + left) == list(range(64)), step


@pytest.mark.gpu
def test_a_batch_keeps_its_lengths_when_the_next_is_planned():
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=16, max_requests=3, max_seq_len=96)
    first = cache.plan(_int([3, 20, 0]), 23)
    second = cache.plan(_int([1, 30, 5]), 36)
    assert first.seq_lens.tolist() == [3, 20, 0] and second.seq_lens.tolist() == [4, 50, 5]
    assert cache.context_lens.tolist() == [4, 50, 5] and second.counts.tolist() == [36, 3, 0, 0]
    assert second.positions.tolist() == [3, *range(20, 50), *range(5)]


def test_step_refuses_bad_arguments():
    lib, p = w4_hip.library(), ctypes.c_void_p(4096)
    #       context fresh table stride width free n_free taken size starts lens pos slots counts batch tokens
    good = [p, p, p, 10, 10, p, 5, p, 16, p, ctypes.c_void_p(8192), p, p, p, 4, 4]
    for at, value, needle in ((8, 12, "page_size"), (14, 0, "requests"), (14, 4097, "requests"), (15, -1, "tokens"), (4, 11, "overlap"),
                              (0, None, "null"), (7, None, "null"), (13, None, "null"), (6, -1, "overlap"), (10, p, "two arrays")):
        args = list(good)
        args[at] = value
        assert lib.tw4_plan_step(*args, None) == w4_hip.TW4_EINVAL, (at, value)
        assert needle in lib.tw4_last_error().decode() and "plan_step" in lib.tw4_last_error().decode(), (at, value)


def _whole(cache, lanes, pages):
    """Every page is in the list or in one row of the table."""
    table = cache.page_table.tolist()
    left = cache.free_pages.tolist()[int(cache.taken):]
    assert sorted([p for r in table[:lanes] for p in r if p >= 0] + left) == list(range(pages))


@pytest.mark.gpu
def test_lengths_taken_back_keep_their_pages():
    """Drafted tokens that are not accepted: the lane's length is lowered, its pages stay with it, the next tokens take them, and release
    returns all."""
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=40, max_requests=3, max_seq_len=200)
    cache.plan(_int([15, 16, 3]), 34)
    rng = random.Random(6)
    lens = [15, 16, 3]
    for step in range(30):
        new = [rng.choice((0, 1, 5, 40)) for _ in range(3)]
        new = [n if lens[i] + n <= 190 else 0 for i, n in enumerate(new)]
        before = [r[:] for r in cache.page_table.tolist()]
        batch = cache.plan(_int(new), sum(new))
        table = cache.page_table.tolist()
        lacking = sum(1 for i in range(3) for p in range(-(-lens[i] // 16), -(-(lens[i] + new[i]) // 16)) if before[i][p] < 0)
        assert batch.counts.tolist() == [sum(new), lacking, 0, 0]
        assert all(b in (-1, a) for old, now in zip(before, table) for b, a in zip(old, now))
        lens = [x + n for x, n in zip(lens, new)]
        assert batch.slots.tolist() == [table[i][j // 16] * 16 + j % 16 for i in range(3) for j in range(lens[i] - new[i], lens[i])]
        _whole(cache, 3, 40)
        back = [rng.randint(0, n) for n in new]  # not accepted
        cache.context_lens -= _int(back)
        lens = [x - n for x, n in zip(lens, back)]
        if step % 7 == 6:
            cache.release([step % 3])
            lens[step % 3] = 0
            assert set(cache.page_table.tolist()[step % 3]) == {-1}
            _whole(cache, 3, 40)
    cache.release([0, 1, 2])
    assert int(cache.taken) == 0 and sorted(cache.free_pages.tolist()) == list(range(40))
    assert cache.context_lens.tolist() == [0, 0, 0]


@pytest.mark.gpu
def test_many_pages_kept_and_given_in_one_step():
    """More new places of the table than the workgroup has threads, kept and missing ones in turn."""
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=6000, max_requests=5, max_seq_len=16 * 900)
    for steps in ([100, 14000, 1, 0, 9000], [5000, 1, 14000, 14000, 0]):
        cache.plan(_int(steps), sum(steps))
        cache.context_lens.clamp_(max=1)
    batch = cache.plan(_int([14000] * 5), 70000)
    assert batch.counts.tolist() == [70000, 5 * 876 - (313 + 875 + 876 + 875 + 563), 0, 0]  # ceil(14001 / 16) = 876 a lane
    _whole(cache, 5, 6000)
    slots, table = batch.slots.tolist(), cache.page_table.tolist()
    assert slots == [table[i][j // 16] * 16 + j % 16 for i in range(5) for j in range(1, 14001)]
    cache.release([4, 2, 0, 1, 3])
    assert int(cache.taken) == 0 and sorted(cache.free_pages.tolist()) == list(range(6000))


@pytest.mark.gpu
def test_tokens_without_a_page_can_be_brought_again():
    """A step that the list had too few pages for: the lane's length is taken back to the last page there is, another lane is released, and
    the tokens come again."""
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=4, max_requests=2, max_seq_len=96)
    cache.plan(_int([40, 10]), 50)
    batch = cache.plan(_int([30, 0]), 30)
    assert batch.counts.tolist() == [30, 0, 2, 0] and cache.page_table.tolist()[0][:5] == [0, 1, 2, -1, -1]
    assert batch.slots.tolist() == [*range(40, 48)] + [-1] * 22
    cache.context_lens[0] = 48
    cache.release([1])
    batch = cache.plan(_int([16, 0]), 16)
    assert batch.counts.tolist() == [16, 1, 0, 0] and batch.slots.tolist() == [*range(48, 64)]
    cache.release([0])
    assert int(cache.taken) == 0 and sorted(cache.free_pages.tolist()) == list(range(4))


@pytest.mark.gpu
def test_a_step_with_too_few_rows_advances_by_those_it_has():
    """Tokens that no row is left for are counted, and come again in a later step: a lane's length has those only that were computed."""
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=16, max_requests=4, max_seq_len=96)
    batch = cache.plan(_int([5, 40, 7, 0]), 20)
    assert batch.counts.tolist() == [52, 5, 0, 32]
    assert batch.query_start.tolist() == [0, 5, 20, 20, 20] and batch.seq_lens.tolist() == [5, 15, 0, 0]
    assert cache.context_lens.tolist() == [5, 15, 0, 0] and batch.positions.tolist() == [*range(5), *range(15)]
    batch = cache.plan(_int([0, 25, 7, 0]), 33)
    assert batch.counts.tolist() == [32, 0, 0, 0] and batch.seq_lens.tolist() == [5, 40, 7, 0]
    table = cache.page_table.tolist()
    assert batch.slots.tolist() == [table[1][j // 16] * 16 + j % 16 for j in range(15, 40)] + [table[2][0] * 16 + j for j in range(7)] + [-1]
    batch = cache.plan(_int([3, 2, 1, 1]), 0)
    assert batch.counts.tolist() == [7, 1, 0, 7] and batch.query_start.tolist() == [0] * 5 and cache.context_lens.tolist() == [5, 40, 7, 0]
    _whole(cache, 4, 16)
    # more rows than one workgroup places
    cache = kv_cache.PagedKVCache(1, 1, 64, num_pages=2000, max_requests=3, max_seq_len=9000)
    cache.plan(_int([1, 2, 3]), 6)
    batch = cache.plan(_int([6000, 5000, 100]), 9001)
    assert batch.query_start.tolist() == [0, 6000, 9001, 9001] and batch.seq_lens.tolist() == [6001, 3003, 3]
    assert batch.positions.tolist() == [*range(1, 6001), *range(2, 3003)] and min(batch.slots.tolist()) >= 0


@pytest.mark.gpu
def test_release_without_table_columns():
    lens, taken = _int([5, 3]), _int([2])
    kv_cache.release_pages(_int([1, 7]), lens, torch.empty((2, 0), dtype=torch.int32, device="cuda"), _int([4, 5]), taken, 16)
    assert lens.tolist() == [5, 0] and taken.tolist() == [2]


@pytest.mark.gpu
def test_pages_past_all_slots_give_none():
    """A page number whose slots have no int32 gives no slot, not another page's."""
    for page, shift in ((16, 4), (256, 8)):
        table = _int([[-1], [-1], [-1]])
        free = _int([(1 << (32 - shift)) + 3, (1 << (31 - shift)) - 1, 1 << (31 - shift)])
        plan = kv_cache.plan_pages(_int([0, 0, 0]), _int([2, 2, 2]), table, free, _int([0]), page, 6)
        top = ((1 << (31 - shift)) - 1) * page
        assert plan.slots.tolist() == [-1, -1, top, top + 1, -1, -1] and table.flatten().tolist() == free.tolist()
