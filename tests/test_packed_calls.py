"""Calls over a cache in 4 bits that its other tests do not make: plans whose rows lie anywhere, calls without what they need, rows and heads of noughts, numbers
at both ends of their range, groups that are no numbers in portions, rows over chosen pages beside others, and the room that a portion takes."""
import math

import pytest
import torch

from test_packed import BF16, F32, GPU, chosen, make_pool, make_table, near, places, plain_attention, poison, tiles_bytes

from beglin_b200.csrc import ops


# ------------------------------------------------------------------------------------------------ plans
@pytest.mark.parametrize("lens,row_start", [([1, 1], [0, 100]), ([1, 1], [0, -1]), ([1, 1], [0, 0]), ([2, 2], [0, 1]), ([1, 1], [1, 2]), ([3], [1]), ([70, 1], [2, 0]),
                                            ([0, 1], [0, 1]), ([1] * 70, list(range(1, 71)))], ids=str)
def test_a_plan_refuses_rows_that_the_step_does_not_have(lens, row_start):
    """Every row of the step is one request's: none lies outside, none is in two requests."""
    with pytest.raises(ops.KernelError, match="first row"):
        ops.packed_plan(lens, 4, 2, 64, BF16, 64, device="cpu", row_start=row_start)


def test_a_plan_takes_rows_in_any_order():
    plan = ops.packed_plan([1, 0, 2, 1], 4, 2, 64, BF16, 64, device="cpu", row_start=[3, -7, 0, 2])
    assert plan.short.view(-1, 3).tolist() == [[0, 3, 1], [2, 0, 2], [3, 2, 1]]


# ------------------------------------------------------------------------------------------------ calls without what they need
def test_rows_need_their_requests(monkeypatch):
    """Only attention knows whose a row is without a list of requests."""
    monkeypatch.setattr(ops, "_here", lambda *a: None)                         # (nothing is launched)
    hd, page, T = 64, 16, 3
    pool, table, positions = make_pool(2, 1, hd, page, True), torch.zeros((T, 1), dtype=torch.int32), torch.zeros(T, dtype=torch.int32)
    src, q = torch.zeros((T, 3 * hd), dtype=BF16), torch.zeros((T, hd), dtype=BF16)
    for call in (lambda: ops.packed_append(src, q, 1, 1, hd, 0, False, None, positions, None, table, pool, page, None),
                 lambda: ops.packed_bounds(pool, positions, None, table, hd, page, None),
                 lambda: ops.packed_rows(pool, positions, None, table, hd, page, torch.empty((T, 2, 1, hd)), None)):
        with pytest.raises(ops.KernelError, match="a request for every row"):
            call()


# ------------------------------------------------------------------------------------------------ portions whose pages are written out
def portion(n, start, nh, nkv, hd, page, monkeypatch, change=None, scale=None, window=0, softcap=0.0, sink=False, dtype=BF16, many=0, most=None, given=True):
    """`n` rows of one request behind `start` positions: (results [n, nh, hd], what 64 bits say).  `change` takes the queries [n, nh, hd] and the pairs (step,
    lowest) of all pages [pages, kv heads, tiles, positions, keys and values, groups, 2]."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", many)
    table, pages = make_table([start + n], page)
    pool = make_pool(pages, nkv, hd, page, seed=3)
    poison(pool, table, [start + n], hd, page)
    q = torch.randn((n, nh, hd), generator=torch.Generator().manual_seed(2))
    if change:
        change(q, pool.unflatten(2, (page // 16, -1))[..., 16 * hd:].view(BF16).unflatten(3, (16, 2, hd // 64, 2)))
    q, scale = q.flatten(1).to(dtype), 1 / math.sqrt(hd) if scale is None else scale
    out, status = torch.full((n, nh * hd), 7.0, dtype=dtype, device="cuda"), ops.new_status("cuda")
    ops.packed_attention(q.cuda(), pool.cuda(), table.cuda(), torch.arange(start, start + n, dtype=torch.int32, device="cuda"), nh, nkv, hd, page,
                         most or start + n - 1, scale, out, status, window=window, softcap=softcap, sink=sink,
                         plan=ops.packed_plan([n], nh, nkv, hd, dtype, page, "cuda", starts=[start] if given else None))
    ops.raise_on_status(status)
    want = plain_attention(q.view(n, nh, hd), pool, table, hd, page, [(0, start + i) for i in range(n)], scale, window, softcap, torch.zeros(nh) if sink else None)
    return out.cpu().view(n, nh, hd), want


@GPU
@pytest.mark.parametrize("options", [dict(), dict(window=50), dict(softcap=9.0, sink=True)], ids=["plain", "window", "squashed"])
@pytest.mark.parametrize("what", ["queries", "a row", "keys", "both", "values too", "tiny"])
@pytest.mark.parametrize("nh,nkv,hd,page,n,start", [(4, 2, 128, 32, 100, 0), (6, 2, 64, 16, 70, 200)])
def test_rows_and_heads_of_noughts_in_a_portion(nh, nkv, hd, page, n, start, what, options, monkeypatch):
    """A row whose scores are all nought is the mean of the values that it sees: padded heads have such queries and keys."""
    def change(q, pairs):
        if what in ("queries", "both", "values too"):
            q[:, :nh // nkv + 1] = 0.0
        if what == "a row":
            q[n // 2] = 0.0
        if what in ("keys", "both", "values too"):
            pairs[:, 0, :, :, 0] = 0.0
        if what == "values too":
            pairs[:, 0, :, :, 1] = 0.0
        if what == "tiny":
            q *= 1e-22
            pairs[..., 0, :, :] *= 1e-22
    near(*portion(n, start, nh, nkv, hd, page, monkeypatch, change, **options), BF16)


@GPU
@pytest.mark.parametrize("key,value,query", [(1e-12, 1e-20, 1e9), (3e6, 1e7, 1e-6), (1e20, 1e30, 1e-20), (1.0, 1e-30, 1.0), (1e-15, 1.0, 1e-15), (1e15, 1.0, 1e15), (1e-30, 1.0, 1.0)])
@pytest.mark.parametrize("hd", [64, 128])
def test_queries_keys_and_values_of_any_scale_in_a_portion(key, value, query, hd, monkeypatch):
    """Queries, keys and values each of a scale of their own, the scores made ordinary by `scale` alone."""
    def change(q, pairs):
        q *= query
        pairs[..., 0, :, :] *= key
        pairs[..., 1, :, :] *= value
        pairs[:, 1] *= 0.01                                                    # the second kv head's scale is another
    got, want = portion(100, 0, 4, 2, hd, 32, monkeypatch, change, scale=1 / (key * query * math.sqrt(hd)))
    for heads, scale in ((slice(0, 2), value), (slice(2, 4), value * 0.01)):
        near(got[:, heads].double() / scale, want[:, heads] / scale, BF16)


@GPU
@pytest.mark.parametrize("key,value,query", [(1e36, 1e36, 1e-36), (1e-36, 1e-34, 1e36)])
def test_numbers_next_to_the_ends_of_their_range_in_a_portion(key, value, query, monkeypatch):
    def change(q, pairs):
        q *= query
        pairs[..., 0, :, :] *= key
        pairs[..., 1, :, :] *= value
    got, want = portion(100, 0, 4, 2, 128, 32, monkeypatch, change)
    near(got.double() / value, want / value, BF16)


@GPU
@pytest.mark.parametrize("options", [dict(), dict(window=40), dict(softcap=9.0, sink=True)], ids=["plain", "window", "squashed"])
@pytest.mark.parametrize("what,places_", [("value", [50]), ("value", [0, 95, 129]), ("key", [50]), ("both", [20, 64, 127])])
@pytest.mark.parametrize("nh,nkv,hd,page,n,start", [(4, 2, 128, 32, 130, 20), (6, 2, 64, 16, 150, 0)])
@pytest.mark.parametrize("many", [0, 1 << 30], ids=["written out", "packed"])
def test_a_group_that_is_no_number_in_a_portion(nh, nkv, hd, page, n, start, what, places_, options, many, monkeypatch):
    """It shows in the rows that see it, in its own features, and in no other: not in those in front of it, nor in those whose window is past it."""
    table, _ = make_table([start + n], page)
    def change(q, pairs):
        for i, pos in enumerate(places_):
            at = int(table[0, pos // page]), 1, pos % page // 16, pos % 16
            if what != "value":
                pairs[at + (0,)][-1] = math.nan
            if what != "key":
                pairs[at + (1,)][-1 if i % 2 else 0] = math.nan
    got, want = portion(n, start, nh, nkv, hd, page, monkeypatch, change, many=many, **options)
    near(got, want, BF16)
    assert bool(torch.isnan(got).any()) and (places_[0] <= start or not bool(torch.isnan(got[0]).any()))


# ------------------------------------------------------------------------------------------------ the room of pages written out
def test_every_portion_has_room_for_what_it_reads():
    starts, lens = [131072 - 300] + [0] * 7, [300] * 8
    plan = ops.packed_plan(lens, 32, 4, 128, BF16, 64, "cpu", starts=starts)
    assert plan.n_long == 8 and plan.rooms(131071)[0] == (2048,) + (5,) * 7 and plan.rooms(131071)[1] == 131072
    assert plan.rooms(131071, 1000)[0] == (22,) + (5,) * 7                     # 1,299 positions that begin anywhere in a page
    assert plan.rooms(131071, 1)[0] == (6,) + (5,) * 7 and plan.rooms(131071, 1 << 30)[0] == (2048,) + (5,) * 7
    assert plan.rooms(999)[0] == (16,) + (5,) * 7                              # (the call's bound holds too)
    unknown = ops.packed_plan(lens[:2], 32, 4, 128, BF16, 64, "cpu")
    assert unknown.rooms(8191)[0] == (128, 128) and unknown.rooms(8191, 100)[0] == (8, 8)
    for start in range(64):                                                    # as many as are touched at the worst
        assert (start + 299 + 1000 - 1) // 64 + 1 <= 22
    with pytest.raises(ops.KernelError, match="first position"):
        ops.packed_plan([300], 8, 4, 128, BF16, 64, "cpu", starts=[-1])


@GPU
@pytest.mark.parametrize("window", [0, 70])
def test_long_and_short_portions_lie_one_behind_the_other(window, monkeypatch):
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 0)
    nh, nkv, hd, page, lens, starts = 4, 2, 64, 16, [70, 90, 1, 3, 65], [5, 4000, 6, 0, 64]
    lengths = [n + s for n, s in zip(lens, starts)]
    table, pages = make_table(lengths, page)
    pool = make_pool(pages, nkv, hd, page, seed=8)
    poison(pool, table, lengths, hd, page)
    rows = [(i, p) for i, (n, s) in enumerate(zip(lens, starts)) for p in range(s, s + n)]
    q = torch.randn((len(rows), nh * hd), generator=torch.Generator().manual_seed(2)).to(BF16)
    want = plain_attention(q.view(-1, nh, hd), pool, table, hd, page, rows, 0.125, window)
    positions, dev = torch.tensor([p for _, p in rows], dtype=torch.int32).cuda(), (q.cuda(), pool.cuda(), table.cuda())
    out, status = torch.empty_like(dev[0]), ops.new_status("cuda")
    asked, rooms, empty = [0], [], torch.empty
    def counted(*a, **kw):
        t = empty(*a, **kw)
        asked[-1] += t.numel() * t.element_size()
        return t
    monkeypatch.setattr(torch, "empty", counted)
    for given in (starts, None):
        plan = ops.packed_plan(lens, nh, nkv, hd, BF16, page, "cuda", starts=given)
        rooms.append(sum(plan.rooms(max(lengths) - 1, window)[0]))
        out.fill_(7.0)
        asked.append(0)
        ops.packed_attention(*dev, positions, nh, nkv, hd, page, max(lengths) - 1, 0.125, out, status, plan=plan, window=window)
        ops.raise_on_status(status)
        near(out.view(-1, nh, hd), want, BF16)
    assert rooms == ([2 + 64 + 3, 3 * 64] if not window else [2 + 4 + 3, 3 * 4])          # (the requests of 70, 90 and 65 rows)
    each = 4 * 64 * nkv * hd + 8 * nkv                                         # bytes of a page: halves, and marks of values that are no numbers
    assert 0 <= (asked[2] - asked[1]) - (rooms[1] - rooms[0]) * each <= 3 * 4 * 64          # (and block tables of as many pages)


@GPU
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("starts,most", [([0, 0], 699), ([600, 0], 699), (None, 99), ([600, 600], 99)], ids=str)
def test_rows_beyond_their_bounds_are_recorded(starts, most, window, monkeypatch):
    """First positions or a bound below the rows' own: what has no room is not written, and the status says so."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 0)
    nh, nkv, hd, page = 4, 2, 64, 16
    table, pages = make_table([700, 700], page)
    q = torch.randn((200, nh * hd), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    positions = torch.arange(600, 700, dtype=torch.int32).repeat(2).cuda()
    status = ops.new_status("cuda")
    ops.packed_attention(q, make_pool(pages, nkv, hd, page).cuda(), table.cuda(), positions, nh, nkv, hd, page, most, 0.125, torch.empty_like(q), status, window=window,
                         plan=ops.packed_plan([100, 100], nh, nkv, hd, BF16, page, "cuda", starts=starts))
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.raise_on_status(status)


# ------------------------------------------------------------------------------------------------ rows over chosen pages beside others
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_plan_has_rows_over_chosen_pages(dtype):
    plan = ops.packed_plan([1, 70, 1, 3, 1], 12, 2, 128, dtype, 64, "cpu", chosen=[True, False, False, False, True])
    assert plan.n_chosen == 2 and plan.chosen.tolist() == [0, 0, 1, 4, 75, 1]
    assert plan.upto_chosen.tolist() == plan.short.tolist() + plan.chosen.tolist() and [2, 71, 1] in plan.short.view(-1, 3).tolist()
    assert sum(plan.short.view(-1, 3)[:, 2].tolist()) + 2 + sum(plan.blocks.view(-1, 3)[:, 2].tolist()) == 76
    for wrong in ([True], [False, True, False, False, False], [False] * 6):
        with pytest.raises(ops.KernelError, match="one row"):
            ops.packed_plan([1, 70, 1, 3, 1], 12, 2, 128, dtype, 64, "cpu", chosen=wrong)
    with pytest.raises(ops.KernelError, match="one row"):
        ops.packed_plan([0], 12, 2, 128, dtype, 64, "cpu", chosen=[True])


@GPU
@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(12, 2, 128, 64, BF16), (14, 2, 64, 16, BF16), (40, 2, 64, 16, BF16), (6, 2, 128, 32, F32)])
@pytest.mark.parametrize("many", [0, 1 << 30], ids=["written out", "packed"])
def test_chosen_pages_beside_portions(nh, nkv, hd, page, dtype, many, monkeypatch):
    """Single tokens over chosen pages, one over all of its pages, a long and a short portion, the requests' rows in another order than the requests."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", many)
    lens, row_start = [1, 70, 1, 3, 1, 1], [72, 0, 70, 73, 71, 76]
    lengths = [30 * page - 5, 200, 12 * page, 9, 50 * page + 1, page + 3]
    pick, top = [True, False, True, False, True, False], 7
    table, count = make_table(lengths, page)
    pool = make_pool(count, nkv, hd, page, bounds=True, seed=4)
    ends = torch.randn((count, nkv, 2, hd), generator=torch.Generator().manual_seed(3)).sort(2).values.to(BF16)
    pool[:, :, tiles_bytes(hd, page):] = ends.flatten(2).view(torch.uint8)
    poison(pool, table, lengths, hd, page)
    rows = [None] * 77
    for i, (n, r0, length) in enumerate(zip(lens, row_start, lengths)):
        rows[r0:r0 + n] = [(i, p) for p in range(length - n, length)]
    q = torch.randn((77, nh * hd), generator=torch.Generator().manual_seed(7)).to(dtype)
    positions, status = torch.tensor([p for _, p in rows], dtype=torch.int32).cuda(), ops.new_status("cuda")
    plan = ops.packed_plan(lens, nh, nkv, hd, dtype, page, "cuda", row_start=row_start, starts=[n - k for n, k in zip(lengths, lens)], chosen=pick)
    pages, out = torch.full((3, nkv, top), 99, dtype=torch.int32, device="cuda"), torch.empty((77, nh * hd), dtype=dtype, device="cuda")
    call = (q.cuda(), pool.cuda(), table.cuda(), positions, nh, nkv, hd, page, max(lengths) - 1)
    ops.packed_select(*call, pages, status, first=1, recent=2, plan=plan)
    mine = [i for i, p in enumerate(pick) if p]
    at = [row_start[i] for i in mine]
    assert torch.equal(pages.cpu(), chosen(q[at], pool, table[mine], [lengths[i] for i in mine], nh, nkv, hd, page, top, 1, 2))
    every = torch.arange(table.shape[1], dtype=torch.int32)[None, None].expand(77, nkv, -1)
    for given in (pages, None):
        which = every.clone()
        if given is not None:
            which[at] = -1
            which[at, :, :top] = pages.cpu()
        out.fill_(7.0)
        ops.packed_attention(*call, 0.1, out, status, plan=plan, pages=given)
        near(out.view(77, nh, hd), plain_attention(q.view(77, nh, hd), pool, table, hd, page, rows, 0.1, pages=which), dtype)
    ops.raise_on_status(status)
    for wrong in (dict(pages=pages[:2]), dict(pages=pages, window=9), dict(pages=pages, plan=ops.packed_plan([77], nh, nkv, hd, dtype, page, "cuda"))):
        with pytest.raises(ops.KernelError):
            ops.packed_attention(*call, 0.1, out, status, **{"plan": plan, **wrong})
    for wrong in (dict(plan=ops.packed_plan([77], nh, nkv, hd, dtype, page, "cuda")), dict(plan=ops.packed_plan([1] * 3, nh, nkv, hd, dtype, page, "cuda", chosen=[True] * 3))):
        with pytest.raises(ops.KernelError):
            ops.packed_select(*call, pages, status, first=1, recent=2, **wrong)


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("options", [dict(scale=math.inf), dict(scale=math.nan), dict(scale=0.0), dict(softcap=math.inf), dict(softcap=math.nan), dict(softcap=-1.0)], ids=str)
def test_scales_and_bounds_of_scores_are_finite(options, monkeypatch):
    monkeypatch.setattr(ops, "_here", lambda *a: None)                         # (nothing is launched)
    hd, page = 64, 16
    q, table, positions = torch.zeros((1, hd), dtype=BF16), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    options = dict(options)
    with pytest.raises(ops.KernelError, match="scale"):
        ops.packed_attention(q, make_pool(2, 1, hd, page), table, positions, 1, 1, hd, page, 0, options.pop("scale", 1.0), torch.zeros_like(q), None, **options)
