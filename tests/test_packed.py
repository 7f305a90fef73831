"""A cache in 4 bits: the append of rows with the rotation on the way, attention over it, the choice of pages by their bounds and attention over those alone,
each against a plain implementation in 64 bits that reads the bytes one by one."""
import math

import pytest
import torch

from beglin_b200.csrc import ops

GPU = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------------------------ the format, in 64 bits
def places(hd, page):
    """For every (position, feature) of a page: the byte and the shift of its key's code and of its value's, and the bytes of their pairs."""
    groups = hd // 64
    codes, tile = 8 * hd, 16 * hd + 128 * groups
    p, f = torch.arange(page)[:, None], torch.arange(hd)[None]
    base, s, group, r = p // 16 * tile, p % 16, f // 64, f % 64
    nib = r % 8 // 2 + 4 * (r % 2)
    key = base + s * (hd // 2) + (r // 16 * groups + group) * 8 + r % 16 // 8 * 4 + nib // 2
    lane = r // 8 * 4 + s % 8 // 2
    if groups == 2:
        value = base + codes + s // 8 * 512 + lane * 16 + s % 2 * 8 + group * 4 + r % 8 // 2
    else:
        value = base + codes + lane * 16 + (s // 8 * 2 + s % 2) * 4 + r % 8 // 2
    pair = base + 2 * codes + s * 8 * groups + group * 4
    return key, (4 * (nib % 2)).expand_as(key), value, (4 * (r % 2)).expand_as(key), pair, pair + groups * 4


def read(pool, hd, page):
    """Keys and values [pages, kv heads, page, hd] in 64 bits, and their codes and pairs (steps, lowest values)."""
    pool = pool.cpu()
    key, ks, value, vs, kp, vp = places(hd, page)
    out = []
    for at, shift, pair in ((key, ks, kp), (value, vs, vp)):
        u = (pool[:, :, at].int() >> shift & 15).double()
        b = pool[:, :, pair[..., None] + torch.arange(4)].contiguous().view(BF16).double()
        out.append((b[..., 1] + b[..., 0] * u, u, b[..., 0], b[..., 1]))
    return out


def tiles_bytes(hd, page):
    return page * (hd + hd // 64 * 8)


def make_pool(pages, nkv, hd, page, bounds=False, seed=0):
    """Pages of any codes with pairs as a cache has them.  (Bytes that nobody has written would do as well: pairs that are no numbers among them.)"""
    g = torch.Generator().manual_seed(seed)
    pool = torch.randint(0, 256, (pages, nkv, ops.packed_page_bytes(hd, page, bounds)), dtype=torch.uint8, generator=g)
    pairs = pool[:, :, :tiles_bytes(hd, page)].unflatten(2, (page // 16, -1))[..., 16 * hd:].view(BF16)
    step = torch.empty(pairs.shape[:-1] + (pairs.shape[-1] // 2,)).uniform_(0.1, 0.4, generator=g)
    pairs[..., 0::2] = step
    pairs[..., 1::2] = -7.5 * step + torch.empty(step.shape).uniform_(-0.5, 0.5, generator=g)
    return pool


def make_table(lengths, page, seed=0, spare=2):
    """A block table in a random order with unused entries behind, and the number of pages."""
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts) + spare, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    table, at = torch.full((len(lengths), max(counts + [1]) + 1), -1, dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, sum(counts) + spare


def poison(pool, table, lengths, hd, page):
    """Every place that no request has written holds what is no number."""
    _, _, _, _, kp, vp = places(hd, page)
    held = torch.zeros((pool.shape[0], page), dtype=torch.bool)
    for row, n in zip(table.tolist(), lengths):
        for i, p in enumerate(row):
            if p >= 0:
                held[p, :max(0, min(page, n - i * page))] = True
    for pages, slots in [torch.nonzero(~held, as_tuple=True)]:
        for at in (kp[slots], vp[slots]):
            spots = (at[..., None] + torch.arange(4)).flatten(1)
            pool[pages[:, None, None], torch.arange(pool.shape[1])[None, :, None], spots[:, None]] = 255


def rows_of(pool, table, hd, page, req, positions):
    """(keys, values) [kv heads, n, hd] in 64 bits at these positions of a request."""
    (k, *_), (v, *_) = read(pool, hd, page)
    at = table[req, positions // page].long()
    return k[at, :, positions % page].transpose(0, 1), v[at, :, positions % page].transpose(0, 1)


def attended(q, k, v, scale, cap=0.0, sink=None):
    """One row q [nh, hd] over [nkv, n, hd] in 64 bits."""
    nh, nkv = q.shape[0], k.shape[0]
    s = torch.einsum("hgd,hnd->hgn", q.double().view(nkv, nh // nkv, -1), k) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    s = s.reshape(nh, -1)
    extra = torch.zeros((nh, 0), dtype=torch.float64) if sink is None else sink.double()[:, None]
    w = torch.softmax(torch.cat([s, extra], dim=1), dim=1)[:, :k.shape[1]]
    return torch.einsum("hgn,hnd->hgd", w.view(nkv, nh // nkv, -1), v).reshape(nh, -1)


def plain_attention(q, pool, table, hd, page, rows, scale, window=0, cap=0.0, sink=None, pages=None):
    """rows: (request, position) of every row of q [T, nh, hd]."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    nkv = pool.shape[1]
    (k, *_), (v, *_) = read(pool, hd, page)
    for t, (req, pos) in enumerate(rows):
        at = torch.arange(max(0, pos - window + 1) if window else 0, pos + 1)
        for h in range(nkv):
            heads = slice(h * (q.shape[1] // nkv), (h + 1) * (q.shape[1] // nkv))
            mine = at if pages is None else torch.cat([at[(at // page) == p] for p in pages[t, h].tolist() if p >= 0] or [at[:0]])
            p = table[req, mine // page].long()
            if mine.numel():
                out[t, heads] = attended(q[t, heads], k[p, h, mine % page][None], v[p, h, mine % page][None], scale, cap, None if sink is None else sink[heads])
    return out


def near(got, want, dtype, steps=0.4):
    """Results against 64 bits.  bfloat16: the result's rounding (2^-8 of it at most half a step: 2^-9), that of the weights times a step (2^-9 of 15 steps) and the
    float sums of codes of up to 143 (a product's 16 positions at a time, 2^-23 each); float32: the sums alone."""
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs()
    off[torch.isnan(want)] = 0.0
    if dtype == BF16:
        bound = 2.0 ** -8 * want.abs() + 2.0 ** -9 * 15 * steps + 64 * 2.0 ** -23 * 143 * steps
    else:
        bound = 2.0 ** -20 * want.abs() + 64 * 2.0 ** -23 * 15 * steps
    assert bool((off[~torch.isnan(want)] <= bound[~torch.isnan(want)]).all()), float((off - bound).max())


# ------------------------------------------------------------------------------------------------ on the host
def test_the_size_of_a_page():
    assert ops.packed_page_bytes(128, 64) == 64 * 144 and ops.packed_page_bytes(64, 16) == 16 * 72
    assert ops.packed_page_bytes(128, 16, bounds=True) == 16 * 144 + 512
    for hd, page in ((80, 64), (256, 64), (0, 16)):
        with pytest.raises(ops.KernelError, match="64 or 128"):
            ops.packed_page_bytes(hd, page)
    for page in (0, -16, 8, 24, 65):
        with pytest.raises(ops.KernelError, match="multiple of 16"):
            ops.packed_page_bytes(128, page)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 16), (64, 48), (128, 64)])
def test_every_code_and_pair_of_a_page_has_a_place_of_its_own(hd, page):
    key, ks, value, vs, kp, vp = places(hd, page)
    spots = torch.cat([(key * 2 + ks // 4).flatten(), (value * 2 + vs // 4).flatten()])
    pairs = torch.cat([torch.unique(kp), torch.unique(vp)])
    every = torch.cat([spots, (pairs[:, None] * 2 + torch.arange(8)).flatten()])
    assert torch.equal(every.sort().values, torch.arange(2 * tiles_bytes(hd, page)))


@pytest.mark.parametrize("lens", [[1], [70, 1, 3, 64], [5] * 9, [0, 2, 0], [200, 64, 63]])
@pytest.mark.parametrize("nh,nkv,hd,dtype", [(12, 2, 128, BF16), (28, 4, 64, BF16), (12, 2, 128, F32), (5, 5, 64, BF16), (40, 1, 128, BF16)])
def test_a_plan_takes_every_row_once(lens, nh, nkv, hd, dtype):
    plan = ops.packed_plan(lens, nh, nkv, hd, dtype, page_size=16, device="cpu")
    taken = []
    for req, r0, n in plan.short.view(-1, 3).tolist():
        assert 1 <= n <= plan.most and plan.most * min(nh // nkv, 8 if dtype == F32 else 16) <= (8 if dtype == F32 else 16)
        taken += [(req, r) for r in range(r0, r0 + n)]
    longs = plan.longs.view(-1, 3).tolist()
    for i, r0, n in plan.blocks.view(-1, 3).tolist():
        assert 1 <= n <= plan.bq
        taken += [(longs[i][0], r) for r in range(r0, r0 + n)]
    assert sorted(taken, key=lambda x: x[1]) == [(i, sum(lens[:i]) + j) for i, n in enumerate(lens) for j in range(n)]
    streams = lambda n: -(-n // max(1, 16 // (nh // nkv))) * nkv * -(-nh // nkv // 16)
    assert [i for i, _, _ in longs] == [i for i, n in enumerate(lens) if dtype == BF16 and n > 1 and streams(n) > ops.PACKED_LONG_STREAMS]


def test_plans_refuse_what_does_not_fit():
    for args, what in ((([1], 5, 2, 128, BF16, 64), "kv heads"), (([-1], 4, 2, 128, BF16, 64), "rows"), (([1], 4, 2, 80, BF16, 64), "64 or 128"),
                       (([1], 4, 2, 64, torch.float16, 64), "float32 or bfloat16"), (([1], 4, 2, 64, BF16, 20), "multiple of 16")):
        with pytest.raises(ops.KernelError, match=what):
            ops.packed_plan(*args, device="cpu")
    with pytest.raises(ops.KernelError, match="first row"):
        ops.packed_plan([1, 2], 4, 2, 64, BF16, 64, device="cpu", row_start=[0])
    with pytest.raises(ops.KernelError, match="first position"):
        ops.packed_plan([1, 2], 4, 2, 64, BF16, 64, device="cpu", starts=[0])


@pytest.mark.parametrize("streams,positions,at_once", [(1, 1, 296), (2, 4096, 296), (128, 8192, 296), (16, 131072, 148), (900, 100, 296), (149, 100000, 296), (5000, 9999, 296)])
def test_ctas_that_share_streams_have_work(streams, positions, at_once):
    n, cluster = ops.packed_ctas(streams, min(streams, 64), positions, at_once)
    units = -(-positions // 256)
    assert n <= at_once and n <= streams * units and cluster in (1, 2, 4, 8) and cluster < 2 * units and (cluster == 1 or cluster * streams <= at_once)
    assert not n or (cluster == 1 and units > 3)
    assert ops.packed_ctas(2, 1025, 100000, 296) == (0, 8)


# ------------------------------------------------------------------------------------------------ append
def quantised(x):
    """(codes, steps, lowest values) of [..., hd] in 64 bits, by groups of 64."""
    g = x.unflatten(-1, (-1, 64))
    lowest = g.amin(-1, keepdim=True).float().to(BF16).double()
    step = ((g.amax(-1, keepdim=True) - lowest) / 15).float().to(BF16).double()
    u = ((g - lowest) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
    return u.flatten(-2), step.expand_as(g).flatten(-2), lowest.expand_as(g).flatten(-2)


def rotated(x, cos_sin, rot, interleaved):
    x, half = x.double().clone(), rot // 2
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos_sin.double()[:, None, :, 0], cos_sin.double()[:, None, :, 1]
    a, b = x[..., one], x[..., two]
    x[..., one], x[..., two] = a * c - b * s, a * s + b * c
    return x


def angles(positions, rot):
    a = positions.double()[:, None] * 1e4 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))
    return torch.stack([a.cos(), a.sin()], dim=2).float()


def appended(src, lens, starts, nh, nkv, hd, rot, interleaved, page, bounds=False, seed=0, dtype=None):
    """Append `src` to a pool of old bytes: (q, pool before, pool after, table, positions, requests)."""
    lengths = [s + n for s, n in zip(starts, lens)]
    table, pages = make_table(lengths, page, seed)
    before = make_pool(pages, nkv, hd, page, bounds, seed)
    positions = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).int()
    req = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).int()
    pool, q = before.cuda(), torch.empty((sum(lens), nh * hd), dtype=dtype or src.dtype, device="cuda")
    status = ops.new_status("cuda")
    ops.packed_append(src.cuda(), q, nh, nkv, hd, rot, interleaved, angles(positions, rot).cuda() if rot else None, positions.cuda(), req.cuda(),
                      table.cuda(), pool, page, status)
    ops.raise_on_status(status)
    return q.cpu(), before, pool, table, positions, req


@GPU
@pytest.mark.parametrize("lens,starts", [([1], [0]), ([1, 1, 1], [63, 64, 5]), ([130, 1, 17], [9, 200, 0])], ids=["one", "singles", "portions"])
@pytest.mark.parametrize("nh,nkv,hd,rot,interleaved,page,dtype", [
    (12, 2, 128, 128, False, 64, BF16), (3, 1, 64, 64, False, 16, F32), (8, 8, 128, 64, True, 32, F32), (5, 1, 64, 12, False, 48, BF16), (4, 2, 128, 0, False, 16, BF16),
    (14, 2, 64, 6, True, 16, BF16), (2, 1, 128, 128, True, 64, F32)])
def test_append_holds_what_64_bits_say(lens, starts, nh, nkv, hd, rot, interleaved, page, dtype):
    T = sum(lens)
    g = torch.Generator().manual_seed(T + hd)
    src = torch.randn((T, (nh + 2 * nkv) * hd), generator=g)
    src[:, 3::29] *= 9.0
    src = src.to(dtype)
    q, before, pool, table, positions, req = appended(src, lens, starts, nh, nkv, hd, rot, interleaved, page)
    x = src.view(T, nh + 2 * nkv, hd)
    turned = rotated(x[:, :nh + nkv], angles(positions, rot), rot, interleaved)
    off = (q.double() - turned[:, :nh].reshape(T, -1)).abs()
    # half a step of the result's type, and float's rounding of two products and their sum
    assert bool((off <= torch.finfo(dtype).eps / 2 * turned[:, :nh].reshape(T, -1).abs() * 1.001 + 2.0 ** -22 * x.double().abs().max()).all())
    after = read(pool, hd, page)
    at = table[req.long(), positions.long() // page].long()
    for (_, u, step, lowest), rows in zip(after, (turned[:, nh:], x[:, nh + nkv:].double())):
        for got, want in zip((u, step, lowest), quantised(rows)):
            assert torch.equal(got[at, :, positions.long() % page], want)
    # what is not the rows' is as it was
    key, _, value, _, kp, vp = places(hd, page)
    kept = torch.ones((pool.shape[0], pool.shape[2]), dtype=torch.bool)
    for p, s in zip(at.tolist(), (positions % page).tolist()):
        for spots in (key[s], value[s], (kp[s][:, None] + torch.arange(4)).flatten(), (vp[s][:, None] + torch.arange(4)).flatten()):
            kept[p, spots] = False
    assert torch.equal(pool.cpu().transpose(1, 2)[kept], before.transpose(1, 2)[kept])


@GPU
def test_append_of_many_rows_is_that_of_64_bits_at_every_border():
    """A hundred thousand groups: some of their values lie so near the border of two codes that float alone would take the other."""
    nh, nkv, hd, page, T = 1, 8, 128, 64, 3000
    src = torch.randn((T, (nh + 2 * nkv) * hd), generator=torch.Generator().manual_seed(4))
    _, _, pool, table, positions, req = appended(src, [T], [11], nh, nkv, hd, hd, False, page)
    at = table[0, positions.long() // page].long()
    turned = rotated(src.view(T, -1, hd)[:, :nh + nkv], angles(positions, hd), hd, False)
    for (_, u, step, lowest), rows in zip(read(pool, hd, page), (turned[:, nh:], src.view(T, -1, hd)[:, nh + nkv:].double())):
        for got, want in zip((u, step, lowest), quantised(rows)):
            assert torch.equal(got[at, :, positions.long() % page], want)


@GPU
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_partial_sums_and_of_rows_apart(hd):
    nh, nkv, T = 3, 1, 9
    g = torch.Generator().manual_seed(2)
    parts = torch.randn((3, T, (nh + 2 * nkv) * hd + 8), generator=g)[:, :, :(nh + 2 * nkv) * hd]
    whole = (parts[0] + parts[1]) + parts[2]
    one = appended(parts, [T], [3], nh, nkv, hd, hd, False, 16, dtype=BF16)
    two = appended(whole.contiguous(), [T], [3], nh, nkv, hd, hd, False, 16, dtype=BF16)
    assert torch.equal(one[0], two[0]) and torch.equal(one[2], two[2])


@GPU
def test_append_of_what_is_not_finite_and_of_groups_of_one_value():
    nh, nkv, hd, page = 1, 1, 128, 16
    src = torch.zeros((6, 3 * hd))
    src[0, hd + 3], src[1, hd + 70], src[2, 2 * hd + 1] = math.inf, math.nan, -math.inf
    src[3, hd:2 * hd] = 1.7                                                  # one value: held as its rounding
    src[4, 2 * hd:2 * hd + 64] = torch.linspace(-3e38, 3e38, 64)             # a range that float does not hold
    src[5, hd:] = torch.linspace(-1e-30, 1e-30, 256)
    _, _, pool, table, positions, _ = appended(src, [6], [0], nh, nkv, hd, 0, False, page)
    (k, *_), (v, *_) = (tuple(t[table[0, 0].long(), 0] for t in kind) for kind in read(pool, hd, page))
    bad_k, bad_v = torch.zeros((6, hd), dtype=torch.bool), torch.zeros((6, hd), dtype=torch.bool)
    bad_k[0, :64] = bad_k[1, 64:] = bad_v[2, :64] = bad_v[4, :64] = True
    assert torch.equal(torch.isnan(k[:6]), bad_k) and torch.equal(torch.isnan(v[:6]), bad_v)
    assert bool((k[3] == float(torch.tensor(1.7).to(BF16))).all()) and bool((v[3] == 0).all())
    assert float((k[5] - src[5, hd:2 * hd].double()).abs().max()) <= 1e-30 / 7


@GPU
@pytest.mark.parametrize("hd,page,dtype", [(128, 64, F32), (64, 16, BF16), (128, 48, BF16)])
def test_rows_are_read_back(hd, page, dtype):
    nkv, lens = 3, [1, 40, 3]
    lengths = [70, 40, 131]
    table, pages = make_table(lengths, page)
    pool = make_pool(pages, nkv, hd, page, seed=5)
    req = torch.tensor([0] + [1] * 40 + [2] * 3, dtype=torch.int32)
    positions = torch.tensor([69] + list(range(40)) + [130, 0, 64], dtype=torch.int32)
    out, status = torch.empty((44, 2, nkv, hd), dtype=dtype, device="cuda"), ops.new_status("cuda")
    ops.packed_rows(pool.cuda(), positions.cuda(), req.cuda(), table.cuda(), hd, page, out, status)
    ops.raise_on_status(status)
    at = table[req.long(), positions.long() // page].long()
    (k, *_), (v, *_) = read(pool, hd, page)
    want = torch.stack([k[at, :, positions.long() % page], v[at, :, positions.long() % page]], dim=1)
    assert torch.equal(out.cpu(), want.float().to(dtype))


@GPU
@pytest.mark.parametrize("hd,page", [(128, 64), (64, 16), (128, 48)])
def test_pages_that_are_filled_get_their_bounds(hd, page):
    nkv = 2
    lengths = [page, 2 * page - 1, 3 * page, 5]
    table, pages = make_table(lengths, page)
    before = make_pool(pages, nkv, hd, page, bounds=True, seed=6)
    before[table[2, 1].long(), 1, 16 * hd:16 * hd + 2] = 255                  # a step that is no number
    positions = torch.tensor([page - 1, 2 * page - 2] + list(range(2 * page - 3, 3 * page)) + [4], dtype=torch.int32)
    req = torch.tensor([0, 1] + [2] * (page + 3) + [3], dtype=torch.int32)
    pool, status = before.cuda(), ops.new_status("cuda")
    ops.packed_bounds(pool, positions.cuda(), req.cuda(), table.cuda(), hd, page, status)
    ops.raise_on_status(status)
    n = tiles_bytes(hd, page)
    assert torch.equal(pool.cpu()[:, :, :n], before[:, :, :n])
    (k, *_), _ = read(before, hd, page)
    got = pool.cpu()[:, :, n:].contiguous().view(BF16).unflatten(2, (2, hd))
    filled = {int(table[0, 0]), int(table[2, 1]), int(table[2, 2])}
    for p in range(pages):
        if p in filled:
            want = torch.stack([k[p].amin(1), k[p].amax(1)], dim=1).float().to(BF16)
            assert torch.equal(torch.isnan(got[p]), torch.isnan(want)) and torch.equal(got[p].nan_to_num(7.0), want.nan_to_num(7.0))
        else:
            assert torch.equal(pool.cpu()[p], before[p])
    assert bool(torch.isnan(got[int(table[2, 1]), 1, :, :64]).all()) and not bool(torch.isnan(got[int(table[2, 1]), 0]).any())


# ------------------------------------------------------------------------------------------------ attention
def single(lengths, nh, nkv, hd, page, dtype, seed=0, most=None, poisoned=True, q=None, **options):
    """Rows of single tokens: (results, what 64 bits say)."""
    table, pages = make_table(lengths, page, seed)
    pool = make_pool(pages, nkv, hd, page, seed=seed)
    if poisoned:
        poison(pool, table, lengths, hd, page)
    T = len(lengths)
    if q is None:
        q = torch.randn((T, nh * hd), generator=torch.Generator().manual_seed(seed + 9)) * 1.3
    q = q.to(dtype)
    out, status = torch.full((T, nh * hd), 7.0, dtype=dtype, device="cuda"), ops.new_status("cuda")
    sink = options.pop("sink_weight", None)
    ops.packed_attention(q.cuda(), pool.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda() - 1, nh, nkv, hd, page,
                         most if most is not None else max(lengths) - 1, 1 / math.sqrt(hd), out, status,
                         sink_weight=None if sink is None else sink.cuda(), **options)
    ops.raise_on_status(status)
    if options.get("sink") and sink is None:
        sink = torch.zeros(nh)
    want = plain_attention(q.view(T, nh, hd), pool, table, hd, page, [(i, n - 1) for i, n in enumerate(lengths)], 1 / math.sqrt(hd), options.get("window", 0),
                           options.get("softcap", 0.0), sink)
    return out.cpu().view(T, nh, hd), want


LENGTHS = [[1], [15, 16, 17, 1, 31, 32, 33], [64, 65, 255, 256, 257, 2, 700]]


@GPU
@pytest.mark.parametrize("lengths", LENGTHS, ids=["one", "short", "longer"])
@pytest.mark.parametrize("nh,nkv,hd,page", [(12, 2, 128, 64), (14, 2, 64, 16), (8, 8, 128, 16), (12, 1, 128, 48), (32, 2, 64, 32), (40, 2, 128, 64), (7, 1, 64, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_single_tokens(lengths, nh, nkv, hd, page, dtype):
    near(*single(lengths, nh, nkv, hd, page, dtype), dtype)


@GPU
@pytest.mark.parametrize("options", [dict(window=1), dict(window=40), dict(window=64, softcap=3.0), dict(sink=True), dict(softcap=20.0), dict(learned=True, softcap=5.0),
                                     dict(learned=True, window=33), dict(window=100000)], ids=str)
@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(12, 2, 128, 64, BF16), (14, 2, 64, 16, BF16), (24, 2, 64, 32, BF16), (6, 2, 128, 32, F32)])
def test_options_of_attention(options, nh, nkv, hd, page, dtype):
    options = dict(options)
    if options.pop("learned", False):
        options["sink_weight"] = torch.linspace(-3.0, 30.0, nh)
    near(*single([1, 33, 64, 290, 130], nh, nkv, hd, page, dtype, **options), dtype)


@GPU
@pytest.mark.parametrize("most", [5000, 131071])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_bound_far_above_the_lengths(most, dtype):
    """As a captured step has it: the ranges are cut for the longest text that there may be."""
    near(*single([3, 700, 65, 2100], 6, 1, 128, 64, dtype, most=most), dtype)


@GPU
def test_long_texts_in_many_ranges():
    near(*single([9001, 20000], 8, 1, 64, 64, BF16), BF16)
    near(*single([9001], 4, 1, 128, 16, F32), F32)


@GPU
def test_many_rows_in_few_ranges():
    near(*single([(37 * i) % 600 + 1 for i in range(150)], 12, 2, 64, 16, BF16), BF16)


@GPU
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores_and_a_row_that_is_no_number(dtype):
    q = torch.randn((3, 6 * 64), generator=torch.Generator().manual_seed(1)) * 200.0
    near(*single([300, 40, 7], 6, 2, 64, 16, dtype, q=q), dtype)
    q = torch.randn((3, 6 * 64), generator=torch.Generator().manual_seed(1))
    q[1, 5] = math.nan
    got, want = single([300, 900, 7], 6, 2, 64, 16, dtype, q=q)
    assert bool(torch.isnan(got[1, 0]).all()) and not bool(torch.isnan(got[1, 1:]).any())
    near(got, want, dtype)


@GPU
@pytest.mark.parametrize("lengths", [[4096, 3000], [2000] * 70], ids=["few", "many"])
def test_weights_are_rounded_beside_the_middle_of_the_codes(lengths):
    """Weights next to equal, so that every one of them is rounded.  A rounding to bfloat16 is off by at most 2^-8, by 2^-8 / sqrt(3) in the root of the mean of
    squares; one such is that of the results, one that of weight and step together, which counts for step (u - 8): as large as the values are, in the root of the
    mean of squares (codes in 0 .. 15 are 4.6 from 8, values are 7.5 steps lower and half a unit beside): 2^-8 sqrt(2 / 3) = 0.0032.  Against u itself, 8.8 in the
    root of the mean of squares, the second would be 1.9 times that."""
    nh, nkv, hd, page = 12, 2, 128, 64
    q = torch.randn((len(lengths), nh * hd), generator=torch.Generator().manual_seed(1)) * 0.05
    got, want = single(lengths, nh, nkv, hd, page, BF16, q=q)
    assert float((got.double() - want).norm() / want.norm()) < 0.0032


@GPU
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", ["key", "value"])
def test_a_held_group_that_is_no_number_shows_where_it_is_seen(dtype, what):
    nh, nkv, hd, page, lengths = 4, 2, 128, 16, [50, 51, 52]
    table, pages = make_table([52], page)
    table = table.expand(3, -1).contiguous()
    pool = make_pool(pages, nkv, hd, page)
    _, _, _, _, kp, vp = places(hd, page)
    spot = int((kp if what == "key" else vp)[50 % page, 70])
    pool[table[0, 50 // page].long(), 1, spot:spot + 2] = 255                 # position 50's second group of kv head 1
    q = torch.randn((3, nh * hd), generator=torch.Generator().manual_seed(3)).to(dtype)
    out, status = torch.empty((3, nh * hd), dtype=dtype, device="cuda"), ops.new_status("cuda")
    args = (pool.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda() - 1, nh, nkv, hd, page, 51, 0.1, out, status)
    ops.packed_attention(q.cuda(), *args)
    plan = ops.packed_plan([3], nh, nkv, hd, dtype, page, "cuda")
    want = plain_attention(q.view(3, nh, hd), pool, table, hd, page, [(i, n - 1) for i, n in enumerate(lengths)], 0.1)
    near(out.view(3, nh, hd), want, dtype)
    assert not bool(torch.isnan(out.view(3, nh, hd)[0]).any()) and bool(torch.isnan(out.view(3, nh, hd)[1, 2:, 64:]).all())
    out.zero_()                                                                # the same rows as one request's: one block, position 50 hidden from its first row
    ops.packed_attention(q.cuda(), *args, plan=plan)
    near(out.view(3, nh, hd), want, dtype)
    ops.raise_on_status(status)


@GPU
@pytest.mark.parametrize("parts", ["1:0", "3:20,1:100,7:0", "64:0", "63:5,65:5", "130:200,1:700,17:30,1:1,200:0", "2:64,2:63,2:62"])
@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(12, 2, 128, 64, BF16), (14, 2, 64, 16, BF16), (20, 1, 128, 48, BF16), (4, 4, 64, 128, BF16), (12, 2, 128, 64, F32),
                                                   (9, 1, 64, 16, F32)])
@pytest.mark.parametrize("options", [dict(), dict(window=50), dict(softcap=9.0, sink=True)], ids=["plain", "window", "squashed"])
@pytest.mark.parametrize("many", [0, 1 << 30], ids=["written out", "packed"])
def test_attention_of_portions(parts, nh, nkv, hd, page, dtype, options, many, monkeypatch):
    if dtype == F32 and not many:
        pytest.skip("float queries have no pages written out")
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", many)
    parts = [tuple(int(v) for v in p.split(":")) for p in parts.split(",")]
    lens, starts = [n for n, _ in parts], [s for _, s in parts]
    lengths = [n + s for n, s in parts]
    table, pages = make_table(lengths, page)
    pool = make_pool(pages, nkv, hd, page, seed=8)
    poison(pool, table, lengths, hd, page)
    rows = [(i, p) for i, (n, s) in enumerate(parts) for p in range(s, s + n)]
    q = (torch.randn((len(rows), nh * hd), generator=torch.Generator().manual_seed(2)) * 1.3).to(dtype)
    want = plain_attention(q.view(-1, nh, hd), pool, table, hd, page, rows, 1 / math.sqrt(hd), options.get("window", 0), options.get("softcap", 0.0),
                           torch.zeros(nh) if options.get("sink") else None)
    positions = torch.tensor([p for _, p in rows], dtype=torch.int32).cuda()
    for given in (None, starts):
        plan = ops.packed_plan(lens, nh, nkv, hd, dtype, page, "cuda", starts=given)
        out, status = torch.full((len(rows) + 2, nh * hd), 7.0, dtype=dtype, device="cuda"), ops.new_status("cuda")
        ops.packed_attention(q.cuda(), pool.cuda(), table.cuda(), positions, nh, nkv, hd, page, max(lengths) - 1, 1 / math.sqrt(hd), out, status, plan=plan, **options)
        ops.raise_on_status(status)
        assert bool((out[len(rows):] == 7.0).all())                            # rows behind the last are left as they were
        got = out[:len(rows)].view(-1, nh, hd)
        # (those of many rows: keys, values and weights in halves, 2^-11 each, well inside what the weights' bfloat16 takes)
        near(got, want, dtype)


@GPU
@pytest.mark.parametrize("key,value,query", [(1e-12, 1e-20, 1e9), (3e6, 1e7, 1e-6), (1e20, 1e30, 1e-20), (1.0, 1e-30, 1.0)])
@pytest.mark.parametrize("hd", [64, 128])
def test_portions_over_keys_and_values_of_any_scale(key, value, query, hd, monkeypatch):
    """Half precision holds the written-out pages by a power of two for each kv head."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 0)
    nh, nkv, page, n = 4, 2, 32, 100
    table, pages = make_table([n], page)
    pool = make_pool(pages, nkv, hd, page, seed=3)
    pairs = pool.unflatten(2, (page // 16, -1))[..., 16 * hd:].view(BF16).unflatten(3, (16, 2, hd // 64, 2))
    pairs[..., 0, :, :] *= key
    pairs[..., 1, :, :] *= value
    pairs[:, 1] *= 0.01                                                        # the second kv head's scale is another
    poison(pool, table, [n], hd, page)
    q = (torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(2)) * query / (key * query)).to(BF16)
    out, status = torch.empty((n, nh * hd), dtype=BF16, device="cuda"), ops.new_status("cuda")
    ops.packed_attention(q.cuda(), pool.cuda(), table.cuda(), torch.arange(n, dtype=torch.int32, device="cuda"), nh, nkv, hd, page, n - 1, 1 / math.sqrt(hd), out, status,
                         plan=ops.packed_plan([n], nh, nkv, hd, BF16, page, "cuda"))
    ops.raise_on_status(status)
    want = plain_attention(q.view(n, nh, hd), pool, table, hd, page, [(0, i) for i in range(n)], 1 / math.sqrt(hd))
    for heads, scale in ((slice(0, 2), value), (slice(2, 4), value * 0.01)):
        near(out.view(n, nh, hd)[:, heads].double() / scale, want[:, heads] / scale, BF16)


# ------------------------------------------------------------------------------------------------ the choice of pages
def chosen(q, pool, table, lengths, nh, nkv, hd, page, top, first, recent):
    n = tiles_bytes(hd, page)
    ends = pool.cpu()[:, :, n:].contiguous().view(BF16).unflatten(2, (2, hd)).double()
    out = torch.full((len(lengths), nkv, top), -1, dtype=torch.int32)
    for r, length in enumerate(lengths):
        pages = -(-length // page)
        for h in range(nkv):
            if pages <= top:
                out[r, h, :pages] = torch.arange(pages)
                continue
            e = ends[table[r, :pages].long(), h]
            w = q[r].double().view(nkv, -1, hd)[h]
            score = torch.stack([torch.where(x > 0, x * e[:, 1], x * e[:, 0]).sum(-1) for x in w])
            score = score.float().nan_to_num(3.4028234e38, posinf=3.4028234e38, neginf=-math.inf).amax(0)
            score[:first] = math.inf
            score[pages - recent:] = math.inf
            out[r, h] = torch.sort(score, descending=True, stable=True).indices[:top].sort().values.int()
    return out


def selection(lengths, nh, nkv, hd, page, dtype, top, first, recent, seed=0, change=None, most=None):
    table, pages = make_table(lengths, page, seed)
    pool = make_pool(pages, nkv, hd, page, bounds=True, seed=seed)
    ends = torch.randn((pages, nkv, 2, hd), generator=torch.Generator().manual_seed(seed + 3)).sort(2).values.to(BF16)
    pool[:, :, tiles_bytes(hd, page):] = ends.flatten(2).view(torch.uint8)
    q = torch.randn((len(lengths), nh * hd), generator=torch.Generator().manual_seed(seed + 4)).to(dtype)
    if change:
        change(q, pool, table, tiles_bytes(hd, page))
    out, status = torch.full((len(lengths), nkv, top), 99, dtype=torch.int32, device="cuda"), ops.new_status("cuda")
    ops.packed_select(q.cuda(), pool.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda() - 1, nh, nkv, hd, page,
                      max(lengths) - 1 if most is None else most, out, status, first=first, recent=recent)
    ops.raise_on_status(status)
    return out.cpu(), chosen(q, pool, table, lengths, nh, nkv, hd, page, top, first, recent), q, pool, table


@GPU
@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(12, 2, 128, 64, BF16), (14, 2, 64, 16, BF16), (9, 1, 128, 16, BF16), (20, 1, 64, 16, BF16), (4, 4, 128, 16, F32)])
@pytest.mark.parametrize("top,first,recent", [(1, 0, 1), (4, 1, 1), (9, 0, 3), (33, 2, 2), (6, 3, 3)])
def test_the_pages_that_score_highest(nh, nkv, hd, page, dtype, top, first, recent):
    lengths = [1, page, 5 * page + 1, 40 * page, 33 * page, 34 * page - 1, 300 * page // (2 if page == 64 else 1) + 7]
    got, want, *_ = selection(lengths, nh, nkv, hd, page, dtype, top, first, recent)
    assert torch.equal(got, want)


@GPU
def test_many_pages_and_a_bound_far_above():
    got, want, *_ = selection([16 * 9000 + 3, 16 * 2100], 3, 1, 64, 16, BF16, 200, 1, 2)
    assert torch.equal(got, want)
    got, want, *_ = selection([700, 16 * 60], 3, 1, 64, 16, BF16, 8, 1, 2, most=16 * 36000 - 1)
    assert torch.equal(got, want)


@GPU
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [1, 9])
def test_scores_that_32_bits_do_not_tell_apart(dtype, heads):
    """Pages whose bounds differ by a unit in one feature, and pages that are equal: the choice is that of 64 bits."""
    def change(q, pool, table, n):
        data = pool[:, :, n:].contiguous().view(BF16)
        one = data[table[0, 3].long()].clone()
        g = torch.Generator().manual_seed(1)
        for i in range(2, 700):
            near = one.clone()
            f = int(torch.randint(0, 256, (1,), generator=g))
            if i % 3:
                near[:, f] = torch.nextafter(near[:, f].float(), torch.tensor(math.inf)).to(BF16) if i % 2 else (near[:, f].float() * (1 + 2.0 ** -7)).to(BF16)
            data[table[0, i].long()] = near
        pool[:, :, n:] = data.view(torch.uint8)
        q.copy_((q.float() * torch.logspace(-3, 3, q.shape[1])).to(q.dtype))
    got, want, *_ = selection([800 * 16], heads, 1, 128, 16, dtype, 150, 1, 2, change=change)
    assert torch.equal(got, want)


@GPU
@pytest.mark.parametrize("what", ["equal", "nought", "nan", "inf", "minus"])
def test_scores_that_are_equal_or_no_numbers(what):
    def change(q, pool, table, n):
        ends = pool[:, :, n:].view(BF16) if pool[:, :, n:].is_contiguous() else None
        assert ends is None
        data = pool[:, :, n:].contiguous().view(BF16)
        if what == "equal":
            data[:] = 1.5
        elif what == "nought":
            data[:] = 0.0
            data[::2] = -0.0
        elif what == "nan":
            data[table[0, 7].long()] = math.nan
            data[table[0, 20].long(), :, 3] = math.nan
        elif what == "inf":
            data[table[0, 9].long(), :, 64:] = math.inf
        else:
            data[table[0, 5:11].long()] = -math.inf
        pool[:, :, n:] = data.view(torch.uint8)
    got, want, *_ = selection([40 * 16 - 3, 25 * 16], 6, 2, 64, 16, BF16, 7, 1, 2, change=change)
    if what in ("nan", "inf"):
        assert {7, 20} <= set(got[0, 0].tolist()) if what == "nan" else True
    if what != "inf":                                  # (infinite bounds: infinities of both signs may meet in a sum)
        assert torch.equal(got, want)
    assert bool((got[:, :, 1:] > got[:, :, :-1]).all())


@GPU
@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(12, 2, 128, 64, BF16), (14, 2, 64, 16, BF16), (40, 2, 64, 16, BF16), (6, 2, 128, 32, F32)])
def test_attention_over_chosen_pages(nh, nkv, hd, page, dtype):
    lengths = [1, page + 3, 30 * page - 5, 12 * page, 50 * page + 1]
    table, count = make_table(lengths, page)
    pool = make_pool(count, nkv, hd, page, bounds=True, seed=4)
    poison(pool, table, lengths, hd, page)
    g = torch.Generator().manual_seed(7)
    pages = torch.full((5, nkv, 9), -1, dtype=torch.int32)
    for r, n in enumerate(lengths):
        have = -(-n // page)
        for h in range(nkv):
            pick = torch.randperm(have, generator=g)[:9 if h else 4].sort().values.int()
            pages[r, h, :pick.numel()] = pick
    pages[3, 0] = -1                                                           # nothing at all
    q = torch.randn((5, nh * hd), generator=g).to(dtype)
    out, status = torch.empty((5, nh * hd), dtype=dtype, device="cuda"), ops.new_status("cuda")
    ops.packed_attention(q.cuda(), pool.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda() - 1, nh, nkv, hd, page, max(lengths) - 1, 0.1, out, status,
                         pages=pages.cuda())
    ops.raise_on_status(status)
    near(out.view(5, nh, hd), plain_attention(q.view(5, nh, hd), pool, table, hd, page, [(i, n - 1) for i, n in enumerate(lengths)], 0.1, pages=pages), dtype)


# ------------------------------------------------------------------------------------------------ together, and where they are called from
class Step:
    """A decoding step of three requests: append, bounds, choice of pages, attention over them, and over everything."""
    nh, nkv, hd, page, top = 6, 2, 64, 16, 5

    def __init__(self, lengths, seed=0):
        self.lengths = lengths
        self.table, pages = make_table([n + 40 for n in lengths], self.page, seed)
        self.pool = make_pool(pages, self.nkv, self.hd, self.page, bounds=True, seed=seed).cuda()
        n, dev = len(lengths), dict(device="cuda")
        self.src = torch.empty((n, (self.nh + 2 * self.nkv) * self.hd), dtype=BF16, **dev)
        self.cos_sin = torch.empty((n, self.hd // 2, 2), dtype=F32, **dev)
        self.positions, self.req, self.dev_table = torch.zeros(n, dtype=torch.int32, **dev), torch.arange(n, dtype=torch.int32, **dev), self.table.cuda()
        self.status = ops.new_status("cuda")
        full = [(i, p) for i, n in enumerate(lengths) for p in range(self.page - 1, n, self.page)]
        req, at = (torch.tensor(v, dtype=torch.int32, **dev) for v in zip(*full)) if full else (self.req[:0], self.req[:0])
        ops.packed_bounds(self.pool, at, req, self.dev_table, self.hd, self.page, self.status)
        self.load(0)

    def load(self, i):
        """Inputs of the i-th step."""
        g = torch.Generator().manual_seed(100 + i)
        at = torch.tensor([n + i for n in self.lengths], dtype=torch.int32)
        self.src.copy_(torch.randn(self.src.shape, generator=g))
        self.positions.copy_(at)
        self.cos_sin.copy_(angles(at, self.hd))

    def __call__(self):
        a = (self.nh, self.nkv, self.hd)
        n, dev = len(self.lengths), self.src.device
        q, out, every = (torch.empty((n, self.nh * self.hd), dtype=BF16, device=dev) for _ in range(3))
        pages = torch.empty((n, self.nkv, self.top), dtype=torch.int32, device=dev)
        ops.packed_append(self.src, q, *a, self.hd, False, self.cos_sin, self.positions, self.req, self.dev_table, self.pool, self.page, self.status)
        ops.packed_bounds(self.pool, self.positions, self.req, self.dev_table, self.hd, self.page, self.status)
        ops.packed_select(q, self.pool, self.dev_table, self.positions, *a, self.page, 2000, pages, self.status, first=1, recent=1)
        ops.packed_attention(q, self.pool, self.dev_table, self.positions, *a, self.page, 2000, 0.125, out, self.status, pages=pages)
        ops.packed_attention(q, self.pool, self.dev_table, self.positions, *a, self.page, 2000, 0.125, every, self.status)
        return q, pages, out, every

    def check(self, q, pages, out, every):
        n, at = len(self.lengths), self.positions.cpu()
        rows = [(i, int(p)) for i, p in enumerate(at)]
        assert torch.equal(pages.cpu(), chosen(q.cpu(), self.pool, self.table, [p + 1 for _, p in rows], self.nh, self.nkv, self.hd, self.page, self.top, 1, 1))
        for got, which in ((out, pages.cpu()), (every, None)):
            near(got.view(n, self.nh, self.hd), plain_attention(q.cpu().view(n, self.nh, self.hd), self.pool.cpu(), self.table, self.hd, self.page, rows, 0.125,
                                                                pages=which), BF16, steps=0.5)


@GPU
def test_steps_one_behind_the_other():
    step = Step([15, 100, 31])
    for i in range(20):
        step.load(i)
        got = step()
        if i in (0, 1, 16, 19):
            step.check(*got)
    ops.raise_on_status(step.status)


@GPU
def test_two_captured_steps_replayed_in_turn():
    steps, graphs = [Step([15, 100, 31], 1), Step([300, 2], 2)], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            s()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = s()
        graphs.append((g, got))
    for i in range(4):
        for s, (g, _) in zip(steps, graphs):
            s.load(i)
            g.replay()
        for s, (g, got) in zip(steps, graphs):
            s.check(*got)


@GPU
def test_on_another_stream():
    step, side = Step([150, 3, 31]), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    step.check(*got)


@GPU
def test_two_streams_at_once():
    steps, sides, got = [Step([1500, 3, 31], 1), Step([700, 701], 2)], [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (step, side) in enumerate(zip(steps, sides)):
            with torch.cuda.stream(side):
                got[i] = step()
    for i, (step, side) in enumerate(zip(steps, sides)):
        side.synchronize()
        step.check(*got[i])


@GPU
def test_rows_apart_in_memory(monkeypatch):
    """Queries, results and portions' rows as parts of wider rows."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 20)                        # (the first request's pages are written out)
    nh, nkv, hd, page, lens = 6, 2, 64, 32, [70, 1, 9]
    lengths = [200, 300, 9]
    table, pages = make_table(lengths, page)
    pool = make_pool(pages, nkv, hd, page, seed=2)
    rows = [(i, p) for i, (n, length) in enumerate(zip(lens, lengths)) for p in range(length - n, length)]
    wide = torch.randn((80, nh * hd + 64), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    q, positions, status = wide[:, 64:], torch.tensor([p for _, p in rows], dtype=torch.int32).cuda(), ops.new_status("cuda")
    room = torch.full((80, nh * hd + 16), 7.0, dtype=BF16, device="cuda")
    ops.packed_attention(q, pool.cuda(), table.cuda(), positions, nh, nkv, hd, page, 299, 0.125, room[:, 8:-8], status,
                         plan=ops.packed_plan(lens, nh, nkv, hd, BF16, page, "cuda"))
    ops.raise_on_status(status)
    near(room[:, 8:-8].reshape(80, nh, hd), plain_attention(q.cpu().view(80, nh, hd), pool, table, hd, page, rows, 0.125), BF16)
    assert bool((room[:, :8] == 7.0).all()) and bool((room[:, -8:] == 7.0).all())
    with pytest.raises(ops.KernelError, match="misaligned"):
        ops.packed_attention(wide[:, 1:1 + nh * hd], pool.cuda(), table.cuda(), positions, nh, nkv, hd, page, 299, 0.125, room[:, 8:-8], status,
                             plan=ops.packed_plan(lens, nh, nkv, hd, BF16, page, "cuda"))


@GPU
def test_pages_beyond_four_gigabytes(monkeypatch):
    """A pool of 5 GB whose last pages are used: every call finds them."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 30)                        # (the portion's pages are written out)
    nh, nkv, hd, page, length = 8, 4, 128, 64, 150
    few = make_pool(3, nkv, hd, page, bounds=True, seed=1)
    pages = 5_000_000_000 // few[0].numel()
    pool = torch.empty((pages, nkv, few.shape[2]), dtype=torch.uint8, device="cuda")
    pool[-3:] = few.cuda()
    small, table = torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    status, g = ops.new_status("cuda"), torch.Generator().manual_seed(5)
    at, req = torch.tensor([length - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    src = torch.randn((1, (nh + 2 * nkv) * hd), generator=g).to(BF16)
    q, values = torch.empty((1, nh * hd), dtype=BF16, device="cuda"), torch.empty((1, 2, nkv, hd), device="cuda")
    ops.packed_append(src.cuda(), q, nh, nkv, hd, 0, False, None, at, req, table, pool, page, status)
    ops.packed_rows(pool, at, req, table, hd, page, values, status)
    for k, (u, step, lowest) in enumerate(map(quantised, (src.view(-1, hd)[nh:nh + nkv].double(), src.view(-1, hd)[nh + nkv:].double()))):
        assert torch.equal(values[0, k].cpu(), (lowest + step * u).float())
    ops.packed_bounds(pool, torch.tensor([63, 127], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), table, hd, page, status)
    near_pool, pick = pool[-3:].cpu(), torch.empty((1, nkv, 2), dtype=torch.int32, device="cuda")
    ops.packed_select(q, pool, table, at, nh, nkv, hd, page, length - 1, pick, status, first=0, recent=1)
    assert torch.equal(pick.cpu(), chosen(q.cpu(), near_pool, small, [length], nh, nkv, hd, page, 2, 0, 1))
    for n in (1, 70):                                                          # single tokens, and a portion by way of pages written out
        rows = q.expand(n, -1).contiguous()
        positions = torch.arange(length - n, length, dtype=torch.int32, device="cuda")
        out = torch.empty_like(rows)
        ops.packed_attention(rows, pool, table, positions, nh, nkv, hd, page, length - 1, 0.1, out, status,
                             plan=ops.packed_plan([n], nh, nkv, hd, BF16, page, "cuda"))
        near(out.view(n, nh, hd), plain_attention(rows.cpu().view(n, nh, hd), near_pool, small, hd, page, [(0, int(p)) for p in positions], 0.1), BF16, steps=0.6)
    ops.raise_on_status(status)


@GPU
def test_the_same_call_twice_is_the_same():
    step = Step([1500, 3, 310])
    one, two = step(), step()
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@GPU
def test_calls_without_rows():
    hd, page = 64, 16
    pool, table = make_pool(2, 1, hd, page, bounds=True).cuda(), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    none, i0 = torch.empty((0, 3 * hd), dtype=BF16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    q = torch.empty((0, hd), dtype=BF16, device="cuda")
    before = pool.clone()
    ops.packed_append(none, q, 1, 1, hd, 0, False, None, i0, i0, table, pool, page, None)
    ops.packed_bounds(pool, i0, i0, table, hd, page, None)
    ops.packed_rows(pool, i0, i0, table, hd, page, torch.empty((0, 2, 1, hd), device="cuda"), None)
    ops.packed_attention(q, pool, table, i0, 1, 1, hd, page, 0, 1.0, torch.empty_like(q), None)
    ops.packed_attention(q, pool, table, i0, 1, 1, hd, page, 0, 1.0, torch.empty_like(q), None, plan=ops.packed_plan([], 1, 1, hd, BF16, page, "cuda"))
    ops.packed_select(q, pool, table, i0, 1, 1, hd, page, 0, torch.empty((0, 1, 2), dtype=torch.int32, device="cuda"), None)
    assert torch.equal(pool, before)


# ------------------------------------------------------------------------------------------------ refusals
@GPU
@pytest.mark.parametrize("entry,request_", [(-1, 0), (9, 0), (-5, 0), (0, 3)])
def test_bad_pages_are_recorded(entry, request_, monkeypatch):
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", 0)                         # (the many rows' pages are written out)
    """A table's entry outside the pool, or a request without a table: nothing outside is touched, and the status says so."""
    hd, page = 64, 16
    pool = make_pool(3, 1, hd, page, bounds=True).cuda()
    before = pool.clone()
    table = torch.tensor([[1, entry if entry else -1]], dtype=torch.int32, device="cuda")
    positions, req = torch.tensor([31], dtype=torch.int32, device="cuda"), torch.tensor([request_], dtype=torch.int32, device="cuda")
    src, q = torch.ones((1, 3 * hd), dtype=BF16, device="cuda"), torch.empty((1, hd), dtype=BF16, device="cuda")
    calls = [lambda s: ops.packed_append(src, q, 1, 1, hd, 0, False, None, positions, req, table, pool, page, s),
             lambda s: ops.packed_bounds(pool, positions, req, table, hd, page, s),
             lambda s: ops.packed_rows(pool, positions, req, table, hd, page, torch.empty((1, 2, 1, hd), device="cuda"), s)]
    if not request_:
        out = torch.empty_like(q)
        calls += [lambda s: ops.packed_attention(src[:, :hd], pool, table, positions, 1, 1, hd, page, 31, 1.0, out, s),
                  lambda s: ops.packed_select(src[:, :hd], pool, table, positions, 1, 1, hd, page, 31, torch.empty((1, 1, 1), dtype=torch.int32, device="cuda"), s,
                                              first=0)]
        many = torch.ones((70, hd), dtype=BF16, device="cuda")
        calls.append(lambda s: ops.packed_attention(many, pool, table.expand(1, 2).contiguous(), torch.arange(-38, 32, dtype=torch.int32, device="cuda").clamp(min=0), 1, 1, hd,
                                                    page, 31, 1.0, torch.empty_like(many), s, plan=ops.packed_plan([70], 1, 1, hd, BF16, page, "cuda")))
    for call in calls:
        status = ops.new_status("cuda")
        call(status)
        with pytest.raises(ops.KernelError, match="block-table"):
            ops.raise_on_status(status)
    assert torch.equal(pool, before)


@GPU
def test_what_does_not_fit_is_refused():
    hd, page, nh, nkv, T = 64, 16, 4, 2, 3
    dev = dict(device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    good = dict(src=torch.zeros((T, 8 * hd), dtype=BF16, **dev), q=torch.zeros((T, nh * hd), dtype=BF16, **dev), cos=torch.zeros((T, 32, 2), **dev),
                positions=torch.zeros(T, **i32), req=torch.arange(T, **i32), table=torch.zeros((T, 2), **i32), pool=make_pool(4, nkv, hd, page, True).cuda(),
                rot=hd, hd=hd, page=page, nh=nh, nkv=nkv, out=torch.zeros((T, nh * hd), dtype=BF16, **dev), pages=torch.zeros((T, nkv, 2), **i32),
                values=torch.zeros((T, 2, nkv, hd), **dev), window=0, plan=None, softcap=0.0, sink=None, first=1, recent=1, most=31, given=None)

    def append(a):
        ops.packed_append(a["src"], a["q"], a["nh"], a["nkv"], a["hd"], a["rot"], False, a["cos"], a["positions"], a["req"], a["table"], a["pool"], a["page"], None)

    def bounds(a):
        ops.packed_bounds(a["pool"], a["positions"], a["req"], a["table"], a["hd"], a["page"], None)

    def rows(a):
        ops.packed_rows(a["pool"], a["positions"], a["req"], a["table"], a["hd"], a["page"], a["values"], None)

    def attend(a):
        ops.packed_attention(a["q"], a["pool"], a["table"], a["positions"], a["nh"], a["nkv"], a["hd"], a["page"], a["most"], 1.0, a["out"], None, plan=a["plan"],
                             window=a["window"], softcap=a["softcap"], sink_weight=a["sink"], pages=a["given"])

    def select(a):
        ops.packed_select(a["q"], a["pool"], a["table"], a["positions"], a["nh"], a["nkv"], a["hd"], a["page"], a["most"], a["pages"], None, first=a["first"],
                          recent=a["recent"])

    every = (append, bounds, rows, attend, select)
    for call in every:
        call(good)
    ops.raise_on_status(ops.new_status("cuda"))
    plain = make_pool(4, nkv, hd, page).cuda()
    wrong = [(every, dict(pool=good["pool"].cpu())), (every, dict(pool=good["pool"].float())), (every, dict(pool=good["pool"][:, :, :-16])), (every, dict(hd=128)),
             (every, dict(page=32)), (every, dict(page=24)), (every, dict(positions=good["positions"].long())), (every, dict(table=good["table"][0])),
             ((append, attend, select), dict(nkv=1)), ((bounds, select), dict(pool=plain)), ((append, bounds, rows), dict(req=good["req"].long())),
             ((append, bounds, rows), dict(req=good["req"][:2])), ((append, attend, select), dict(positions=good["positions"][:2])),
             ((append,), dict(src=good["src"][:, :-1])), ((append,), dict(q=good["src"])), ((append,), dict(rot=66)), ((append,), dict(rot=7)), ((append,), dict(cos=None)),
             ((append,), dict(cos=good["cos"].to(BF16))), ((append,), dict(src=good["src"].half())), ((append,), dict(src=torch.zeros((T, 8 * hd + 1), dtype=BF16, **dev)[:, 1:])),
             ((rows,), dict(values=good["values"][:2])), ((rows,), dict(values=good["values"].half())),
             ((attend,), dict(out=good["out"].float())), ((attend,), dict(q=good["q"].half())), ((attend,), dict(out=good["out"][:2])), ((attend,), dict(nh=3)),
             ((attend,), dict(window=-1)), ((attend,), dict(softcap=-1.0)), ((attend,), dict(sink=torch.zeros(3, **dev))), ((attend,), dict(table=good["table"][:2])),
             ((attend,), dict(plan=ops.packed_plan([2], nh, nkv, hd, BF16, page, "cuda"))), ((attend,), dict(plan=ops.packed_plan([3], 2, nkv, hd, BF16, page, "cuda"))),
             ((attend,), dict(given=good["pages"][:2])), ((attend,), dict(given=good["pages"].long())), ((attend,), dict(given=good["pages"], window=3)),
             ((attend,), dict(given=good["pages"], plan=ops.packed_plan([1, 1, 1], nh, nkv, hd, BF16, page, "cuda"))),
             ((select,), dict(recent=0)), ((select,), dict(first=2)), ((select,), dict(first=-1)), ((select,), dict(pages=good["pages"].long())),
             ((select,), dict(pages=good["pages"][:2])), ((select,), dict(most=16 * 36000)), ((select,), dict(q=good["q"].half()))]
    for calls, change in wrong:
        for call in calls:
            with pytest.raises(ops.KernelError):
                call(good | change)
