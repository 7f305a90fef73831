"""Attention of single tokens over positions that their requests share: against a plain restatement in 64 bits, against the attention that
shares nothing (bit for bit in float32), and the host's cutting of the work."""
import math

import numpy as np
import pytest
import torch

from beglin_b200.cache import SharedPrefix
from beglin_b200.csrc import ops, shared_plan

DEV = "cuda:0"


class Case:
    """Requests of a step of single tokens: `groups` [(rows, shared positions)], `lengths` positions of every row.  Pages in shuffled order, those that
    nobody holds and positions behind a request's end poisoned, a page that sharing ends inside held by every row of the group."""

    def __init__(self, groups, lengths, nh, nkv, hd, page, dtype, seed=0, vd=None, q_pad=0, poison=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.groups, self.lengths, self.nh, self.nkv, self.hd, self.vd, self.page = groups, lengths, nh, nkv, hd, vd or hd, page
        T, vd = len(lengths), vd or hd
        rnd = lambda *s: torch.randn(*s, generator=g)
        common, pages = {}, 0
        for rows, n in groups:
            k, v = rnd(n, nkv, hd), rnd(n, nkv, vd)
            for r in rows:
                common[r] = (list(range(pages, pages + n // page)), n, k, v)
            pages += n // page
        tables = []
        self.keys, self.values = [], []
        for r, length in enumerate(lengths):
            together, n, k, v = common.get(r, ([], 0, rnd(0, nkv, hd), rnd(0, nkv, vd)))
            length = max(length, n)                        # (a row may see less than its group shares)
            self.keys.append(torch.cat([k, rnd(length - n, nkv, hd)]).to(dtype))
            self.values.append(torch.cat([v, rnd(length - n, nkv, vd)]).to(dtype))
            more = -(-length // page) - len(together)
            tables.append(together + list(range(pages, pages + more)))
            pages += more
        pages += 3
        order = torch.randperm(pages, generator=g).tolist()
        flat = torch.full((pages, nkv * page * (hd + vd)), poison, dtype=dtype)
        ks = flat[:, :nkv * page * hd].view(pages, nkv, page, hd)
        vs = flat[:, nkv * page * hd:].view(pages, nkv, page, vd)
        self.table = torch.full((T, max(len(t) for t in tables) + 2), -1, dtype=torch.int32)
        for r, t in enumerate(tables):
            for i, p in enumerate(t):
                self.table[r, i] = order[p]
                n = min(page, self.keys[r].shape[0] - i * page)
                ks[order[p], :, :n] = self.keys[r][i * page:i * page + n].transpose(0, 1)
                vs[order[p], :, :n] = self.values[r][i * page:i * page + n].transpose(0, 1)
        self.pool = flat if vd != hd else flat.view(pages, 2, nkv, page, hd)
        self.q = (rnd(T, nh * hd + q_pad) * 1.5).to(dtype)[:, :nh * hd]
        self.positions = torch.tensor(lengths, dtype=torch.int32) - 1
        self.scale = 1.0 / math.sqrt(hd)
        self.shared = SharedPrefix(T, groups)

    def plain(self, sink=None, cap=0.0):
        """(result, sum of weight times magnitude of value) float64 [T, nh * vd]."""
        per, out, size = self.nh // self.nkv, [], []
        for r, n in enumerate(self.lengths):
            k, v = self.keys[r][:n].double().repeat_interleave(per, 1), self.values[r][:n].double().repeat_interleave(per, 1)
            s = torch.einsum("hd,nhd->hn", self.q[r].double().view(self.nh, self.hd), k) * self.scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if sink is not None:
                s = torch.cat([s, sink.double()[:, None]], 1)
            w = torch.softmax(s, 1)[:, :n]
            out.append(torch.einsum("hn,nhd->hd", w, v).reshape(-1))
            size.append(torch.einsum("hn,nhd->hd", w, v.abs()).reshape(-1))
        return torch.stack(out), torch.stack(size)

    def run(self, prefer=None, sink=None, cap=0.0, fixed=False, max_position=None, plan=None, split=256):
        to = lambda t: t.to(DEV)
        buf = torch.full((self.q.shape[0], self.q.stride(0)), 3.0, dtype=self.q.dtype, device=DEV)
        q = buf[:, :self.q.shape[1]]
        q.copy_(self.q)
        prefer = prefer or ("tc" if self.pool.dtype == torch.bfloat16 else "auto")
        plan = plan or ops.shared_plan(self.shared, self.nh, self.nkv, self.hd, self.pool.dtype, page_size=self.page, vd=self.vd, split=split, prefer=prefer,
                                       device=DEV, fixed=fixed)
        wide = torch.full((len(self.lengths), self.nh * self.vd + 8), 7.0, dtype=self.q.dtype, device=DEV)
        out, status = wide[:, :self.nh * self.vd], ops.new_status(DEV)
        ops.shared_attention(q, to(self.pool), to(self.table), to(self.positions), plan, max(self.lengths) - 1 if max_position is None else max_position,
                             self.scale, out, status, sink_weight=None if sink is None else to(sink), softcap=cap)
        ops.raise_on_status(status)
        assert bool((wide[:, self.nh * self.vd:] == 7.0).all())
        return out.cpu(), plan

    def alone(self, split=256, sink=None, cap=0.0):
        """The attention that shares nothing, by the float kernels."""
        T = len(self.lengths)
        kernel, bq, tile = ops.attention_plan(self.nh // self.nkv, self.hd, self.pool.dtype, True, "generic", self.page, vd=self.vd)
        out, status = torch.empty(T, self.nh * self.vd, dtype=self.q.dtype, device=DEV), ops.new_status(DEV)
        blocks = torch.tensor([(r, r, 1) for r in range(T)], dtype=torch.int32, device=DEV)
        q = self.q.contiguous().to(DEV)
        ops.attention(q, q.stride(0), self.pool.to(DEV), self.table.to(DEV), self.positions.to(DEV), blocks, T, max(self.lengths) - 1, T, self.nh, self.nkv,
                      self.hd, 0, split, tile, bq, self.scale, out, status, kernel, vd=self.vd, sink_weight=None if sink is None else sink.to(DEV), softcap=cap)
        ops.raise_on_status(status)
        return out.cpu()


def _one(n, shared, lo=1, hi=70, front=0, back=0):
    """One group of n rows between rows of their own, lengths that differ."""
    lengths = [30 + 17 * i for i in range(front)] + [shared + lo + (13 * i) % (hi - lo + 1) for i in range(n)] + [5 + 64 * i for i in range(back)]
    return [(list(range(front, front + n)), shared)], lengths


SETS = {
    "two": _one(2, 64, 1, 1), "short": _one(3, 7, 1, 9), "odd": _one(5, 333, 1, 70), "many": _one(45, 1000, 1, 300, 1, 2), "long": _one(9, 5000, 1, 700),
    "mixed": ([([3, 0, 6], 200), ([1, 5], 1030), ([2], 64)], [210, 1031, 300, 201, 9, 2000, 777, 1]),
    "inside": ([([0, 1, 2, 3], 300)], [20, 300, 301, 65]),           # rows that see less than their group shares
    "none": ([], [1, 64, 65, 700]),
}


def bound(size, want, dtype):
    """Weights rounded to bfloat16 (2^-8 of weight times value each), a result rounded once (2^-8 of it); the rest, exponentials of 2^-22 and sums of floats
    over scores below 2^6 whose own error is 2^-17, is below 2^-10 of the first."""
    assert dtype == torch.bfloat16
    return 2.0 ** -8 * (size * (1 + 2.0 ** -10 * 4) + want.abs()) + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("name", SETS)
@pytest.mark.parametrize("nh,nkv,hd,page", [(12, 2, 128, 64), (14, 2, 64, 16), (4, 4, 128, 8), (32, 2, 64, 64), (7, 1, 128, 1)])
def test_shared_attention_on_tensor_cores(name, nh, nkv, hd, page):
    groups, lengths = SETS[name]
    c = Case(groups, lengths, nh, nkv, hd, page, torch.bfloat16, seed=len(name) + hd)
    got, plan = c.run()
    assert plan.kernel == "tc"
    want, size = c.plain()
    assert torch.isfinite(got.float()).all()
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("block,length", [(128, 192), (256, 192), (256, 64), (256, 6400)])
@pytest.mark.parametrize("name", ["many", "long", "mixed"])
@pytest.mark.parametrize("nh,nkv,hd", [(12, 2, 128), (32, 2, 64), (16, 1, 128)])
def test_shared_attention_in_blocks_of_one_and_of_two_tiles_of_rows(name, nh, nkv, hd, block, length, monkeypatch):
    monkeypatch.setattr(shared_plan, "cut_ranges", lambda *a: (block, length, 0.0))
    monkeypatch.setattr(shared_plan, "items_room", lambda *a: 3000)
    monkeypatch.setattr(ops.SharedPlan, "MOST_RANGES", 100)
    c = Case(*SETS[name], nh, nkv, hd, 64, torch.bfloat16, seed=nh)
    got, plan = c.run()
    assert int(plan.items[:plan.n_items, 2].max()) == min(block, nh // nkv * max(len(g) for g, _ in c.groups))
    want, size = c.plain()
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["odd", "mixed", "many"])
@pytest.mark.parametrize("options", [dict(sink=True), dict(cap=20.0), dict(sink=True, cap=5.0)], ids=["sink", "cap", "both"])
def test_shared_attention_options(name, options):
    groups, lengths = SETS[name]
    c = Case(groups, lengths, 12, 4, 128, 64, torch.bfloat16, seed=3, q_pad=24)
    sink = torch.linspace(-3, 4, 12) if options.get("sink") else None
    got, _ = c.run(sink=sink, cap=options.get("cap", 0.0))
    want, size = c.plain(sink, options.get("cap", 0.0))
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())
    got, plan = c.run(sink=sink, cap=options.get("cap", 0.0), prefer="generic")
    assert plan.kernel == "generic"
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", SETS)
@pytest.mark.parametrize("nh,nkv,hd,vd,page,split", [(12, 2, 128, 128, 64, 256), (6, 3, 64, 64, 16, 64), (4, 2, 80, 80, 5, 128), (5, 1, 36, 20, 24, 64),
                                                     (2, 1, 256, 256, 16, 64), (16, 1, 128, 64, 64, 64)])
def test_shared_attention_in_float_is_that_without_sharing(name, nh, nkv, hd, vd, page, split):
    groups, lengths = SETS[name]
    c = Case(groups, lengths, nh, nkv, hd, page, torch.float32, seed=len(name) + hd, vd=vd, poison=float("nan") if name != "inside" else 0.0)
    got, plan = c.run(split=split)
    assert plan.kernel == "generic"
    assert torch.equal(got, c.alone(split))
    want, size = c.plain()
    # scores: sums of hd products of floats, each operand's parts good to 2^-24, so off by at most hd 2^-24 sum|q k| scale (below 2^-13 here); weights and
    # values likewise, and sums over the keys of one split after the other
    assert bool(((got.double() - want).abs() <= 2.0 ** -13 * size).all())
    sink = torch.linspace(-1, 2, nh)
    assert torch.equal(c.run(split=split, sink=sink, cap=9.0)[0], c.alone(split, sink, 9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shared_attention_of_fixed_shape_follows_its_groups(dtype):
    """A captured call serves the groups that its plan is renewed for."""
    sets = ["many", "none", "odd", "long"]
    cases = {}
    for name in sets:
        groups, lengths = SETS[name]
        n = 48                                             # rows that share nothing fill the batch
        cases[name] = Case(groups, lengths + [1 + 3 * i for i in range(n - len(lengths))], 12, 2, 128, 64, dtype, seed=4)
    pages = max(c.pool.shape[0] for c in cases.values())
    width = max(c.table.shape[1] for c in cases.values())
    c = cases["many"]
    plan = ops.shared_plan(c.shared, 12, 2, 128, dtype, prefer="tc" if dtype == torch.bfloat16 else "auto", device=DEV, fixed=True)
    q = torch.zeros(48, 12 * 128, dtype=dtype, device=DEV)
    pool = torch.zeros((pages,) + tuple(c.pool.shape[1:]), dtype=dtype, device=DEV)
    table = torch.full((48, width), -1, dtype=torch.int32, device=DEV)
    positions, out, status = torch.zeros(48, dtype=torch.int32, device=DEV), torch.zeros_like(q), ops.new_status(DEV)
    call = lambda: ops.shared_attention(q, pool, table, positions, plan, 8191, c.scale, out, status)

    def load(c):
        q.copy_(c.q)
        pool.zero_()
        pool[:c.pool.shape[0]].copy_(c.pool)
        table.fill_(-1)
        table[:, :c.table.shape[1]].copy_(c.table)
        positions.copy_(c.positions)
        plan.update(c.shared)

    load(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for name in sets + sets[:1]:
        load(cases[name])
        out.fill_(9.0)
        graph.replay()
        ops.raise_on_status(status)
        want, size = cases[name].plain()
        got = out.cpu().double()
        if dtype == torch.float32:
            assert torch.equal(out.cpu(), cases[name].alone())
        else:
            assert bool(((got - want).abs() <= bound(size, want, dtype)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kept", [0, 1, 2])
def test_shared_attention_of_groups_that_pay(kept, monkeypatch):
    """Groups that are left to their rows' own pages beside groups that are read once."""
    monkeypatch.setattr(shared_plan, "worth_sharing", lambda shared, *a: shared.groups[:kept])
    c = Case(*SETS["mixed"], 12, 2, 128, 64, torch.bfloat16, seed=5)
    got, plan = c.run(prefer="auto")
    assert plan.shares == (kept > 0)
    want, size = c.plain()
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 4.0])
@pytest.mark.parametrize("sink", [None, 0.0, 30.0])
@pytest.mark.parametrize("lengths", [[1], [0, 65, 64, 1, 130], [(37 * i) % 190 + (i != 5) for i in range(90)]], ids=["one", "few", "many"])
@pytest.mark.parametrize("nh,nkv,hd,page", [(12, 2, 128, 64), (32, 2, 128, 16), (14, 2, 64, 64), (9, 3, 64, 8)])
def test_rows_that_share_nothing_are_finished_by_one_kernel(nh, nkv, hd, page, lengths, sink, cap):
    """Rows that share nothing and are short, a row that sees nothing among them; few rows the same with the joining (a bound on the positions that cuts them into
    ranges)."""
    c = Case([], lengths, nh, nkv, hd, page, torch.bfloat16, seed=len(lengths))
    weight = None if sink is None else torch.linspace(-2.0, 2.0, nh) + sink
    want, size = c.plain(weight, cap)
    before = ops.launch_count()
    got, plan = c.run(sink=weight, cap=cap)
    assert plan.n_items == 0 and ops.launch_count() - before == 1
    assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())
    before = ops.launch_count()
    joined, _ = c.run(sink=weight, cap=cap, plan=plan, max_position=20000)
    assert ops.launch_count() - before == (2 if len(lengths) < 10 else 1)
    assert bool(((joined.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())
    assert bool((got[[n == 0 for n in lengths]] == 0).all()) and bool((joined[[n == 0 for n in lengths]] == 0).all())


@pytest.mark.gpu
def test_a_page_that_is_not_there_is_recorded_where_nothing_is_shared():
    for page in (9999, -1):
        c = Case([], [200, 100, 130], 4, 2, 128, 64, torch.bfloat16)
        c.table[1, 1] = page
        with pytest.raises(ops.KernelError, match="page pool"):
            c.run()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shared_attention_twice_is_the_same(dtype):
    c = Case(*SETS["many"], 12, 2, 128, 64, dtype, seed=9)
    a, plan = c.run()
    assert torch.equal(a, c.run(plan=plan)[0])
    assert torch.equal(a, c.run()[0])


@pytest.mark.gpu
@pytest.mark.parametrize("prefer", ["tc", "generic"])
@pytest.mark.parametrize("row,entry", [(0, 1), (4, 6)])
def test_shared_attention_records_bad_pages(prefer, row, entry):
    """A page beyond the pool, or none, in what the group shares (the first row's table counts) or among a row's own."""
    c = Case(*SETS["odd"], 4, 2, 128, 64, torch.bfloat16, seed=1)
    c.lengths = [n if i != 4 else 450 for i, n in enumerate(c.lengths)]
    c.positions = torch.tensor(c.lengths, dtype=torch.int32) - 1
    for page in (c.pool.shape[0], -1):
        c.table[row, entry] = page
        with pytest.raises(ops.KernelError, match="page pool"):
            c.run(prefer=prefer)


# ------------------------------------------------------------------------------------------------ without a GPU
def test_groups_are_checked():
    with pytest.raises(ValueError, match="outside"):
        SharedPrefix(3, [([1, 3], 64)])
    with pytest.raises(ValueError, match="twice"):
        SharedPrefix(3, [([0, 1], 64), ([1, 2], 64)])
    with pytest.raises(ValueError, match="shares"):
        SharedPrefix(3, [([0, 1], -1)])
    assert SharedPrefix(3, [([0, 1], 0), ([2], 9)]).groups == []
    assert SharedPrefix(3, [([0, 2], 9)]) == SharedPrefix(3, [((0, 2), 9)]) != SharedPrefix(3, [((2, 0), 9)])


def _random_groups(rng):
    n = int(rng.integers(1, 90))
    order, groups, at = rng.permutation(n).tolist(), [], 0
    while at < n and rng.random() < 0.8:
        k = int(rng.integers(1, n - at + 1))
        groups.append((order[at:at + k], int(2 ** rng.uniform(0, 15))))
        at += k
    return SharedPrefix(n, groups)


@pytest.mark.parametrize("seed", range(25))
def test_every_position_of_a_row_is_taken_once(seed):
    rng = np.random.default_rng(seed)
    shared = _random_groups(rng)
    n, bq, nkv, split = shared.n_rows, int(rng.integers(1, 40)), int(rng.choice([1, 2, 8])), 64 * int(rng.integers(1, 5))
    of_row = {r: (g[0], p) for g, p in shared.groups for r in g}
    blocks, rows = shared_plan.shared_blocks(shared, bq, split, shared_plan.blocks_room(n))
    taken = {r: [] for r in range(n)}
    for req, at, k, lo, hi, last, _, _ in blocks.tolist():
        for r in rows[at:at + k].tolist():
            assert req == (r if hi == shared_plan.MOST else of_row[r][0]) and k <= bq or k == 1
            taken[r].append((lo, hi))
            assert last == (hi * split - 1 if hi != shared_plan.MOST else shared_plan.MOST)
    for r, spans in taken.items():
        whole = of_row.get(r, (0, 0))[1] // split
        assert sorted(spans) == ([(0, whole)] if whole else []) + [(whole, shared_plan.MOST)]
    heads = int(rng.choice([1, 6, 7, 16]))
    room = shared_plan.items_room(n, heads, nkv, 148)
    items, rows, first, parts = shared_plan.shared_items(shared, heads, nkv, 148, room, 64)
    spans = {(r, h): {} for r in range(n) for h in range(heads)}
    for req, at, k, lo, hi, slot, _, _ in items.tolist():
        assert k <= 256 and lo % shared_plan.TILE == 0
        for i in range(at, at + k):
            r, h = int(rows[i // heads]), i % heads
            assert req == of_row[r][0] and lo < hi and slot not in spans[r, h]
            spans[r, h][slot] = (lo, hi)
    for r in range(n):
        p = of_row.get(r, (0, 0))[1]
        for h in range(heads):
            assert first[r] == p and parts[r] == len(spans[r, h]) <= 64
            at = 0
            for slot in range(len(spans[r, h])):
                assert spans[r, h][slot][0] == at
                at = spans[r, h][slot][1]
            assert at == p


def test_groups_that_pay_are_kept():
    """Few rows of few positions are left alone; many rows of many positions are not."""
    own, alone = (lambda streams, positions: ops.own_ranges(streams, positions, 148)), (lambda streams, positions: ops.decode_splits(streams, positions, 148))
    args = (6, 2, 148, 444, 64, own, alone, 512)
    keep = lambda n, groups: shared_plan.worth_sharing(SharedPrefix(n, groups), *args)
    assert keep(2, [([0, 1], 512)]) == []
    assert keep(64, [(range(64), 8192)]) == [(tuple(range(64)), 8192)]
    big, small = (tuple(range(40)), 20000), ((40, 41), 64)
    assert big in keep(42, [small, big])
    assert keep(3, []) == []


def test_shared_attention_refuses_what_does_not_fit():
    with pytest.raises(ops.KernelError, match="multiple"):
        ops.shared_plan(SharedPrefix(2, []), 5, 2, 64, torch.bfloat16, device="cpu")
    with pytest.raises(ops.KernelError, match="choice"):
        ops.shared_plan(SharedPrefix(2, []), 4, 2, 64, torch.bfloat16, prefer="best", device="cpu")
    with pytest.raises(ops.KernelError, match="do not take"):
        ops.shared_plan(SharedPrefix(2, []), 4, 2, 96, torch.bfloat16, prefer="tc", device="cpu")
    with pytest.raises(ops.KernelError, match="do not take"):
        ops.shared_plan(SharedPrefix(2, []), 34, 2, 64, torch.bfloat16, prefer="tc", device="cpu")
    with pytest.raises(ops.KernelError, match="not supported"):
        ops.shared_plan(SharedPrefix(2, []), 4, 2, 300, torch.float32, device="cpu")
    with pytest.raises(ops.KernelError, match="whole tiles"):
        ops.shared_plan(SharedPrefix(2, []), 4, 2, 64, torch.float32, split=100, device="cpu")
    plan = ops.shared_plan(SharedPrefix(2, [([0, 1], 64)]), 4, 2, 64, torch.bfloat16, device="cpu")
    with pytest.raises(ops.KernelError, match="groups of 3 rows"):
        plan.update(SharedPrefix(3, []))
    q, pool = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(5, 2, 2, 64, 64, dtype=torch.bfloat16)
    table, positions = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def refused(match, q=q, pool=pool, table=table, positions=positions, most=70, out=None, **kw):
        with pytest.raises(ops.KernelError, match=match):
            ops.shared_attention(q, pool, table, positions, plan, most, 0.125, torch.zeros_like(q) if out is None else out, None, **kw)

    refused("CUDA device only")
    refused("q is", q=q.float())
    refused("q is", q=q[:1])
    refused("q is", q=torch.zeros(256, 2, dtype=torch.bfloat16).t())
    refused("out is", out=torch.zeros(2, 128))
    refused("int32", positions=positions.long())
    refused("for every row", positions=positions[:1])
    refused("for every row", table=table[:1])
    refused("kv_pool", pool=pool[:, :, :1])
    refused("kv_pool", pool=pool.float())
    refused("sink", sink_weight=torch.zeros(3))
    refused("not negative", most=-1)
    refused("not negative", softcap=-1.0)


@pytest.mark.parametrize("heads,hd,dtype,bq", [(64, 128, torch.float32, 2), (48, 64, torch.float32, 2), (64, 256, torch.float32, 1), (32, 256, torch.bfloat16, 1),
                                               (64, 80, torch.bfloat16, 2), (12, 256, torch.bfloat16, 2)])
@pytest.mark.parametrize("sizes", [(2,), (3, 3, 3), (4,), (5, 2, 3, 7), (3,) * 20, (1, 41), (2,) * 9])
def test_blocks_of_one_and_of_two_rows_have_room(heads, hd, dtype, bq, sizes):
    """Many query heads to a kv head: a block of the float units' kernels holds two rows, or one, which then has nobody to share with."""
    groups, at = [], 1
    for k in sizes:
        groups.append((range(at, at + k), 700))
        at += k
    for fixed in (False, True):
        plan = ops.shared_plan(SharedPrefix(at, groups), heads, 1, hd, dtype, split=64, device="cpu", fixed=fixed)
        assert (plan.kernel, plan.bq) == ("generic", bq) and plan.shares == (bq > 1)
        blocks = plan.items[plan.items[:, 2] > 0].tolist()
        assert sorted(r for b in blocks if b[4] == shared_plan.MOST for r in plan.rows[b[1]:b[1] + b[2]].tolist()) == list(range(at))
        together = [r for b in blocks if b[4] != shared_plan.MOST for r in plan.rows[b[1]:b[1] + b[2]].tolist()]
        assert sorted(together) == sorted(r for g, _ in groups if len(g) > 1 for r in g)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,hd,dtype", [(64, 128, torch.float32), (48, 64, torch.float32), (32, 256, torch.bfloat16)])
def test_shared_attention_of_many_heads_to_a_kv_head(nh, hd, dtype):
    groups = [([1, 2, 3], 200), ([4, 6, 8], 130), ([9, 7, 5], 500), ([10, 11, 12, 13], 64)]
    lengths = [70, 210, 201, 260, 131, 501, 150, 600, 140, 505, 65, 70, 128, 129]
    c = Case(groups, lengths, nh, 1, hd, 16, dtype, seed=nh)
    got, plan = c.run(prefer="generic", split=64)
    assert plan.shares == (dtype == torch.float32)
    assert torch.equal(got, c.alone(64))


def test_long_requests_beside_a_family_count():
    """Times measured with heads of 128 in pages of 64, microseconds with sharing and row by row: the choice is the faster one."""
    own, alone = (lambda streams, positions: ops.own_ranges(streams, positions, 148)), (lambda streams, positions: ops.decode_splits(streams, positions, 148))
    for rows, shared, own_each, lone, nkv, sharing, without in ((63, 8192, 200, [16384], 4, 249.4, 181.4), (63, 4096, 200, [32000], 4, 458.2, 272.8),
                                                                (60, 2048, 300, [4000, 8000, 16000, 32000], 4, 468.8, 260.0), (16, 8192, 200, [16384], 2, 45.9, 30.6),
                                                                (8, 4096, 200, [4000] * 8, 2, 21.4, 13.6), (32, 4096, 200, [4000] * 32, 4, 82.8, 73.5),
                                                                (63, 32000, 200, [32000], 4, 485.4, 468.9), (63, 8192, 200, [16384], 2, 95.3, 102.8),
                                                                (63, 4096, 200, [32000], 2, 164.2, 196.9), (63, 8192, 200, [200], 4, 29.4, 111.1),
                                                                (63, 8192, 3000, [16384], 2, 115.7, 129.2)):
        group = (tuple(range(rows)), shared)
        for front in (0, 1):                               # (lone requests first or last)
            n = rows + len(lone)
            group = (tuple(range(front * len(lone), front * len(lone) + rows)), shared)
            lengths = lone * front + [shared + own_each + 7 * i % 50 for i in range(rows)] + lone * (1 - front)
            kept = shared_plan.worth_sharing(SharedPrefix(n, [group], lengths), 6, nkv, 148, shared_plan.items_room(n, 6, nkv, 148), 64, own, alone, 512)
            assert kept == ([group] if sharing < without else []), (rows, shared, lone, nkv)
    with pytest.raises(ValueError, match="lengths"):
        SharedPrefix(3, [([0, 1], 64)], [1, 2])
    with pytest.raises(ValueError, match="lengths"):
        SharedPrefix(3, [([0, 1], 64)], [1, 2, -1])
    assert SharedPrefix(2, [([0, 1], 64)], [70, 80]) == SharedPrefix(2, [([0, 1], 64)])


@pytest.mark.parametrize("nh,nkv", [(12, 2), (28, 4), (64, 8), (16, 16), (7, 1)])
def test_a_captured_call_has_room_for_one_wave_of_ranges(nh, nkv):
    rng = np.random.default_rng(nh)
    sets = [_random_groups(rng) for _ in range(8)] + [SharedPrefix(90, [(range(90), 120000)]), SharedPrefix(90, [([0, 1], 60000), (range(2, 90), 64)])]
    for shared in sets:
        plan = ops.shared_plan(shared, nh, nkv, 128, torch.bfloat16, prefer="tc", device="cpu", fixed=True)
        items = plan.items[plan.items[:, 2] > 0]
        assert plan.slots <= min(64, -(-148 // nkv)) and (not len(items) or int(items[:, 5].max()) < plan.slots)
        assert int(plan.parts.max()) <= plan.slots
        for group, positions in shared.groups:
            assert sorted((a, b) for req, _, _, a, b, _, _, _ in items.tolist() if req == group[0] and a == 0)
            assert max(b for req, _, _, _, b, _, _, _ in items.tolist() if req == group[0]) == positions


def test_the_exponentials_of_the_float_units_are_as_near_as_is_said():
    """The polynomial in place of 2^f, evaluated in 64 bits from the numbers that the kernel holds: 2.7e-6 of it on [-1/2, 1/2]."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(ops.__file__), "attention_tcgen05.cu")).read()
    body = text[text.index("at_ex2_float2(unsigned long long x) {"):text.index("const unsigned long long two_n")]
    numbers = [float(a) for a, b in re.findall(r"pair2\((0\.\d+)f, (0\.\d+)f\)", body) if a == b]
    assert len(numbers) == 5
    f = np.linspace(-0.5, 0.5, 200001)
    worst = np.abs(np.polyval(np.asarray(numbers, dtype=np.float32).astype(np.float64), f) / np.exp2(f) - 1.0).max()
    assert worst <= 2.7e-6


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["two", "many", "long", "none"])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("sink", [False, True])
def test_a_row_that_is_no_number_shows_it(name, what, sink):
    """A query that is not a number, or infinite (its scores are then no numbers either): its row is no number, as without sharing, and the others are theirs."""
    c = Case(*SETS[name], 12, 2, 128, 64, torch.bfloat16, seed=2)
    c.q[1] = what
    weight = torch.linspace(-1, 2, 12) if sink else None
    rest = [r for r in range(len(c.lengths)) if r != 1]
    want, size = c.plain(weight)
    for most in (None, 20000):                             # (ranges of a row's own positions, and for rows that share nothing one kernel or two)
        got, _ = c.run(sink=weight, max_position=most)
        assert bool(torch.isnan(got[1].float()).all())
        assert bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16))[rest].all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_weights_of_nothing(hd):
    """Scores so far apart that all weights but one are nothing (below 2^-126 of the largest), among the shared positions and among a row's own."""
    c = Case(*SETS["many"], 12, 2, hd, 64, torch.bfloat16, seed=hd)
    for row, at in ((1, 17), (7, 999), (20, 1000), (30, c.lengths[30] - 1)):
        c.q[row] = (16.0 * c.keys[row][at].float().repeat_interleave(6, 0)).reshape(-1).to(torch.bfloat16)
    got, plan = c.run()
    want, size = c.plain()
    # (with hd features the largest score leads by more than 16 sqrt(hd) less the rest's spread, some 100 in base two: what is left of the others is nothing
    # beside the bound, and so is a score's own error)
    assert plan.n_items > 0 and bool(((got.double() - want).abs() <= bound(size, want, torch.bfloat16)).all())
