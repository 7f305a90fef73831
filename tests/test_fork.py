"""Requests that go on from another's text: the accounting of shared pages, families of completions in the scheduler, and the engine's results against those of
requests that each bring the whole text; and tokens chosen under rules."""
import importlib
import random

import numpy as np
import pytest
import torch

from beglin_b200.cache import CacheError, CacheManager, OutOfPages, PagePool, SharedPrefix
from beglin_b200.engine.scheduler import Request, Scheduler
from beglin_b200.parts.cache_need import FixedStateNeed, PagedKVNeed, PagedLatentNeed


# ------------------------------------------------------------------------------------------------ accounting (no GPU)
def test_a_page_is_free_when_its_last_holder_gives_it_back():
    p = PagePool(4)
    a, b = p.alloc(2)
    p.share([a])
    p.check()
    assert p.shared == 1 and p.holders(a) == 2
    p.free([a, b])
    p.check()
    assert p.num_free == 3 and p.shared == 0
    p.free([a])
    assert p.num_free == 4
    for pages in ([a], [9]):
        with pytest.raises(CacheError):
            p.share(pages)
        with pytest.raises(CacheError):
            p.free(pages)


def _hold(m, rid, length):
    if not m.has(rid):
        m.add_request(rid)
    m.reserve([(rid, length)])
    m.commit([(rid, length)])


def test_fork_shares_whole_pages_and_refuses_without_a_trace():
    m = CacheManager([PagedKVNeed(1, 8), None, FixedStateNeed((3,))], 4, 8, 4)
    _hold(m, "a", 10)
    table = list(m.kv_groups[0].tables["a"])
    m.fork("a", ["b", "c"])
    m.check()
    assert m.length("b") == m.length("c") == 10
    for r in "bc":
        assert m.kv_groups[0].tables[r][:2] == table[:2] and m.kv_groups[0].tables[r][2] not in table
    assert m.free_pages() == 8 - 3 - 2
    assert len({m.births[r] for r in "abc"}) == 3 and len({m.slots[r] for r in "abc"}) == 3
    before = (m.free_pages(), dict(m.lengths), {r: list(t) for r, t in m.kv_groups[0].tables.items()})
    for error, rid, new in ((CacheError, "x", ["d"]), (CacheError, "a", ["b"]), (CacheError, "a", ["d", "d"]), (CacheError, "a", ["d", "e"])):
        with pytest.raises(error):
            m.fork(rid, new)
    _hold(m, "a", 20)                                      # every page is held now
    assert m.free_pages() == 1
    m.release("c")
    _hold(m, "b", 17)
    assert m.free_pages() == 0
    with pytest.raises(OutOfPages):
        m.fork("b", ["d"])
    assert not m.has("d")
    m.check()
    m.release("b")
    _hold(m, "a", 20)
    m.fork("a", ["d"])                                     # a text that ends with its page needs none
    assert m.kv_groups[0].tables["d"] == m.kv_groups[0].tables["a"]
    m.check()
    m.release("a")
    m.check()
    assert m.pages_held("d") == 5
    m.release("d")
    assert m.free_pages() == 8 and before[0] == 3


@pytest.mark.parametrize("seed", range(8))
def test_random_forks_keep_the_books(seed):
    """Requests that grow, fork and end in any order, over groups with and without a window: no page is lost, and none is taken from a holder."""
    rng = random.Random(seed)
    m = CacheManager([PagedKVNeed(1, 8), PagedKVNeed(1, 8, window=7), PagedKVNeed(1, 8, block=10), PagedLatentNeed(5, window=6)], 4, 60, 9, max_context=80)
    live, n = [], 0
    for _ in range(400):
        what = rng.random()
        if what < 0.15 and m.can_add():
            m.add_request(n); live.append(n); n += 1
        elif what < 0.3 and live:
            new = list(range(n, n + rng.randint(1, 3)))
            parent = rng.choice(live)
            try:
                m.fork(parent, new)
                live += new
                n += len(new)
            except (CacheError, OutOfPages):
                assert not any(m.has(r) for r in new)
        elif what < 0.4 and live:
            m.release(live.pop(rng.randrange(len(live))))
        elif live:
            some = rng.sample(live, rng.randint(1, len(live)))
            plan = [(r, m.length(r) + rng.randint(1, 6)) for r in some]
            short = None if any(length > m.max_context for _, length in plan) else m.pages_short(plan)
            try:
                m.reserve(plan)
                assert short == 0
                if rng.random() < 0.2:
                    m.trim(some)
                else:
                    m.commit(plan)
            except OutOfPages:
                assert short > 0
            except CacheError as e:
                assert "context limit" in str(e)
        m.check()
        for g in m.kv_groups:                              # what a request writes next belongs to it alone
            for r in live:
                k = m.length(r) // 4
                if m.length(r) % 4 and k < len(g.tables[r]) and g.tables[r][k] >= 0:
                    assert g.pool.holders(g.tables[r][k]) == 1
    for r in live:
        m.release(r)
    m.check()
    assert all(g.pool.num_free == 60 for g in m.kv_groups)


def test_groups_of_rows_that_share_pages():
    m = CacheManager([PagedKVNeed(1, 8, window=5), PagedKVNeed(1, 8)], 4, 40, 8)
    assert m.shared_prefix([]) is None
    _hold(m, "a", 10); _hold(m, "z", 9)
    assert m.shared_prefix(["a", "z"]) is None
    m.fork("a", ["b"])
    _hold(m, "a", 23)
    m.fork("a", ["c"])
    assert m.shared_prefix(["a", "b"]) == SharedPrefix(2, [((0, 1), 8)])
    assert m.shared_prefix(["z", "c", "a"]) == SharedPrefix(3, [((1, 2), 20)])
    assert m.shared_prefix(["c", "z", "b", "a"]) == SharedPrefix(4, [((0, 2, 3), 8)])
    assert m.shared_prefix(["c", "z"]) is None
    assert CacheManager([PagedKVNeed(1, 8, window=5)], 4, 40, 8).shared_prefix(["a"]) is None


# ------------------------------------------------------------------------------------------------ families in the scheduler (no GPU)
def _drive(sched, check=None):
    """Run the schedule as the engine does, with tokens that count up; returns the steps."""
    steps = 0
    while True:
        plan = sched.plan()
        if plan is None:
            return steps
        steps += 1
        assert steps < 1000
        sched.cache.commit(plan.lengths)
        wanted = sched.wanted(plan)
        started = [r for lead in sched.leads(plan) for r in sched.adopt(lead)]
        sched.first_tokens(started, [100] * len(started))
        sched.update(plan, [100 + len(r.output) for r in wanted], committed=True)
        sched.cache.check()
        if check:
            check()


def _family(i, prompt, n, k, **kw):
    rs = [Request(rid=(i, j), prompt=list(range(prompt)), max_new_tokens=n, **kw) for j in range(k)]
    rs[0].siblings = rs[1:]
    return rs


@pytest.mark.parametrize("slots,pages,mixed", [(8, 60, True), (3, 60, True), (1, 60, True), (8, 9, True), (8, 60, False), (2, 7, False)])
def test_families_end_complete(slots, pages, mixed):
    m = CacheManager([PagedKVNeed(1, 8)], 4, pages, slots)
    sched = Scheduler(m, max_batch=slots, max_step_tokens=16, mixed=mixed)
    families = [_family(0, 10, 6, 4), _family(1, 8, 3, 1), _family(2, 13, 1, 3)]
    for f in families:
        sched.add(f[0])
    _drive(sched)
    for f, n in zip(families, (6, 3, 1)):
        assert [r.output for r in f] == [[100 + i for i in range(n)]] * len(f)
        assert all(r.finish_reason == "length" for r in f)
    assert not m.live() and m.free_pages() == pages
    assert len(sched.finished) == 8


def test_a_family_whose_lead_cannot_run_ends_with_it():
    m = CacheManager([PagedKVNeed(1, 8)], 4, 4, 4)
    sched = Scheduler(m, max_batch=4)
    long, big = _family(0, 16, 2, 3), _family(1, 15, 9, 2)
    sched.add(long[0]); sched.add(big[0])
    _drive(sched)
    assert [r.finish_reason for r in long] == ["context_limit"] * 3
    assert all(r.finish_reason in ("context_limit", "out_of_pages", "length") and r.phase == "done" for r in big)
    assert not m.live()


def test_a_prompt_goes_through_once():
    m = CacheManager([PagedKVNeed(1, 8)], 4, 60, 8)
    sched = Scheduler(m, max_batch=8)
    family = _family(0, 30, 5, 6)
    sched.add(family[0])
    _drive(sched)
    assert sched.counters.prefill_rows == 30 and sched.counters.decode_rows == 6 * 4


# ------------------------------------------------------------------------------------------------ rules (no GPU)
def test_rules_are_checked():
    from beglin_b200.sampling import LogitRules
    for bad, match in ((dict(repetition=0.0), "repetition"), (dict(repetition=float("inf")), "repetition"), (dict(frequency=float("nan")), "frequency"),
                       (dict(bias={10: 1.0}), "outside"), (dict(bias={-1: 1.0}), "outside"), (dict(bias={1: float("nan")}), "not a number"), (dict(bias={i: 1.0 for i in range(513)}), "at most")):
        with pytest.raises(ValueError, match=match):
            LogitRules(**bad).check(10)
    assert LogitRules().plain and not LogitRules(presence=0.1).plain
    mask = lambda allowed, vocab=70: LogitRules(allowed=lambda made: allowed).mask([], vocab)
    assert mask(None) is None and LogitRules().mask([], 70) is None
    words = mask([0, 31, 32, 69])
    assert words.dtype == np.int32 and words.view(np.uint32).tolist() == [1 | 1 << 31, 1, 1 << 5]
    truth = np.zeros(70, dtype=bool)
    truth[[0, 31, 32, 69]] = True
    assert mask(truth).tolist() == words.tolist()
    packed = words.view(np.uint32).copy()
    assert mask(packed).tolist() == words.tolist() and mask(np.stack([packed, packed], axis=1)[:, 0]).tolist() == words.tolist()
    assert mask(np.asarray([5], dtype=np.uint32), vocab=3).tolist() == [5] and mask(np.asarray([1 << 31], dtype=np.uint32), vocab=32) is not None
    for bad, match in (([70], "outside"), ([-1], "outside"), ([], "no token"), (np.zeros(70, dtype=bool), "no token"), (np.ones(5, dtype=bool), "truth values"),
                       (np.zeros(3, dtype=np.uint32), "no token"), (np.asarray([0, 0, 1 << 6], dtype=np.uint32), "no token"), (np.ones(2, dtype=np.uint32), "packed bits")):
        with pytest.raises(ValueError, match=match):
            mask(bad)


def test_tables_of_a_replayed_step_follow_the_rules():
    """What a replayed step's tables hold is loaded again when the rules change, when a step in between ran without them and when one was given up."""
    from types import SimpleNamespace
    from beglin_b200.engine.decode_graph import DecodeGraph
    from beglin_b200.sampling import LogitRules
    from beglin_b200.sampling.rules import RuleTables
    g = DecodeGraph.__new__(DecodeGraph)
    g.n, g._rules_of, g._rules_next, g.rules = 2, None, None, RuleTables(2, 50, 16, "cpu")
    g.engine, loads = SimpleNamespace(vocab=50), []
    load = g.rules.load
    g.rules.load = lambda rows: loads.append(1) or load(rows)

    def step(rules, made, at, runs=True):
        variant = g._load_rules(("a",), [at], None if rules is None else [(rules, [1, 2], made)])[0]
        if runs:
            g._rules_of = g._rules_next
        return variant, len(loads)

    first, second = LogitRules(bias={3: 1.0}), LogitRules(bias={3: -1.0})
    assert step(first, [4], 2) == ("rules", 1)
    assert step(first, [4, 5], 3) == ("rules", 1)                      # nothing new
    assert step(LogitRules(bias={3: 1.0}), [4, 5, 6], 4) == ("rules", 1)
    assert step(second, [4, 5, 6, 7], 5) == ("rules", 2) and float(g.rules.bias_values[0]) == -1.0
    assert step(None, [], 6) == ("", 2) and step(second, [4, 5, 6, 7, 8, 9], 7) == ("rules", 3)
    assert step(second, [4, 5, 6, 7, 8, 9, 9], 8, runs=False) == ("rules", 3) and step(second, [4, 5, 6, 7, 8, 9, 9], 8) == ("rules", 4)
    assert step(second, [4], 9) == ("rules", 4)                        # the device keeps count
    never = LogitRules(allowed=lambda made: [])
    with pytest.raises(ValueError, match="no token"):
        step(never, [4, 5, 6, 7, 8, 9, 9, 9, 9], 10)
    assert g._rules_of is None
    for rules, made, at in ((first, [4], 10), (LogitRules(allowed=lambda made: [1]), [4], 3), (LogitRules(bias={50: 1.0}), [4], 2)):
        with pytest.raises(ValueError, match="position|outside"):
            step(rules, made, at)
    with pytest.raises(ValueError, match="rules for"):
        g._load_rules(("a", "b"), [2, 2], [(first, [1, 2], [4])])
    given = {3: 1.0}
    kept = LogitRules(bias=given)
    given[3] = 2.0
    assert kept.bias == {3: 1.0}


# ------------------------------------------------------------------------------------------------ the engine
DESIGNS = {"qwen2": ("helpers", "D"), "qwen2 window": ("helpers", "C"), "sukisun": ("sukisun_helpers", None), "nadilorn": ("nadilorn_helpers", None),
           "sofudra": ("sofudra_helpers", None), "tuzupel": ("tuzupel_helpers", None), "dinatar": ("dinatar_helpers", None), "fanitar": ("fanitar_helpers", None)}


def _folder(root, design, dtype):
    module, name = DESIGNS[design]
    h = importlib.import_module(module)
    name = name or sorted(h.CONFIGS)[0]
    return h.make_model(root, name, seed=5, dtype=dtype), (h.TINY if module == "helpers" else h.CONFIGS)[name][2 if module == "helpers" else 1]


def _engine(folder, dtype, page, **kw):
    from beglin_b200 import Engine
    eng = Engine.from_folder(folder, dtype=dtype, max_tokens=kw.pop("max_tokens", 4096), page_size=page, max_requests=kw.pop("max_requests", 12), kv_split=64, **kw)
    for g in eng.cache.kv_groups:                          # what nobody has written poisons who reads it
        g.device_pool.fill_(float("nan"))
        g.device_pool[:, eng.cache.dump_page].zero_()
    for g in eng.cache.state_groups:
        g.slab.fill_(float("nan"))
        g.slab[:, eng.cache.dump_slot].zero_()
    return eng


def _ids(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design", DESIGNS)
def test_forked_requests_are_those_that_bring_the_text(model_root, design, dtype, graph):
    """Forks of a text that ends inside a page and of one that ends with it, forks of forks, the first request ended: every later token's row against that of a
    request that went through the same text by itself, in float32 bit for bit."""
    folder, page = _folder(model_root, design, torch.float32 if dtype == "float32" else torch.bfloat16)
    eng = _engine(folder, dtype, page)
    text, more = _ids(4 * page + 3, eng.vocab, 1), _ids(200, eng.vocab, 2)
    names = ["a", "b", "c", "d", "e", "f"]
    step = {}

    def bring(rid, tokens):                                # (the same portions for both kinds)
        for at in range(0, len(tokens), 3 * page):
            eng.step([(rid, tokens[at:at + 3 * page], [])])

    def single(rids, tokens):
        if not graph:
            return eng.step([(r, [t], [0]) for r, t in zip(rids, tokens)])
        eng.decode(rids, tokens)
        return eng.decode_graph(len(rids)).logits[:len(rids)].clone()

    def both(pairs):
        rows = single([p[0] for p in pairs], [p[2] for p in pairs])
        want = single([p[1] for p in pairs], [p[2] for p in pairs])
        if dtype == "float32":
            assert torch.equal(rows, want)
        else:
            assert float((rows - want).abs().max()) <= 2e-2 * float(want.abs().max())
        assert torch.isfinite(rows).all()

    bring("a", text)
    eng.fork("a", ["b", "c"])
    for r in "ABC":
        bring(r, text)
    it = iter(more)
    for _ in range(page - 1):                              # on to the end of a page
        both([(r, r.upper(), next(it)) for r in "abc"])
    while eng.cache.length("a") % page:
        both([(r, r.upper(), next(it)) for r in "abc"])
    eng.cache.check()
    history = {}
    eng.fork("b", ["d"])                                   # ends with its page
    eng.release("a"); eng.release("A")
    history["D"] = None
    eng.fork("B", ["D"])                                   # (its pages were brought by B itself)
    for _ in range(page + 2):
        both([(r, r.upper(), next(it)) for r in "bcd"])
    assert eng.cache.shared_prefix(["b", "c", "d"]) is not None or not any(not g.gives_back for g in eng.cache.kv_groups)
    for r in "bcdBCD":
        eng.release(r)
    eng.cache.check()
    assert eng.cache.free_pages() == eng.cache.num_pages


WIDE = {"architectures": ["Qwen2ForCausalLM"], "model_type": "qwen2", "num_hidden_layers": 2, "hidden_size": 768, "num_attention_heads": 12, "num_key_value_heads": 2,
        "head_dim": 128, "intermediate_size": 512, "vocab_size": 500, "rope_theta": 1000000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True,
        "use_sliding_window": False, "max_position_embeddings": 32768}


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_many_forks_of_a_long_text_read_it_once(model_root, graph, monkeypatch):
    """The benchmark's heads: the tensor-core kernel of shared positions runs, and rows agree with those of the attention that shares nothing."""
    from helpers import make_model
    from beglin_b200.csrc import ops
    eng = _engine(make_model(model_root, "wide", config=WIDE), "bfloat16", 64, max_tokens=16384, max_requests=40)
    for at, part in enumerate((_ids(2048, 500, 1), _ids(2000, 500, 2))):
        eng.step([(0, part, [])])
    eng.fork(0, list(range(1, 40)))
    plans = []
    real = ops.shared_plan
    monkeypatch.setattr(ops, "shared_plan", lambda *a, **kw: plans.append(real(*a, **kw)) or plans[-1])
    tokens = [_ids(40, 500, 10 + i) for i in range(5)]

    def run():
        out = []
        for t in tokens:
            if graph:
                eng.decode(list(range(40)), t)
                out.append(eng.decode_graph(40).logits[:40].clone())
            else:
                out.append(eng.step([(r, [v], [0]) for r, v in enumerate(t)]))
        return out

    got = run()
    assert plans and all(p.kernel == "tc" and p.shares for p in plans) and len(plans) == (1 if graph else 5)
    # the same from the same lengths without groups
    eng.cache.lengths.update({r: eng.cache.length(r) - 5 for r in range(40)})
    eng.cache.trim(list(range(40)))
    monkeypatch.setattr(type(eng.cache), "shared_prefix", lambda self, rids: None)
    eng._graphs.clear()
    for a, b in zip(got, run()):
        # both round weights to bfloat16 once a layer: half a step of 2^-8 of a row's attention each, which the tests of whole models allow 2e-2 of the
        # largest logit for
        assert float((a - b).abs().max()) <= 2e-2 * float(b.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("design", ["qwen2", "sofudra", "sukisun"])
def test_completions(model_root, design):
    """In float32 a request's tokens do not depend on who else is in the batch: completions are the same with few slots and many, on few pages and many,
    the first is the only one's, and greedy ones are all alike."""
    folder, page = _folder(model_root, design, torch.float32)
    prompts = [_ids(2 * page + 5, 150, 3), _ids(7, 150, 4), _ids(3 * page, 150, 5)]
    kw = dict(max_new_tokens=9, stop_ids=(), seed=4)
    many = _engine(folder, "float32", page)
    one = many.generate(prompts, temperature=0.9, **kw)
    got = many.generate(prompts, temperature=0.9, completions=4, **kw)
    assert [len(c) for c in got] == [4, 4, 4] and all(len(t) == 9 for c in got for t in c)
    assert [c[0] for c in got] == one
    if design == "qwen2":                                  # (a decisive model draws the same token at any number)
        assert any(len(set(map(tuple, c))) > 1 for c in got)
    assert many.cache.free_pages() == many.cache.num_pages
    few = _engine(folder, "float32", page, max_requests=3, max_tokens=10 * page)
    assert few.generate(prompts, temperature=0.9, completions=4, **kw) == got
    plain = _engine(folder, "float32", page, use_graphs=False)
    assert plain.generate(prompts, temperature=0.9, completions=4, **kw) == got
    greedy = many.generate(prompts, completions=3, **kw)
    assert all(c == [c[0]] * 3 for c in greedy) and [c[0] for c in greedy] == many.generate(prompts, **kw)
    assert many.generate(prompts[:1], completions=2, max_new_tokens=1, stop_ids=()) == [[greedy[0][0][:1]] * 2]
    with pytest.raises(ValueError, match="completions"):
        many.generate(prompts, completions=0)


def _ruled(row, rules, prompt, made):
    x = row.double().cpu()
    for t in set(prompt) | set(made):
        x[t] = x[t] / rules.repetition if x[t] > 0 else x[t] * rules.repetition
    for t in set(made):
        x[t] -= rules.frequency * made.count(t) + rules.presence
    for t, b in rules.bias.items():
        x[t] += b
    if rules.allowed is not None:
        left = rules.allowed(made)
        if left is not None:
            out = torch.full_like(x, -float("inf"))
            out[left] = x[left]
            x = out
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_generation_under_rules(model_root, graphs):
    """Greedy tokens under rules against the rules applied in 64 bits to the step function's logits: the chosen token's value lies within a rounding of the
    largest, and is the largest where that is clear."""
    from beglin_b200 import LogitRules
    folder, page = _folder(model_root, "qwen2", torch.float32)
    eng = _engine(folder, "float32", page, use_graphs=graphs)
    prompts = [_ids(20, 200, 1), _ids(3, 200, 2), _ids(40, 200, 3)]
    small = LogitRules(repetition=1.3, frequency=0.2, presence=0.1, bias={7: 0.5, 9: -2.0, 199: 0.25})
    grammar = LogitRules(allowed=lambda made: list(range(50, 60)) if len(made) % 3 else None, repetition=0.9)
    rules = [small, grammar, None]
    out = eng.generate(prompts, max_new_tokens=12, stop_ids=(), rules=rules)
    again = eng.generate(prompts, max_new_tokens=12, stop_ids=(), rules=rules, max_step_tokens=8)
    assert out == again
    assert out[2] == eng.generate(prompts[2:], max_new_tokens=12, stop_ids=())[0]
    assert all(50 <= t < 60 for i, t in enumerate(out[1]) if i % 3)
    assert out[0] != eng.generate(prompts[:1], max_new_tokens=12, stop_ids=())[0]
    for prompt, made, r in zip(prompts[:2], out, rules):
        rows = eng.step([("x", prompt + made, list(range(len(prompt) - 1, len(prompt) + 11)))], end=["x"])
        for i, t in enumerate(made):
            x = _ruled(rows[i], r, prompt, made[:i])
            slack = 1e-5 * float(x[x > -float("inf")].abs().max())
            assert float(x.max() - x[t]) <= slack
            if float((x.max() - x.topk(2).values[1])) > slack:
                assert t == int(x.argmax())
    # a family under rules, in one batch with a request without
    both = eng.generate(prompts, max_new_tokens=12, stop_ids=(), rules=rules, completions=2)
    assert [c[0] for c in both] == out and [c[1] for c in both] == out
    with pytest.raises(ValueError, match="rules for"):
        eng.generate(prompts, rules=[small])
    with pytest.raises(ValueError, match="outside"):
        eng.generate(prompts, rules=LogitRules(bias={200: 1.0}))


@pytest.mark.gpu
def test_a_prompts_last_token_fed_by_a_decoding_step_is_the_prompts(model_root):
    """A request whose prompt is in the cache but for its last token, which the first decoding step under rules brings: that token is no generated one."""
    from beglin_b200 import LogitRules
    folder, page = _folder(model_root, "qwen2", torch.float32)
    eng = _engine(folder, "float32", page)
    prompt, rules = _ids(20, 200, 1), LogitRules(frequency=3.0, presence=2.0, repetition=1.2)
    for rid in "ab":
        eng.step([(rid, prompt[:-1], [])])
    made, row = [], eng.step([("a", prompt[-1:], [0])])[0]
    for _ in range(3):
        made += eng.decode(["b"], prompt[-1:] if not made else made[-1:], rules=[(rules, prompt, list(made))])
        got, want = eng.decode_graph(1).logits[0].double().cpu(), _ruled(row, rules, prompt, made[:-1])
        # the two step functions' rows agree in float32 to rounding, and three roundings more come with the rules
        assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())
        row = eng.step([("a", made[-1:], [0])])[0]


@pytest.mark.gpu
def test_a_step_that_was_given_up_leaves_nothing_for_the_next(model_root):
    """A decoding step that its rules end when its positions have gone to the device; later another step's positions are those that the last whole step
    left, in a page that has become another request's too."""
    from beglin_b200 import LogitRules
    folder, page = _folder(model_root, "qwen2", torch.float32)
    eng = _engine(folder, "float32", page)
    text, never, at = _ids(4 * page, 200, 1), LogitRules(allowed=lambda made: []), 2 * page - 4
    eng.step([("a", text[:at + 5], []), ("b", text[:at], []), ("c", text[:at], [])])
    eng.decode(["a"], text[:1])                            # on to position at + 6
    with pytest.raises(ValueError, match="no token"):
        eng.decode(["b"], text[at:at + 1], rules=[(never, text[:at], text[at:at + 1])])
    eng.step([("b", text[at:at + 6], []), ("c", text[at:at + 6], [])])
    eng.fork("b", ["d"])
    rows = {rid: [] for rid in "bcd"}
    for rid in "bcd":
        for t in text[at + 6:at + 9]:
            eng.decode([rid], [t])
            rows[rid].append(eng.decode_graph(1).logits[0].clone())
    for rid in "bd":
        assert all(torch.equal(x, y) for x, y in zip(rows[rid], rows["c"]))


@pytest.mark.gpu
def test_pages_that_were_made_ready_are_asked_for_again_after_a_step_that_was_given_up(model_root, monkeypatch):
    """A step that ends between the upload of its block tables and its replay (a capture that fails): the tables of the step before are not the device's any more."""
    from beglin_b200 import LogitRules
    folder, page = _folder(model_root, "qwen2", torch.float32)
    eng = _engine(folder, "float32", page)
    text = _ids(40, 200, 1)
    for rid in "ac":
        eng.step([(rid, text[:page + 3], [])])
    eng.step([("b", _ids(page + 3, 200, 2), [])])
    eng.decode(["c"], text[page + 3:page + 4])
    eng.decode(["c"], text[page + 4:page + 5])
    want = eng.decode_graph(1).logits[0].clone()
    eng.decode(["a"], text[page + 3:page + 4])
    graph = eng.decode_graph(1)
    with monkeypatch.context() as m:
        m.setattr(graph, "_capture", lambda *which: (_ for _ in ()).throw(RuntimeError("no room")))
        with pytest.raises(RuntimeError, match="no room"):
            eng.decode(["b"], [1], rules=[(LogitRules(bias={1: 1.0}), [0] * (page + 3), [1])])
    eng.decode(["a"], text[page + 4:page + 5])
    assert torch.equal(graph.logits[0], want)


@pytest.mark.gpu
def test_a_page_made_ready_and_given_back_is_asked_for_again(model_root, monkeypatch):
    """A decoding step makes room for its next one; a portion of the same request that fails gives that page back, and another request takes it."""
    folder, page = _folder(model_root, "qwen2", torch.float32)
    eng = _engine(folder, "float32", page)
    text, other = _ids(4 * page, 200, 1), _ids(2 * page + 1, 200, 2)
    eng.step([("a", text[:2 * page - 1], [])])
    eng.decode(["a"], text[2 * page - 1:2 * page])         # the next position begins a page
    with monkeypatch.context() as m:
        m.setattr(eng.model, "forward", lambda *a: (_ for _ in ()).throw(RuntimeError("no room")))
        with pytest.raises(RuntimeError, match="no room"):
            eng.step([("a", text[2 * page:2 * page + 3], [])])
    eng.step([("b", other[:-1], [])])
    got = []
    for t in text[2 * page:2 * page + 4]:
        eng.decode(["a"], [t])
        got.append(eng.decode_graph(1).logits[0].clone())
    eng.cache.check()
    eng.step([("c", text[:2 * page], []), ("d", other[:-1], [])])
    for t, row in zip(text[2 * page:], got):
        eng.decode(["c"], [t])
        assert torch.equal(eng.decode_graph(1).logits[0], row)
    rows = eng.step([("b", other[-1:], [0]), ("d", other[-1:], [0])])
    assert torch.equal(rows[0], rows[1])


def test_groups_know_their_requests_lengths():
    m = CacheManager([PagedKVNeed(1, 8)], 4, 40, 8)
    _hold(m, "a", 10); _hold(m, "z", 33)
    m.fork("a", ["b"])
    _hold(m, "b", 15)
    assert m.shared_prefix(["b", "z", "a"]).lengths == (15, 33, 10)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_long_request_beside_a_family_is_not_left_to_one_block(model_root, graph, monkeypatch):
    """A family beside a request that is much longer goes row by row, and in a captured step by the same graph, until it ends; then its pages are read once."""
    from helpers import make_model
    from beglin_b200.csrc import ops
    eng = _engine(make_model(model_root, "wide", config=WIDE), "bfloat16", 64, max_tokens=32768, max_requests=40)
    for part in range(4):
        eng.step([("family", _ids(2048, 500, part), [])])
    eng.fork("family", list(range(30)))
    for part in range(9):
        eng.step([("long", _ids(2048, 500, part), [])])
    real, calls = ops.shared_attention, []
    monkeypatch.setattr(ops, "shared_attention", lambda *a, **kw: calls.append(1) or real(*a, **kw))

    def step(rids):
        calls.clear()
        if graph:
            g = eng.decode_graph(len(rids))
            eng.decode(rids, [3] * len(rids))
            return g._shares
        eng.step([(r, [3], [0]) for r in rids])
        return bool(calls)

    family = list(range(30)) + ["family"]
    if graph:
        step(family + ["long"])                            # (the first step of forked requests makes the plans, which answer from then on)
    assert not step(family + ["long"])
    assert step(family)


@pytest.mark.gpu
def test_whether_sharing_pays_is_asked_again_as_requests_grow(model_root, monkeypatch):
    from helpers import make_model
    from beglin_b200.csrc import shared_plan
    from beglin_b200.engine.decode_graph import DecodeGraph
    eng = _engine(make_model(model_root, "wide", config=WIDE), "bfloat16", 64, max_tokens=8192, max_requests=8)
    eng.step([("a", _ids(200, 500, 1), [])])
    eng.fork("a", ["b", "c"])
    asked = []
    monkeypatch.setattr(shared_plan, "worth_sharing", lambda shared, *a: asked.append(shared.lengths) or (shared.groups if shared.lengths[0] < 205 else []))
    monkeypatch.setattr(DecodeGraph, "REGROUP", 4)
    eng.decode(["a", "b", "c"], [1, 2, 3])                 # positions 200 .. 202 with sharing, to be asked again at 204
    g = eng.decode_graph(3)
    assert asked == [(200, 200, 200, 0)] and g._shares
    for i in range(12):
        eng.decode(["a", "b", "c"], [1, 2, 3])
        assert g._shares == (eng.cache.length("a") <= 208)
    assert asked == [(n, n, n, 0) for n in (200, 204, 208, 212)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["latent", "pages of 48"])
def test_models_that_do_not_read_shared_positions_keep_one_graph(model_root, kind):
    """Where no layer reads shared positions, or only by a kernel that its own is ahead of, forked requests go through the graph that every step goes through."""
    from helpers import make_model
    if kind == "latent":
        import sukisun_helpers
        page, dtype, folder = 16, "float32", sukisun_helpers.make_model(model_root, "sharp", seed=5)
    else:                                                  # (a size that the tensor-core kernel of shared positions does not take)
        page, dtype, folder = 48, "bfloat16", make_model(model_root, "wide", config=WIDE)
    eng = _engine(folder, dtype, page)
    text = _ids(3 * page + 2, 150, 1)
    eng.step([("a", text, []), ("x", text[:5], []), ("y", text[:9], [])])
    eng.decode(["x", "y"], [1, 2])
    eng.fork("a", ["b"])
    for _ in range(2):
        eng.decode(["a", "b"], [1, 2])
    assert len(eng.decode_graph(2).graphs) == 1


@pytest.mark.parametrize("text", [([3, 50], []), ([3], [4, -1]), ([2 ** 33], [1])])
def test_a_text_with_a_token_outside_the_vocabulary_is_refused(text):
    """The host has the texts: what the kernel would pass over and record is refused before it goes to the device."""
    from beglin_b200.sampling import LogitRules
    from beglin_b200.sampling.rules import RuleTables
    tables = RuleTables(2, 50, 8, "cpu")
    before = tables.history.clone()
    with pytest.raises(ValueError, match="outside the vocabulary"):
        tables.load([(None, [1], []), (LogitRules(presence=1.0),) + text])
    assert torch.equal(tables.history, before)
    tables.load([(None, [1], []), (LogitRules(presence=1.0), [49], [0])])
    assert tables.history[1, :2].tolist() == [49, 0]


@pytest.mark.gpu
def test_what_is_recorded_under_rules_reaches_the_caller(monkeypatch):
    from beglin_b200.csrc import ops
    from beglin_b200.sampling import LogitRules, Sampler
    from beglin_b200.sampling.rules import RuleTables
    status = ops.new_status("cuda:0")
    sampler, rules = Sampler("cuda:0", status), LogitRules(presence=1.0)
    logits = torch.arange(100, dtype=torch.float32, device="cuda:0").repeat(2, 1)
    assert sampler.sample(logits.clone(), [0.0, 0.0], [0.0, 0.0], [(rules, [3], [99]), (None, [3], [99])]) == [98, 99]
    ops.raise_on_status(status)
    monkeypatch.setattr(RuleTables, "load", lambda self, rows: (self.history.fill_(100), self.penalties.fill_(2.0)))
    sampler.sample(logits.clone(), [0.0, 0.0], [0.0, 0.0], [(rules, [3], [99]), (None, [3], [99])])
    with pytest.raises(ops.KernelError, match="token id"):
        ops.raise_on_status(status)
    with pytest.raises(ops.KernelError, match="token id"):
        Sampler("cuda:0").sample(logits.clone(), [0.0, 0.0], [0.0, 0.0], [(rules, [3], [99]), (None, [3], [99])])


def test_the_biases_of_rules_stay_as_they_are():
    """Replayed steps keep the tables of rules that they know: rules do not change behind them."""
    import copy
    import pickle
    from beglin_b200.sampling import LogitRules
    rules = LogitRules(bias={3: 1.0})
    for change in (lambda b: b.update({3: 2.0}), lambda b: b.__setitem__(4, 1.0), lambda b: b.pop(3), lambda b: b.clear(), lambda b: b.popitem(), lambda b: b.setdefault(5, 1.0),
                   lambda b: b.__delitem__(3), lambda b: b.__ior__({5: 1.0})):
        with pytest.raises(TypeError, match="stay"):
            change(rules.bias)
    for same in (copy.copy(rules), copy.deepcopy(rules), pickle.loads(pickle.dumps(rules))):
        assert same == rules == LogitRules(bias={3: 1.0}) and same.bias == {3: 1.0}
    assert {**rules.bias, 4: 1.0} == {3: 1.0, 4: 1.0} and LogitRules(bias=rules.bias) == rules


def test_ids_of_a_mask_are_whole_numbers():
    from beglin_b200.sampling import LogitRules
    for bad in ([1.5], [3.0], ["5"], [2 ** 70], np.asarray([1.0, 2.0])):
        with pytest.raises(ValueError, match="whole numbers"):
            LogitRules(allowed=lambda made: bad).mask([], 70)
    assert LogitRules(allowed=lambda made: np.asarray([5], dtype=np.int16)).mask([], 70).tolist() == [32, 0, 0]


@pytest.mark.parametrize("slots,completions,runs", [(3, 9, 3), (8, 16, 2), (1, 4, 4), (4, 5, 2)])
def test_what_is_left_of_a_family_is_one(slots, completions, runs):
    """Completions that find no slot bring the prompt again for as many of them as find one then, not each for itself."""
    m = CacheManager([PagedKVNeed(1, 8)], 4, 200, slots)
    sched = Scheduler(m, max_batch=slots)
    family = _family(0, 30, 5, completions)
    sched.add(family[0])
    _drive(sched)
    assert sched.counters.prefill_rows == 30 * runs
    assert [r.output for r in family] == [[100 + i for i in range(5)]] * completions and len(sched.finished) == completions


@pytest.mark.parametrize("needs", [[PagedKVNeed(1, 8)], [PagedKVNeed(1, 8), FixedStateNeed((3,))], [FixedStateNeed((3,))]])
def test_a_fork_whose_copies_cannot_be_made_leaves_no_request(needs):
    from beglin_b200.csrc import ops
    m = CacheManager(needs, 4, 8, 4)
    m.allocate("cpu", torch.float32)                       # (the kernel copies on a device only)
    _hold(m, "a", 10)
    before = (m.free_pages(), list(m._free_slots))
    with pytest.raises(ops.KernelError, match="CUDA device only"):
        m.fork("a", ["b", "c"])
    assert m.live() == ["a"] and m.free_pages() == before[0] and sorted(m._free_slots) == sorted(before[1])
    m.check()
