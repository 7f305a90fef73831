"""Tokens over chosen pages of a cache in 4 bits do not hang on who shares a step or on how prompts are cut: those that are decoded read chosen pages, those of a
prompt all of it."""
import pytest
import torch

from helpers import make_model, rel_err, seeded_ids
from test_packed_engine import GPU, WIDE, engine

from beglin_b200.cache import CacheManager
from beglin_b200.csrc import ops
from beglin_b200.engine.batch import Entry, StepBatch
from beglin_b200.engine.engine import check_packed
from beglin_b200.engine.scheduler import Request, Scheduler
from beglin_b200.parts.cache_need import CompositeNeed, PagedPackedNeed
from beglin_b200.parts.context import BuildContext


def test_entries_say_whether_they_are_of_a_prompt():
    cache = CacheManager([PagedPackedNeed(2, 64)], 16, 40, 4, 200)
    s = Scheduler(cache, max_step_tokens=6)
    for rid, n in (("a", 5), ("b", 7)):
        s.add(Request(rid=rid, prompt=list(range(n)), max_new_tokens=3))
    seen = []
    while (plan := s.plan()) is not None:
        seen.append([(e.rid, len(e.tokens), e.prompt) for e in plan.entries])
        s.update(plan, [1] * len(s.wanted(plan)))
    assert seen == [[("a", 5, True), ("b", 1, True)], [("a", 1, False), ("b", 5, True)], [("a", 1, False), ("b", 1, True)], [("b", 1, False)], [("b", 1, False)]]
    batch = StepBatch([Entry("a", [1]), Entry("b", [1], prompt=True), Entry("c", [1, 2]), Entry("d", [3, 4], prompt=True)], [5, 6, 7, 8], "cpu")
    assert batch.decoding == [True, False, False, False] and not batch.decode_only
    plan = batch.packed_plan(4, 2, 64, torch.bfloat16, 16, choose=True)
    assert plan.chosen.tolist() == [0, 0, 1] and plan.n_short and batch.packed_plan(4, 2, 64, torch.bfloat16, 16).n_chosen == 0


@GPU
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-5), ("bfloat16", 2e-2)])
def test_a_decoded_token_reads_the_same_pages_whoever_shares_its_step(model_root, dtype, tol):
    folder = make_model(model_root, "packedW", config=WIDE, std=0.05, bias_std=0.05)
    ids, other = seeded_ids(700, 200, 3), seeded_ids(200, 200, 4)
    every, alone, beside = (engine(folder, dtype, sparse_pages=n) for n in (0, 6, 6))
    for eng in (every, alone, beside):
        eng.step([("a", ids[:600], []), ("b", ids[:500], [])])
    for i, n in enumerate((1, 3, 100, 40)):
        tokens = lambda entries: [(rid, ids[at + i:at + i + 1], [0]) for rid, at in entries]
        full, want = (eng.step(tokens((("a", 600), ("b", 500)))) for eng in (every, alone))
        portion = Entry("c", other[i:i + n] if n > 1 else other[:1], [], prompt=True)
        got = beside.step(tokens((("a", 600),)) + [portion] + tokens((("b", 500),)))
        assert rel_err(got, want) < tol, (i, n)
        assert dtype == "bfloat16" or rel_err(want, full) > 100 * tol          # (which differ from those over all pages)


@GPU
def test_a_prompts_single_token_reads_all_of_it(model_root):
    folder = make_model(model_root, "packedW", config=WIDE, std=0.05, bias_std=0.05)
    ids = seeded_ids(700, 200, 3)
    every, some, mixed = (engine(folder, "float32", sparse_pages=n, portion_graph_rows=1) for n in (0, 6, 6))
    for eng in (every, some, mixed):
        eng.step([("a", ids[:600], []), ("b", ids[:500], [])])
    for i in range(600, 603):
        want = every.step([("a", ids[i:i + 1], [0])])
        assert rel_err(some.step([{"id": "a", "tokens": ids[i:i + 1], "want": [0], "prompt": True}]), want) < 1e-5
        got = mixed.step([("b", ids[i - 100:i - 99], [0]), Entry("a", ids[i:i + 1], [0], prompt=True)])
        assert rel_err(got[1:], want) < 1e-5
    want, got = every.step([("a", ids[603:604], [0])]), some.step([("a", ids[603:604], [0])])
    assert rel_err(got, want) > 1e-3


@GPU
def test_both_orders_of_prompts_give_the_same_tokens(model_root):
    folder = make_model(model_root, "packedW", config=WIDE, std=0.05, bias_std=0.05)
    prompts = [seeded_ids(n, 200, n) for n in (300, 1, 257, 129, 65)]
    made = []
    for graphs in (False, True):
        for mixed in (True, False):
            for budget in (64, 2048):
                eng = engine(folder, "float32", sparse_pages=4, use_graphs=graphs)
                made.append(eng.generate(prompts, max_new_tokens=24, temperature=1.0, seed=5, stop_ids=(), mixed=mixed, max_step_tokens=budget))
    assert all(m == made[0] for m in made)


# ------------------------------------------------------------------------------------------------ more pages than can be chosen of
def test_a_context_of_more_pages_than_can_be_chosen_of_is_refused():
    most, ctx = ops.packed_select_most(), lambda **kw: BuildContext(torch.device("cpu"), torch.bfloat16, page_size=16, cache_bits=4, **kw)
    bounded, plain = CompositeNeed((PagedPackedNeed(2, 64, None, True),)), PagedPackedNeed(2, 64)
    check_packed([plain, bounded], ctx(sparse_pages=8), 16 * most)
    check_packed([plain], ctx(sparse_pages=8), 16 * most + 1)                  # (a layer with a window has all of it read)
    check_packed([bounded], ctx(sparse_pages=most + 1), 16 * most + 1)         # (never are pages chosen)
    with pytest.raises(ValueError, match=f"sparse_pages=8.*{16 * most + 1}.*{most}"):
        check_packed([plain, bounded], ctx(sparse_pages=8), 16 * most + 1)


@GPU
def test_an_engine_of_such_a_context_is_not_built(model_root):
    folder = make_model(model_root, "packedFar", config=dict(WIDE, max_position_embeddings=1 << 20), std=0.05, bias_std=0.05)
    with pytest.raises(ValueError, match="sparse_pages=6"):
        engine(folder, "bfloat16", sparse_pages=6, max_context=16 * 36000 + 1)
    eng = engine(folder, "bfloat16", sparse_pages=6, max_context=16 * 36000)
    assert len(eng.generate([seeded_ids(200, 200, 1)], max_new_tokens=4, stop_ids=())[0]) == 4
