"""The engine over a cache in 4 bits: its logits against the plain implementation whose keys and values are rounded as such a cache holds them, replayed steps,
requests that go on from another's text, single tokens that read chosen pages, and what is refused."""
import os
import subprocess
import sys

import pytest
import torch

import helpers
from helpers import TINY_A, TINY_D, make_model, plain, rel_err, seeded_ids
from test_packed import quantised

from beglin_b200.cache import CacheManager
from beglin_b200.csrc import ops
from beglin_b200.parts.cache_need import PagedKVNeed, PagedPackedNeed
from beglin_b200.parts.context import BuildContext

GPU = pytest.mark.gpu
WIDE = dict(TINY_D, head_dim=128, num_attention_heads=4, num_key_value_heads=1, use_sliding_window=False)


def held(x):
    u, step, lowest = quantised(x.double().cpu())
    return (lowest + step * u).to(x.dtype)


def oracle(folder, ids):
    """Logits [T, vocab] in 64 bits with keys and values as the cache holds them."""
    cfg, w = helpers.plain_model(folder)
    plainly = plain.attention_fast
    plain.attention_fast = lambda q, k, v, group, window=None: plainly(q, held(k), held(v), group, window)
    try:
        return plain.forward(cfg, w, list(ids))
    finally:
        plain.attention_fast = plainly


# ------------------------------------------------------------------------------------------------ on the host
def test_a_need_of_bytes():
    need = PagedPackedNeed(2, 128, bounds=True)
    assert need.page_shape(64) == (2, 64 * 144 + 512) and need == PagedPackedNeed(2, 128, None, True) != PagedPackedNeed(2, 128)
    m = CacheManager([need, PagedKVNeed(2, 128), need, PagedPackedNeed(2, 128, 100)], 64, 5, 2)
    m.allocate("cpu", torch.float32)
    pools = [g.device_pool for g in m.kv_groups]
    assert [p.dtype for p in pools] == [torch.uint8, torch.float32, torch.uint8] and tuple(pools[0].shape) == (2, 6, 2, 64 * 144 + 512)
    part, = need.page_parts(pools[0], 64)
    assert tuple(part.shape) == (2, 6, 1, 1, 2 * (64 * 144 + 512)) and part.data_ptr() == pools[0].data_ptr()
    m.add_request("a")
    m.reserve([("a", 200)])
    m.commit([("a", 200)])
    m.reserve([("a", 260)])
    assert [g.tables["a"].count(-1) for g in m.kv_groups] == [0, 0, 1]        # a window gives its pages back
    m.check()


def test_what_a_build_does_not_take():
    with pytest.raises(ValueError, match="cache_bits"):
        BuildContext(torch.device("cpu"), torch.bfloat16, cache_bits=8)
    for bits, pages in ((16, 8), (4, 3), (4, -1)):
        with pytest.raises(ValueError, match="sparse_pages"):
            BuildContext(torch.device("cpu"), torch.bfloat16, cache_bits=bits, sparse_pages=pages)


# ------------------------------------------------------------------------------------------------ the engine
def engine(folder, dtype, **kw):
    from beglin_b200 import Engine
    return Engine.from_folder(folder, dtype=dtype, device="cuda:0", **{**dict(max_tokens=4096, page_size=16, max_requests=6, max_context=1024, cache_bits=4), **kw})


@GPU
@pytest.mark.parametrize("name,config", [("D", TINY_D), ("W", WIDE)])
@pytest.mark.parametrize("dtype,tol", [("float32", 2e-3), ("bfloat16", 8e-2)])
@pytest.mark.parametrize("many", [20, 240])
def test_logits_are_those_of_keys_and_values_in_4_bits(model_root, name, config, dtype, tol, many, monkeypatch):
    """float32: a key or value may lie so near the border of two codes that the layer's own rounding takes the other (a step of one feature of one position).
    bfloat16: many do.  A number that is off by d before it is rounded to steps of s crosses a border with probability d / s, and is then off by s: by sqrt(d s) in
    the mean of squares.  Of 64 normal numbers the largest and smallest lie 4.7 deviations apart, so s = 4.7 / 15 = 0.31 of one; d is what bfloat16 is allowed
    without such rounding, 2e-2: sqrt(2e-2 * 0.31) = 7.9e-2."""
    monkeypatch.setattr(ops, "PACKED_LONG_STREAMS", many)                      # (portions by either way)
    folder = make_model(model_root, "packed" + name, config=config, std=0.05, bias_std=0.05)
    ids, other = seeded_ids(170, config["vocab_size"], 5), seeded_ids(90, config["vocab_size"], 6)
    want, want_other = oracle(folder, ids), oracle(folder, other)
    eng = engine(folder, dtype)
    rows = [eng.step([("a", ids[:100], range(100))])]
    rows.append(eng.step([("a", ids[100:137], range(37)), ("b", other[:80], [79])]))       # a short portion beside a long one
    rows.append(eng.step([("a", ids[137:140], range(3)), ("b", other[80:81], [0])]))
    for i in range(140, 145):
        rows.append(eng.step([("a", ids[i:i + 1], [0]), ("b", other[i - 59:i - 58], [0])]))
    for i in range(145, 150):
        rows.append(eng.step([("a", ids[i:i + 1], [0])]))
    got_a = torch.cat([rows[0], rows[1][:37], rows[2][:3]] + [r[:1] for r in rows[3:]])
    got_b = torch.cat([rows[1][37:], rows[2][3:]] + [r[1:] for r in rows[3:8]])
    assert rel_err(got_a, want[:150]) < tol and rel_err(got_b, want_other[79:86]) < tol
    assert rel_err(want, helpers.plain_logits(folder, ids)) > tol              # (the rounding is what is tested, not lost in the tolerance)


@GPU
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replayed_steps_and_families(model_root, dtype):
    folder = make_model(model_root, "packedD", config=TINY_D, std=0.05, bias_std=0.05)
    prompts = [seeded_ids(n, 200, n) for n in (130, 3, 45)]
    made = {}
    for graphs in (False, True):
        eng = engine(folder, dtype, use_graphs=graphs, portion_graph_rows=32)
        made[graphs] = [eng.generate(prompts, max_new_tokens=20, stop_ids=()) for _ in range(2)]
        assert made[graphs][0] == made[graphs][1]
        eng.cache.check()
    family = engine(folder, dtype).generate(prompts[:2], max_new_tokens=20, stop_ids=(), completions=3)
    if dtype == "float32":
        assert made[True] == made[False]
        assert family == [[t] * 3 for t in made[True][0][:2]]
    assert all(len(t) == 20 for ts in made[True] + family for t in (ts if isinstance(ts[0], list) else [ts]))


@GPU
def test_a_fork_goes_on_from_the_same_page(model_root):
    folder = make_model(model_root, "packedW", config=WIDE, std=0.05, bias_std=0.05)
    ids = seeded_ids(75, 200, 9)
    eng = engine(folder, "float32")
    eng.step([("a", ids[:70], [])])
    eng.fork("a", ["b", "c"])
    alone = eng.step([("a", ids[70:71], [0])])
    both = eng.step([("b", ids[70:71], [0]), ("c", ids[71:72], [0])])
    assert rel_err(both[0], alone[0]) < 1e-5
    later = eng.step([("a", ids[71:75], range(4)), ("b", ids[71:75], range(4))])
    assert rel_err(later[4:], later[:4]) < 1e-5
    assert rel_err(later[:4], oracle(folder, ids)[71:75]) < 2e-3


@GPU
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_single_tokens_that_read_chosen_pages(model_root, dtype):
    folder = make_model(model_root, "packedW", config=WIDE, std=0.05, bias_std=0.05)
    ids = seeded_ids(700, 200, 3)
    every, some, enough = (engine(folder, dtype, sparse_pages=n) for n in (0, 6, 64))
    for eng in (every, some, enough):
        eng.step([("a", ids[:60], []), ("b", ids[:600], [])])
    assert some.cache.kv_groups[0].device_pool.shape[-1] == every.cache.kv_groups[0].device_pool.shape[-1] + 512
    for i in range(600, 650):
        a, b, c = (eng.step([("a", ids[i - 540:i - 539], [0]), ("b", ids[i:i + 1], [0])]) for eng in (every, some, enough))
        assert torch.equal(a, c)                                               # (as many pages as there are)
        if i < 620:                                                            # request a: at most 80 + 1 positions of 6 pages
            assert rel_err(b[0], a[0]) < (1e-5 if dtype == "float32" else 1e-2)
        assert bool(torch.isfinite(b).all())
    assert not torch.equal(a[1], b[1])
    graphs = [eng.generate([ids[:600], ids[:20]], max_new_tokens=8, stop_ids=()) for eng in (engine(folder, dtype, sparse_pages=6, use_graphs=g) for g in (False, True))]
    assert dtype == "bfloat16" or graphs[0] == graphs[1]


@GPU
def test_models_without_such_a_layer_are_refused(model_root):
    from beglin_b200 import Engine
    narrow = make_model(model_root, "A", seed=1)
    with pytest.raises(ValueError, match="no layer"):
        Engine.from_folder(narrow, device="cuda:0", max_tokens=128, page_size=16, cache_bits=4)
    folder = make_model(model_root, "packedD", config=TINY_D, std=0.05, bias_std=0.05)
    with pytest.raises(ValueError, match="no layer"):
        Engine.from_folder(folder, device="cuda:0", max_tokens=128, page_size=8, cache_bits=4)
    assert TINY_A["hidden_size"] // TINY_A["num_attention_heads"] == 16
    plainly = Engine.from_folder(folder, device="cuda:0", max_tokens=4096, page_size=16)
    packed = engine(folder, "bfloat16")
    assert 3.5 * packed.cache.device_bytes() < plainly.cache.device_bytes() < 3.6 * packed.cache.device_bytes()


@GPU
def test_the_command_line_has_both(model_root, tmp_path):
    folder = make_model(model_root, "packedD", config=TINY_D, std=0.05, bias_std=0.05)
    ids = tmp_path / "ids.i32"
    torch.tensor(seeded_ids(90, 200, 2), dtype=torch.int32).numpy().tofile(ids)
    env = dict(os.environ, QWEN_BASE=folder, QWEN_PROMPT=str(ids), QWEN_DTYPE="fp32", QWEN_SAFETENSORS_MAXSEQ="256", QWEN_PAGE_SIZE="16")
    exe = [sys.executable, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bin", "qwen_infer"), "greedy", "8"]
    lines = []
    for more in ({"QWEN_KV_INT4": "1"}, {"QWEN_KV_INT4": "1", "QWEN_SPARSE_PAGES": "16"}):
        r = subprocess.run(exe, env=dict(env, **more), capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr
        lines.append(r.stdout.strip().splitlines()[-1])
    want = engine(folder, "float32").generate([seeded_ids(90, 200, 2)], max_new_tokens=8, stop_ids=())[0]
    assert lines[0] == lines[1] == "greedy: " + " ".join(map(str, want))
    r = subprocess.run(exe, env=dict(env, QWEN_SPARSE_PAGES="16"), capture_output=True, text=True, timeout=600)
    assert r.returncode != 0 and "sparse_pages" in r.stderr
