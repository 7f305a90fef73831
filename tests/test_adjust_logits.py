"""Penalties, biases and masks of logits against a plain restatement in 64 bits, token by token from the lists."""
import math
from collections import Counter

import pytest
import torch

from beglin_b200.csrc import ops

DEV = "cuda:0"


def _plain(x, history, lengths, prompts, newest, rep, freq, pres, bias, allowed, allowed_row):
    """float64 [n, V], and the sum of the magnitudes that meet at each logit (what a rounding is relative to)."""
    x = x.double().clone()
    size = torch.zeros_like(x)
    n, V = x.shape
    for r in range(n):
        held = [] if history is None else history[r, :int(lengths[r])].tolist()
        given = len(held) if prompts is None else min(int(prompts[r]), len(held))
        given = 0 if prompts is None else given
        made = held[given:] + ([] if newest is None else [int(newest[r])])
        f, p = (0.0 if t is None else float(t[r]) for t in (freq, pres))
        k = 1.0 if rep is None else float(rep[r])
        for t in set(held[:given]) | set(made):
            v = float(x[r, t])
            x[r, t] = v / k if v > 0 else v * k
        size[r] = x[r].abs()
        for t, c in Counter(made).items():
            x[r, t] -= f * c + p
            size[r, t] += abs(f * c) + abs(p)
        if bias is not None:
            ids, values, begins = bias
            for j in range(int(begins[r]), int(begins[r + 1])):
                x[r, int(ids[j])] += float(values[j])
                size[r, int(ids[j])] += abs(float(values[j]))
        row = -1 if allowed is None else r if allowed_row is None else int(allowed_row[r])
        if row >= 0:
            t = torch.arange(V)
            x[r, (allowed[row].long()[t >> 5] >> (t & 31)) & 1 == 0] = -math.inf
    return x, size


def _case(n, V, held, seed, penalties=True, bias=0, masks="none", pad=0, offset=0, newest=True, prompts=True):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(n, V + pad + offset, generator=g) * 3
    x = buf[:, offset:offset + V]
    if V > 4:
        x[0, V // 2] = -math.inf
        x[-1, 1] = math.inf
        x[-1, 2] = math.nan
    lengths = torch.randint(0, held + 1, (n,), generator=g, dtype=torch.int32)
    lengths[0] = held
    if n > 2:
        lengths[2] = 0
    history = torch.randint(0, max(1, V // 3), (n, held + 2), generator=g, dtype=torch.int32)
    history = torch.where(torch.rand(n, held + 2, generator=g) < 0.3, torch.randint(0, V, (n, held + 2), generator=g, dtype=torch.int32), history)
    one = lambda lo, hi: torch.empty(n).uniform_(lo, hi, generator=g)
    a = {"history": history, "lengths": lengths, "prompts": (lengths.float() * torch.rand(n, generator=g)).int() if prompts else None,
         "newest": torch.randint(0, V, (n,), generator=g, dtype=torch.int32) if newest else None}
    a.update(rep=one(0.7, 1.5) if penalties else None, freq=one(-0.5, 1.0) if penalties else None, pres=one(-0.5, 1.0) if penalties else None,
             bias=None, allowed=None, allowed_row=None)
    if bias:
        ids, values, begins = [], [], [0]
        for r in range(n):
            k = bias if r != 1 else 0                     # a row without any
            few = torch.randint(0, V, (k,), generator=g).sort().values
            ids.append(few); values.append(torch.randn(k, generator=g)); begins.append(begins[-1] + k)
        a["bias"] = (torch.cat(ids).int(), torch.cat(values), torch.tensor(begins, dtype=torch.int32))
    if masks != "none":
        m = n if masks == "own" else 2
        words = torch.randint(-2 ** 31, 2 ** 31, (m, -(-V // 32) + 1), generator=g).to(torch.int32)
        words[0] = 0                                      # a mask that leaves nothing
        if m > 1:
            words[1] = -1
        a["allowed"] = words
        a["allowed_row"] = None if masks == "own" else torch.arange(n, dtype=torch.int32) % 3 - 1
    return x, a


def _run(x, a, in_place, device=DEV):
    move = lambda t: None if t is None else t.to(device)
    if in_place:
        base = torch.full((x.shape[0], x.stride(0) + 4), 7.0)
        base[:, :x.shape[1]] = x
        buf = base.to(device)
        logits = out = buf[:, :x.shape[1]]
    else:                                                  # x as it lies: rows apart, off 16 bytes
        buf = x.new_full((x.shape[0] * x.stride(0) + 64,), 7.0).to(device)
        start = x.storage_offset() % 4
        logits = buf[start:start + x.shape[0] * x.stride(0)].view(x.shape[0], x.stride(0))[:, :x.shape[1]]
        logits.copy_(x)
        out = torch.full(x.shape, 5.0, device=device)
    history = move(a["history"])
    bias = None if a["bias"] is None else tuple(move(t) for t in a["bias"])
    status = ops.new_status(device)
    ops.adjust_logits(logits, out, history=history, lengths=move(a["lengths"]), prompts=move(a["prompts"]), newest=move(a["newest"]),
                      repetition=move(a["rep"]), frequency=move(a["freq"]), presence=move(a["pres"]), bias=bias, allowed=move(a["allowed"]),
                      allowed_row=move(a["allowed_row"]), status=status)
    ops.raise_on_status(status)
    if in_place:
        assert bool((buf[:, x.shape[1]:] == 7.0).all())    # nothing behind a row is touched
    else:
        assert torch.equal(logits.cpu().nan_to_num(9.0), x.nan_to_num(9.0))
    return out.cpu(), history.cpu()


CASES = [dict(n=1, V=1, held=1), dict(n=2, V=31, held=0, masks="own"), dict(n=3, V=32, held=5, bias=3), dict(n=3, V=33, held=40, masks="some", bias=2),
         dict(n=4, V=4096, held=300, masks="own", bias=40), dict(n=4, V=4097, held=64, masks="some", pad=3, bias=5),
         dict(n=5, V=16387, held=1000, masks="some", bias=300, pad=1), dict(n=2, V=5000, held=2000, pad=3, offset=1),
         dict(n=3, V=9000, held=50, newest=False), dict(n=3, V=9000, held=50, prompts=False, masks="own"),
         dict(n=70, V=3001, held=37, masks="some", bias=4), dict(n=2, V=40000, held=77, penalties=False, masks="some", bias=9),
         dict(n=1, V=151936, held=513, bias=3),
         # many rows: a copy and a mending kernel; texts in a table of their tokens, longer ones and more biases than a thread holds, texts without a table
         dict(n=70, V=20011, held=300, masks="some", bias=4, pad=1), dict(n=140, V=10000, held=40, bias=3), dict(n=40, V=33000, held=9000, bias=1500, masks="some"),
         dict(n=40, V=33001, held=13000, bias=300, pad=3), dict(n=75, V=16390, held=900, penalties=False, bias=50), dict(n=64, V=20000, held=70, newest=False, masks="own")]


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_adjusted_logits(case, in_place):
    x, a = _case(seed=len(str(case)) + case["V"], **case)
    got, history = _run(x, a, in_place)
    want, size = _plain(x, **{k: v for k, v in a.items()})
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)].double(), want[~fine & ~torch.isnan(want)])
    # roundings, each of at most 2^-24 of what has come together at a logit: the division or product by the penalty, frequency times count, two
    # subtractions, one addition a biased entry (at most `most` entries of a token in these cases) and 1 for the products of these terms
    most = 0 if a["bias"] is None else max(int(torch.unique(a["bias"][0][a["bias"][2][r]:a["bias"][2][r + 1]], return_counts=True)[1].max())
                                           for r in range(case["n"]) if a["bias"][2][r + 1] > a["bias"][2][r])
    off = (got.double() - want).abs()
    assert bool((off[fine] <= 2.0 ** -24 * (5 + most) * size[fine]).all())
    if a["newest"] is not None:
        for r in range(case["n"]):
            k = int(a["lengths"][r])
            assert int(history[r, k]) == int(a["newest"][r])
            a["history"][r, k] = history[r, k]
    assert torch.equal(history, a["history"])              # and nothing else of the history


@pytest.mark.gpu
def test_adjusted_logits_step_after_step_is_one_history():
    """`newest` token by token gives what the whole list gives at once."""
    g = torch.Generator().manual_seed(3)
    V, prompt = 700, [5, 9, 5, 1]
    made = torch.randint(0, 20, (9,), generator=g).tolist()
    x = torch.randn(1, V, generator=g).to(DEV)
    history = torch.full((1, 16), 3, dtype=torch.int32, device=DEV)
    history[0, :4] = torch.tensor(prompt, dtype=torch.int32)
    lengths, i32 = torch.tensor([4], dtype=torch.int32, device=DEV), lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    rules = dict(repetition=torch.tensor([1.2], device=DEV), frequency=torch.tensor([0.3], device=DEV), presence=torch.tensor([0.4], device=DEV))
    for i, token in enumerate(made):
        out = torch.empty_like(x)
        ops.adjust_logits(x, out, history=history, lengths=lengths, prompts=i32(4), newest=i32(token), **rules)
        lengths += 1
        whole = torch.empty_like(x)
        held = torch.tensor([prompt + made[:i + 1]], dtype=torch.int32, device=DEV)
        ops.adjust_logits(x, whole, history=held, lengths=i32(held.shape[1]), prompts=i32(4), **rules)
        assert torch.equal(out, whole)
    assert history[0, :13].tolist() == prompt + made


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["history", "newest", "bias", "order", "full", "mask"])
def test_adjusted_logits_record_what_is_not_there(what):
    V, n = 100, 2
    x = torch.zeros(n, V, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    a = dict(history=torch.zeros((n, 3), dtype=torch.int32, device=DEV), lengths=i32(1, 2), repetition=torch.full((n,), 2.0, device=DEV))
    if what == "history":
        a["history"][1, 1] = V
    elif what == "newest":
        a["newest"] = i32(4, -2)
    elif what == "full":
        a.update(newest=i32(4, 5), lengths=i32(3, 1))
    elif what == "bias":
        a["bias"] = (i32(3, V), torch.ones(2, device=DEV), i32(0, 1, 2))
    elif what == "order":
        a["bias"] = (i32(3, 2, 7), torch.ones(3, device=DEV), i32(0, 2, 3))
    else:
        a.update(allowed=torch.full((1, 4), -1, dtype=torch.int32, device=DEV), allowed_row=i32(0, 1))
    status, out = ops.new_status(DEV), torch.empty_like(x)
    ops.adjust_logits(x, out, status=status, **a)
    with pytest.raises(ops.KernelError, match="token id"):
        ops.raise_on_status(status)
    assert bool(torch.isfinite(out).all())


def test_adjusted_logits_refuse_what_does_not_fit():
    x, i32 = torch.zeros(2, 40), lambda *v: torch.tensor(v, dtype=torch.int32)
    history, lengths, words = torch.zeros((2, 4), dtype=torch.int32), i32(1, 1), torch.zeros((2, 2), dtype=torch.int32)

    def refused(match, logits=x, out=None, **kw):
        with pytest.raises(ops.KernelError, match=match):
            ops.adjust_logits(logits, torch.zeros_like(logits) if out is None else out, **kw)

    refused("CUDA device only")
    refused("float32", logits=x.double())
    refused("float32", out=torch.zeros(2, 41))
    refused("side by side", logits=torch.zeros(40, 2).t())
    refused("side by side", out=torch.zeros(1, 40).expand(2, 40))
    both = torch.zeros(3, 40)
    refused("memory apart", logits=both[:2], out=both[1:])
    refused("goes with its lengths", history=history)
    refused("history", newest=lengths)
    refused("history is", history=history[:1].contiguous(), lengths=lengths)
    refused("int32", history=history.long(), lengths=lengths)
    refused("one number per row", history=history, lengths=i32(1))
    refused("one number per row", history=history, lengths=lengths, prompts=i32(1, 1, 1))
    refused("one number per row", repetition=torch.ones(2, dtype=torch.float64))
    refused("begins", bias=(i32(1), torch.ones(1), i32(0, 1)))
    refused("bias is", bias=(i32(1), torch.ones(2), i32(0, 1, 1)))
    refused("expected", allowed=words[:, :1].contiguous())
    refused("mask for each", allowed=words[:1].contiguous())
    refused("goes with masks", allowed_row=i32(0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,V,held,bias", [(3, 300, 5, 0), (70, 20011, 40, 3), (40, 33001, 13000, 2)])
def test_the_newest_token_is_the_prompts_where_its_place_is(n, V, held, bias, in_place):
    """A token in front of the prompt's end counts as the prompt's whether it is the newest or lies in the history: one kernel, a table of the text's tokens and
    ranges of the vocabulary."""
    x, a = _case(n, V, held, seed=n + V, bias=bias)
    rows = torch.arange(n)
    a["prompts"] = (a["lengths"] + torch.tensor([1, 7, 0])[rows % 3]).int()
    whole = dict(a, history=a["history"].clone(), lengths=a["lengths"] + 1, newest=None)
    whole["history"][rows, a["lengths"].long()] = a["newest"]
    got, history = _run(x, a, in_place)
    want, size = _plain(x, **whole)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    # (the roundings of test_adjusted_logits, and at most four biases of one token)
    assert bool(((got.double() - want).abs()[fine] <= 2.0 ** -24 * (5 + 4) * size[fine]).all())
    assert torch.equal(got.nan_to_num(9.0), _run(x, whole, in_place)[0].nan_to_num(9.0))
    assert torch.equal(history, whole["history"])


def test_one_row_of_logits_lies_side_by_side_too():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    row, apart, same = torch.zeros(1, 40), torch.zeros(1, 80)[:, ::2], torch.zeros(1, 1).expand(1, 40)
    column = torch.zeros(40, 3).t()[:1]
    for bad in (apart, same, column):
        for logits, out in ((bad, row), (row, bad), (bad, bad)):
            with pytest.raises(ops.KernelError, match="side by side"):
                ops.adjust_logits(logits, out, history=torch.zeros((1, 4), dtype=torch.int32), lengths=i32(1))
    # (one logit a row has nothing beside it, and one row nothing behind it)
    for fine in (torch.zeros(1, 80)[:, :40], torch.zeros(1, 8)[:, ::8], torch.zeros(3, 8)[:, ::8], torch.zeros(2, 40)[:1], torch.zeros(1, 40).as_strided((1, 40), (7, 1))):
        with pytest.raises(ops.KernelError, match="CUDA device only"):
            ops.adjust_logits(fine, torch.zeros(fine.shape))
