"""What generating several completions of one prompt needs beside a model's layers, as measurable cases.

Three operators.  Attention of decoding rows whose requests share the first positions of their cache: the shared positions
are read once for all rows of a group, each row's own ones behind them by itself.  The adjustment of logits before a token is
chosen: penalties for tokens that a request holds already, biases, and masks of the tokens that a grammar allows.  And the
copy of the positions at the end of a prompt that do not fill a page, for requests that go on from them separately.

`run` computes them in their plain form from elementary operations in 32 bits, or, where `own` is set, with this framework's
kernels.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # two completions of a short prompt, a few tokens in: the smallest step, all latency
        {"name": "shared_two", "kind": "shared", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "groups": "2:512",
         "alone": 0, "own_lo": 1, "own_hi": 16, "cap": 0.0, "sink": 0},
        # eight completions of a prompt of some 4,000 tokens, lengths apart
        {"name": "shared_eight", "kind": "shared", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "groups": "8:3968",
         "alone": 0, "own_lo": 5, "own_hi": 300, "cap": 0.0, "sink": 0},
        # sixty-four samples of one long prompt: best of n
        {"name": "shared_sixtyfour", "kind": "shared", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64,
         "groups": "64:8192", "alone": 0, "own_lo": 60, "own_hi": 500, "cap": 0.0, "sink": 0},
        # a mixed batch: three prompts with some completions each beside requests of their own, pages of 16, a layer with a
        # learned sink
        {"name": "shared_groups", "kind": "shared", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 16,
         "groups": "20:5008,7:1040,3:12000", "alone": 5, "own_lo": 1, "own_hi": 900, "cap": 0.0, "sink": 1},
        # small heads, squashed scores
        {"name": "shared_narrow", "kind": "shared", "dtype": "bfloat16", "heads": 14, "kv_heads": 2, "dim": 64, "page": 64, "groups": "33:1984",
         "alone": 1, "own_lo": 1, "own_hi": 200, "cap": 30.0, "sink": 0},
        # a server whose requests all begin with one long document
        {"name": "shared_document", "kind": "shared", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "groups": "256:32768", "alone": 0, "own_lo": 100, "own_hi": 800, "cap": 0.0, "sink": 0},
        # the 32-bit path
        {"name": "shared_float", "kind": "shared", "dtype": "float32", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "groups": "16:4096",
         "alone": 0, "own_lo": 3, "own_hi": 300, "cap": 0.0, "sink": 0},
        # one request under penalties
        {"name": "logits_one", "kind": "logits", "rows": 1, "vocab": 151936, "held": 700, "prompt": 0.6, "bias": 0, "masked": 0.0, "pad": 0},
        # a server's batch: long histories, a bias list each, grammars in half of the rows
        {"name": "logits_batch", "kind": "logits", "rows": 64, "vocab": 151936, "held": 4096, "prompt": 0.8, "bias": 300, "masked": 0.5, "pad": 0},
        # an odd vocabulary, rows apart in memory, every row under a grammar
        {"name": "logits_odd", "kind": "logits", "rows": 9, "vocab": 50257, "held": 130, "prompt": 0.5, "bias": 7, "masked": 1.0, "pad": 3},
        # one more completion of a prompt: the end of the prompt for 28 layers
        {"name": "copy_one", "kind": "copy", "dtype": "bfloat16", "stages": 28, "kv_heads": 2, "dim": 128, "page": 64, "copies": 1, "sources": 1,
         "positions": 29},
        # sixty-three more of it
        {"name": "copy_many", "kind": "copy", "dtype": "bfloat16", "stages": 28, "kv_heads": 2, "dim": 128, "page": 64, "copies": 63, "sources": 1,
         "positions": 45},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "logits", "logits", "copy"])
    if kind == "shared":
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        kv = rng.choice([1, 2, 2, 4, 8])
        heads = kv * rng.randint(1, 8)
        page = rng.choice([16, 64, 64])
        cost = 40e6 if dtype == "float32" else 400e6             # query heads times positions that the batch may take
        groups, rows = [], 0
        for _ in range(rng.choice([1, 1, 1, 2, 3])):
            n = _log(rng, 2, 64 if dtype == "float32" else 200)
            most = min(32768, int(cost / (n * heads)))
            positions = _log(rng, 64, max(most, 65))
            groups.append("%d:%d" % (n, positions if rng.random() < 0.4 else max(1, positions // page) * page))
            rows += n
        lo = _log(rng, 1, 64)
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": rng.choice([64, 128, 128]), "page": page,
                "groups": ",".join(groups), "alone": rng.choice([0, 0, 1, 6]), "own_lo": lo, "own_hi": lo + _log(rng, 1, 700),
                "cap": rng.choice([0.0, 0.0, 0.0, 20.0]), "sink": rng.choice([0, 0, 0, 1])}
    if kind == "logits":
        return {"kind": kind, "rows": _log(rng, 1, 128), "vocab": _log(rng, 2000, 160000), "held": _log(rng, 1, 6000), "prompt": rng.random(),
                "bias": rng.choice([0, 1, 30, 300]), "masked": rng.choice([0.0, 0.0, 0.5, 1.0]), "pad": rng.choice([0, 0, 1, 64])}
    page = rng.choice([16, 64])
    return {"kind": kind, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "stages": rng.randint(2, 48), "kv_heads": rng.choice([1, 2, 4]),
            "dim": rng.choice([64, 80, 128]), "page": page, "copies": _log(rng, 1, 63), "sources": rng.choice([1, 1, 3]),
            "positions": rng.randint(1, page)}


# ------------------------------------------------------------------------------------------------ inputs, from the seed alone
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _groups(c):
    """[(rows, shared positions)] of the batch, requests of their own as groups of one that share nothing.  The groups lie one behind
    the other, the requests of their own at both ends."""
    out, row = [], 0
    front = c["alone"] // 2
    for i in range(front):
        out.append(([row], 0))
        row += 1
    for text in c["groups"].split(","):
        n, positions = (int(v) for v in text.split(":"))
        out.append((list(range(row, row + n)), positions))
        row += n
    for i in range(c["alone"] - front):
        out.append(([row], 0))
        row += 1
    return out


def _own_lengths(c, seed):
    """Positions of a request behind those that it shares, the newest token's included."""
    n = sum(len(rows) for rows, _ in _groups(c))
    g = torch.Generator().manual_seed(int(seed) * 7919 + 13)
    return torch.randint(c["own_lo"], c["own_hi"] + 1, (n,), generator=g).tolist()


def _shared_inputs(c, seed):
    g, ps, dt = _generator(seed), c["page"], DTYPES[c["dtype"]]
    groups, own_len = _groups(c), _own_lengths(c, seed)
    n = len(own_len)
    lengths, tables, pages = [0] * n, [None] * n, 0
    for rows, shared in groups:
        whole = shared // ps                               # pages that all rows of the group hold together
        common = list(range(pages, pages + whole))
        pages += whole
        for r in rows:
            lengths[r] = shared + own_len[r]
            more = -(-lengths[r] // ps) - whole
            tables[r] = common + list(range(pages, pages + more))
            pages += more
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()
    width = max(len(t) for t in tables) + 3
    table = torch.tensor([[order[p] for p in t] + [-1] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
    H, kv, d = c["heads"], c["kv_heads"], c["dim"]
    pool = torch.empty((pages, 2, kv, ps, d), dtype=dt, device="cuda")
    for p0 in range(0, pages, 4096):
        pool[p0:p0 + 4096] = _normal(g, min(4096, pages - p0), 2, kv, ps, d, dtype=dt)
    for rows, shared in groups:                            # a page that sharing ends in: every row holds the same positions
        if shared % ps:
            first = order[tables[rows[0]][shared // ps]]
            for r in rows[1:]:
                pool[order[tables[r][shared // ps]], :, :, :shared % ps] = pool[first, :, :, :shared % ps]
    return {"q": _normal(g, n, H * d, std=1.5, dtype=dt), "pool": pool, "table": table,
            "positions": torch.tensor([v - 1 for v in lengths], dtype=torch.int32).cuda(), "lengths": lengths, "groups": groups,
            "sink": _normal(g, H, std=2.0) if c["sink"] else None, "scale": 1.0 / math.sqrt(d)}


def _logits_inputs(c, seed):
    g, n, V = _generator(seed), c["rows"], c["vocab"]
    cpu = torch.Generator().manual_seed(int(seed) * 104729 + 7)
    buf = _normal(g, n, V + c["pad"], std=3.0)
    logits = buf[:, :V]
    logits[:, V - max(1, V // 500):] = -math.inf          # ids that a head has rows for and a tokenizer has no tokens
    lengths = torch.randint(max(1, c["held"] // 2), c["held"] + 1, (n,), generator=cpu)
    prompts = (lengths.double() * c["prompt"]).to(torch.int64)
    cap = c["held"] + 2
    # texts: most tokens come from a small part of the vocabulary, and come again
    often = torch.randint(0, V, (n, max(1, c["held"] // 5)), generator=cpu)
    pick = torch.randint(0, often.shape[1], (n, cap), generator=cpu)
    history = torch.where(torch.rand((n, cap), generator=cpu) < 0.7, torch.gather(often, 1, pick), torch.randint(0, V, (n, cap), generator=cpu))
    newest = torch.gather(often, 1, pick[:, :1])[:, 0]
    one = lambda lo, hi: torch.empty(n, dtype=torch.float32).uniform_(lo, hi, generator=cpu)
    state = {"logits": logits, "history": history.to(torch.int32).cuda(), "lengths": lengths.to(torch.int32).cuda(),
             "prompts": prompts.to(torch.int32).cuda(), "newest": newest.to(torch.int32).cuda(), "repetition": one(0.8, 1.4).cuda(),
             "frequency": one(-0.2, 0.6).cuda(), "presence": one(-0.3, 0.8).cuda(), "bias": None, "allowed": None, "allowed_row": None}
    if c["bias"]:
        ids = [torch.randperm(V, generator=cpu)[:c["bias"]].sort().values for _ in range(n)]
        state["bias"] = (torch.cat(ids).to(torch.int32).cuda(), _normal(g, n * c["bias"], std=4.0),
                         torch.arange(n + 1, dtype=torch.int32).cuda() * c["bias"])
    if c["masked"] > 0.0:
        words = -(-V // 32)
        masked = [r for r in range(n) if r < max(1, round(c["masked"] * n))]
        rows = []
        for i in range(len(masked)):
            if i % 2 == 0:                                 # few tokens allowed: a structure's next symbols
                bits = torch.zeros(words * 32, dtype=torch.bool)
                bits[torch.randint(0, V, (20,), generator=cpu)] = True
            else:                                          # most allowed: inside a text
                bits = torch.rand(words * 32, generator=cpu) < 0.97
            rows.append((bits.view(words, 32).to(torch.int64) << torch.arange(32)).sum(1))
        packed = torch.stack(rows)
        state["allowed"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32).cuda()
        where = torch.full((n,), -1, dtype=torch.int32)
        where[torch.tensor(masked)] = torch.arange(len(masked), dtype=torch.int32)
        state["allowed_row"] = where.cuda()
    return state


def _copy_inputs(c, seed):
    g, k, s = _generator(seed), c["copies"], min(c["sources"], c["copies"])
    pages = k + s + 5
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 11)).tolist()
    pool = torch.empty((c["stages"], pages, 2, c["kv_heads"], c["page"], c["dim"]), dtype=DTYPES[c["dtype"]], device="cuda")
    for i in range(c["stages"]):
        pool[i] = _normal(g, *pool.shape[1:], dtype=pool.dtype)
    return {"pool": pool, "src": [order[i % s] for i in range(k)], "dst": order[s:s + k], "positions": c["positions"]}


_INPUTS = {"shared": _shared_inputs, "logits": _logits_inputs, "copy": _copy_inputs}


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    state["case"] = case
    if case["kind"] == "shared":
        state["out"] = torch.empty_like(state["q"])
        if own:
            from beglin_b200.cache.shared import SharedPrefix
            from beglin_b200.csrc import ops
            c = case
            shared = SharedPrefix(len(state["lengths"]), [(rows, n) for rows, n in state["groups"] if len(rows) > 1])
            state["plan"] = ops.shared_plan(shared, c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]], page_size=c["page"], device="cuda")
            state["status"] = ops.new_status("cuda")
    elif case["kind"] == "logits":
        state["out"] = torch.empty((case["rows"], case["vocab"]), dtype=torch.float32, device="cuda")
        if own:
            from beglin_b200.csrc import ops
            state["status"] = ops.new_status("cuda")
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state)
    return _PLAIN[state["case"]["kind"]](state)


def _own_shared(s):
    from beglin_b200.csrc import ops
    ops.shared_attention(s["q"], s["pool"], s["table"], s["positions"], s["plan"], max(s["lengths"]) - 1, s["scale"], s["out"], s["status"],
                         sink_weight=s["sink"], softcap=s["case"]["cap"])
    return s["out"]


def _own_logits(s):
    from beglin_b200.csrc import ops
    ops.adjust_logits(s["logits"], s["out"], history=s["history"], lengths=s["lengths"], prompts=s["prompts"], newest=s["newest"],
                      repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias=s["bias"], allowed=s["allowed"],
                      allowed_row=s["allowed_row"], status=s["status"])
    return {"logits": s["out"], "history": s["history"]}


def _own_copy(s):
    from beglin_b200.csrc import ops
    ops.copy_pages(s["pool"], s["src"], s["dst"], s["positions"])
    return s["pool"]


_OWN = {"shared": _own_shared, "logits": _own_logits, "copy": _own_copy}


def _keys(pool, pages, first, last):
    """Keys and values [kv heads, last - first, features] as float32 of the positions first .. last - 1 of a table's pages."""
    ps = pool.shape[3]
    p0, p1 = first // ps, -(-last // ps)
    t = pool[pages[p0:p1].long()].float().permute(1, 2, 0, 3, 4)               # 2, kv, pages, positions, features
    t = t.reshape(2, pool.shape[2], -1, pool.shape[4])[:, :, first - p0 * ps:last - p0 * ps]
    return t[0], t[1]


def _weigh(q, k, v, scale, cap):
    """Running maximum, sum and weighted values of queries [kv, m, d] over keys [kv, n, d]."""
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    if cap > 0.0:
        s = cap * torch.tanh(s / cap)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _plain_shared(s):
    c, pool, table, out = s["case"], s["pool"], s["table"], s["out"]
    H, kv, d = c["heads"], c["kv_heads"], c["dim"]
    per = H // kv
    q = s["q"].float().view(-1, kv, per, d)
    sink = None if s["sink"] is None else s["sink"].view(kv, per, 1)
    for rows, shared in s["groups"]:
        r0, n = rows[0], len(rows)
        if shared:
            parts = []
            for h in range(kv):                            # a kv head at a time, the scores of all take too much room
                k, v = _keys(pool[:, :, h:h + 1], table[r0], 0, shared)
                parts.append(_weigh(q[r0:r0 + n, h].reshape(1, n * per, d), k, v, s["scale"], c["cap"]))
            ma, la, oa = (torch.cat([p[i] for p in parts]).view(kv, n, per, -1) for i in range(3))
        for i, r in enumerate(rows):
            k, v = _keys(pool, table[r], shared, s["lengths"][r])
            m, l, o = _weigh(q[r], k, v, s["scale"], c["cap"])
            if shared:
                top = torch.maximum(m, ma[:, i])
                a, b = torch.exp(ma[:, i] - top), torch.exp(m - top)
                m, l, o = top, la[:, i] * a + l * b, oa[:, i] * a + o * b
            if sink is not None:
                top = torch.maximum(m, sink)
                b = torch.exp(m - top)
                l, o = l * b + torch.exp(sink - top), o * b
            out[r] = (o / l).reshape(-1).to(out.dtype)
    return out


def _plain_logits(s):
    x, n, V = s["logits"].clone(), s["logits"].shape[0], s["logits"].shape[1]
    at, lengths = torch.arange(s["history"].shape[1], device=x.device), s["lengths"].long()
    s["history"].scatter_(1, lengths[:, None], s["newest"][:, None])           # the newest token is held from now on
    ids = s["history"].long()
    held = at[None] <= lengths[:, None]
    given = held & (at[None] < s["prompts"][:, None])
    made = held & ~given
    count = torch.zeros((n, V + 1), dtype=torch.float32, device=x.device)
    count.scatter_add_(1, torch.where(made, ids, V), torch.ones_like(ids, dtype=torch.float32))
    seen = count > 0
    seen.scatter_(1, torch.where(given, ids, V), torch.ones_like(given))
    count, seen = count[:, :V], seen[:, :V]
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - torch.where(count > 0, s["presence"][:, None], torch.zeros_like(x))
    if s["bias"] is not None:
        b_ids, b_values, b_rows = s["bias"]
        row = torch.searchsorted(b_rows, torch.arange(b_ids.numel(), device=x.device, dtype=torch.int32), right=True) - 1
        x.view(-1).index_add_(0, row * V + b_ids.long(), b_values)
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        bits = bits.reshape(bits.shape[0], -1)[:, :V] != 0
        where = s["allowed_row"].long()
        ok = bits[where.clamp(min=0)] | (where < 0)[:, None]
        x = torch.where(ok, x, torch.full_like(x, -math.inf))
    s["out"].copy_(x)
    return {"logits": s["out"], "history": s["history"]}


def _plain_copy(s):
    pool, n = s["pool"], s["positions"]
    src, dst = (torch.tensor(s[k], device=pool.device) for k in ("src", "dst"))
    pool[:, dst, :, :, :n] = pool[:, src, :, :, :n]
    return pool


_PLAIN = {"shared": _plain_shared, "logits": _plain_logits, "copy": _plain_copy}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "shared":
        size, d, kv, H = DTYPES[c["dtype"]].itemsize, c["dim"], c["kv_heads"], c["heads"]
        mean_own = (c["own_lo"] + c["own_hi"]) / 2
        read = pairs = rows = 0
        for g, shared in _groups(c):
            read += shared + len(g) * mean_own
            pairs += len(g) * (shared + mean_own)
            rows += len(g)
        return {"bytes": int(read * 2 * kv * d * size + 2 * rows * H * d * size + 4 * read / c["page"]), "flops": int(4 * pairs * H * d)}
    if c["kind"] == "logits":
        n, V = c["rows"], c["vocab"]
        masked = max(1, round(c["masked"] * n)) if c["masked"] > 0.0 else 0
        return {"bytes": 8 * n * V + 3 * n * c["held"] + 8 * n * c["bias"] + 4 * masked * -(-V // 32), "flops": 2 * n * V}
    one = c["stages"] * 2 * c["kv_heads"] * c["positions"] * c["dim"] * DTYPES[c["dtype"]].itemsize
    return {"bytes": one * (c["copies"] + min(c["sources"], c["copies"])), "flops": 0}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    return _EXACT[case["kind"]](case, s)


def _exact_shared(c, s):
    """Row by row: softmax over all of a row's positions, each looked up in the row's own table (a page that sharing ends in
    holds the same positions for every row)."""
    H, kv, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    result = torch.empty((len(s["lengths"]), H * d), dtype=torch.float64, device="cuda")
    for r, length in enumerate(s["lengths"]):
        at = torch.arange(length, device="cuda")
        page, slot = s["table"][r].long()[at // ps], at % ps
        for h in range(kv):
            key, value = s["pool"][page, 0, h, slot].double(), s["pool"][page, 1, h, slot].double()
            heads = slice(h * (H // kv), (h + 1) * (H // kv))
            score = torch.einsum("gd,nd->gn", s["q"][r].double().view(H, d)[heads], key) * s["scale"]
            if c["cap"] > 0.0:
                score = c["cap"] * torch.tanh(score / c["cap"])
            if s["sink"] is not None:
                score = torch.cat([score, s["sink"].double()[heads, None]], dim=1)
            weight = torch.softmax(score, dim=1)[:, :length]
            result[r].view(H, d)[heads] = torch.einsum("gn,nd->gd", weight, value)
    return result


def _exact_logits(c, s):
    """Row by row, from the lists of tokens."""
    x, history = s["logits"].double(), s["history"].clone()
    V, ids_all = c["vocab"], torch.arange(c["vocab"], device="cuda")
    for r in range(c["rows"]):
        length, prompt = int(s["lengths"][r]), int(s["prompts"][r])
        history[r, length] = s["newest"][r]
        made, counts = torch.unique(history[r, prompt:length + 1].long(), return_counts=True)
        seen, rep = torch.unique(history[r, :length + 1].long()), s["repetition"][r].double()
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        x[r, made] -= counts.double() * s["frequency"][r].double() + s["presence"][r].double()
        if s["bias"] is not None:
            lo, hi = int(s["bias"][2][r]), int(s["bias"][2][r + 1])
            x[r, s["bias"][0][lo:hi].long()] += s["bias"][1][lo:hi].double()
        if s["allowed"] is not None and int(s["allowed_row"][r]) >= 0:
            word = s["allowed"][int(s["allowed_row"][r])].long()[ids_all >> 5]
            x[r, ((word >> (ids_all & 31)) & 1) == 0] = -math.inf
    return {"logits": x, "history": history}


def _exact_copy(c, s):
    pool = s["pool"].clone()
    for a, b in zip(s["src"], s["dst"]):
        pool[:, b, :, :, :c["positions"]] = s["pool"][:, a, :, :, :c["positions"]]
    return pool


_EXACT = {"shared": _exact_shared, "logits": _exact_logits, "copy": _exact_copy}
