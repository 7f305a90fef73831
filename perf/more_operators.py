"""What serving with a cache held in 4 bits needs, as measurable cases.

Three operators.  Appending a step's keys and values to pages that hold them in 4 bits, with the rotation of queries and keys on
the way.  Attention over such pages: single tokens, and prompt portions beside them.  And sparse attention for single tokens: for
every row and kv head the pages whose keys can score highest, by the smallest and largest value that a page holds of every
feature, and attention over those pages alone.

A page holds, for each kv head, tiles of 16 positions: the keys' codes, the values' codes and, for every position, a (step, lowest)
pair in bfloat16 for each group of 64 features of its key and of its value; the value that a code u stands for is lowest + step u.
Behind the tiles may stand the smallest and the largest value of every feature of the page's keys, in bfloat16.

`run` computes them in their plain form from elementary operations, or, where `own` is set, with this framework's kernels.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
TILE, GROUP = 16, 64


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one request's next token: the smallest append
        {"name": "append_one", "kind": "append", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "rows": "1", "hi": 3000,
         "rot": 128, "interleaved": 0, "bounds": 0},
        # a decoding step of a server's batch, larger layers
        {"name": "append_batch", "kind": "append", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64, "rows": "1*64", "hi": 8000,
         "rot": 128, "interleaved": 0, "bounds": 1},
        # portions of two long prompts beside single tokens; every page that is filled gets its bounds
        {"name": "append_portion", "kind": "append", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64, "rows": "4096,1*20,801",
         "hi": 9000, "rot": 128, "interleaved": 0, "bounds": 1},
        # one request, a few thousand tokens in: latency
        {"name": "attend_one", "kind": "attend", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "rows": 1, "lo": 4000, "hi": 4096,
         "window": 0, "cap": 0.0, "sink": 0},
        # a server's batch, lengths apart
        {"name": "attend_batch", "kind": "attend", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "rows": 64, "lo": 2048, "hi": 8192,
         "window": 0, "cap": 0.0, "sink": 0},
        # few requests with very long texts, which is what 4 bits make room for
        {"name": "attend_long", "kind": "attend", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64, "rows": 4, "lo": 120000, "hi": 131072,
         "window": 0, "cap": 0.0, "sink": 0},
        # small heads, small pages, squashed scores and a learned sink
        {"name": "attend_narrow", "kind": "attend", "dtype": "bfloat16", "heads": 14, "kv_heads": 2, "dim": 64, "page": 16, "rows": 33, "lo": 1, "hi": 5000,
         "window": 0, "cap": 30.0, "sink": 1},
        # the 32-bit path
        {"name": "attend_float", "kind": "attend", "dtype": "float32", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "rows": 8, "lo": 1000, "hi": 4096,
         "window": 0, "cap": 0.0, "sink": 0},
        # a prompt of some 2,000 tokens in one portion
        {"name": "portion_prompt", "kind": "portion", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "requests": "2048:0"},
        # a mixed step: a portion of a long prompt, a short one, and decoding requests
        {"name": "portion_mixed", "kind": "portion", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "requests": "1:8000,1000:15000,1:3111,17:300,1:12000,1:63,1:700"},
        # very long texts of which a step reads 64 pages
        {"name": "sparse_long", "kind": "sparse", "dtype": "bfloat16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64, "rows": 4, "lo": 120000,
         "hi": 131072, "top": 64, "first": 1, "recent": 2},
        # a server's batch of long texts, some of them no longer than what is read
        {"name": "sparse_batch", "kind": "sparse", "dtype": "bfloat16", "heads": 12, "kv_heads": 2, "dim": 128, "page": 64, "rows": 32, "lo": 1500,
         "hi": 32768, "top": 32, "first": 1, "recent": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "portion", "sparse"])
    kv = rng.choice([1, 2, 2, 4, 8])
    c = {"kind": kind, "dtype": "bfloat16", "heads": kv * rng.randint(1, 8), "kv_heads": kv, "dim": rng.choice([64, 128, 128]),
         "page": rng.choice([16, 32, 64, 64])}
    if kind == "append":
        c["dtype"] = rng.choice(["bfloat16", "bfloat16", "float32"])
        many = rng.choice(["1*%d" % _log(rng, 1, 128), "%d" % _log(rng, 2, 4096), "%d,1*%d" % (_log(rng, 2, 3500), rng.randint(1, 40))])
        return c | {"rows": many, "hi": _log(rng, 1, 9000), "rot": rng.choice([c["dim"], c["dim"], c["dim"] // 2, 0]),
                    "interleaved": rng.choice([0, 0, 1]), "bounds": rng.choice([0, 1])}
    if kind == "attend":
        c["dtype"] = rng.choice(["bfloat16"] * 4 + ["float32"])
        rows = _log(rng, 1, 128)
        # (what the batch may take: query heads times positions, and what it reads of the cache)
        most = max(2, min(131072, int((4e6 if c["dtype"] == "float32" else 14e6) / (rows * c["heads"])), 2000000 // (rows * kv)))
        hi = _log(rng, 1, most)
        return c | {"rows": rows, "lo": rng.choice([1, max(1, hi // 2), hi]), "hi": hi, "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                    "cap": rng.choice([0.0, 0.0, 0.0, 20.0]), "sink": rng.choice([0, 0, 0, 1])}
    if kind == "portion":
        n = _log(rng, 2, 2048)
        start = rng.choice([0, _log(rng, 1, max(2, int(4e8 / (n * c["heads"])) - n))])
        parts = ["%d:%d" % (n, min(start, 30000))]
        parts += ["%d:%d" % (rng.choice([1, 1, rng.randint(2, 40)]), _log(rng, 1, 12000) - 1) for _ in range(rng.randint(0, 6))]
        rng.shuffle(parts)
        return c | {"requests": ",".join(parts)}
    rows = _log(rng, 1, 48)
    hi = _log(rng, c["page"], max(2 * c["page"], min(131072, 14000000 // (rows * c["heads"]), 2000000 // (rows * kv))))
    first, recent = rng.randint(0, 2), rng.randint(1, 3)
    return c | {"rows": rows, "lo": rng.choice([1, hi // 2 + 1]), "hi": hi, "top": first + recent + _log(rng, 1, 100), "first": first, "recent": recent}


# ------------------------------------------------------------------------------------------------ inputs, from the seed alone
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _sizes(c):
    """(groups of 64 features, bytes of a tile's keys, of a tile, of a page's tiles for one kv head)."""
    groups = c["dim"] // GROUP
    codes = TILE * c["dim"] // 2
    tile = 2 * codes + TILE * 2 * groups * 4
    return groups, codes, tile, c["page"] // TILE * tile


def _tables(lengths, page, seed, pages=0):
    """A block table of pages in a random order for requests of these lengths; how many pages there are (or of `pages`, where that is more)."""
    counts = [-(-n // page) for n in lengths]
    pages = max(pages, sum(counts) + 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()
    rows, at, width = [], 0, max(counts) + 2
    for n in counts:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32).cuda(), pages


def _pool(c, g, pages, bounds):
    """Pages as a cache holds them: any codes, the spread and the middle of a group of features as rotated keys have them, and the bounds of
    every page's keys."""
    groups, codes, tile, tiles = _sizes(c)
    pool = torch.randint(0, 256, (pages, c["kv_heads"], tiles + (4 * c["dim"] if bounds else 0)), dtype=torch.uint8, device="cuda", generator=g)
    at = pool[:, :, :tiles].unflatten(2, (-1, tile))[..., 2 * codes:].view(torch.bfloat16).unflatten(3, (TILE, 2, groups, 2))
    step = torch.empty(at.shape[:-1], device="cuda").uniform_(0.15, 0.45, generator=g)
    drift = _normal(g, pages, c["kv_heads"], 1, 1, 2, groups, std=0.4)
    at[..., 0] = step
    at[..., 1] = -7.5 * step + drift + torch.empty(at.shape[:-1], device="cuda").uniform_(-0.2, 0.2, generator=g)
    if bounds:
        for p0 in range(0, pages, 1024):
            k, _ = _values(c, pool[p0:p0 + 1024, :, :tiles])
            ends = torch.stack([k.amin(2), k.amax(2)], dim=2).to(torch.bfloat16)
            pool[p0:p0 + 1024, :, tiles:].view(torch.bfloat16).copy_(ends.flatten(2))
    return pool


def _requests(text):
    """[rows of each request] of "4096,1*20,801"."""
    out = []
    for part in text.split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def _append_inputs(c, seed):
    g = _generator(seed)
    cpu = torch.Generator().manual_seed(int(seed) * 7919 + 13)
    lens = _requests(c["rows"])
    starts = [int(torch.randint(0, c["hi"], (1,), generator=cpu)) for _ in lens]
    T, H, kv, d = sum(lens), c["heads"], c["kv_heads"], c["dim"]
    table, pages = _tables([s + n for s, n in zip(starts, lens)], c["page"], seed, sum(-(-(c["hi"] + n) // c["page"]) for n in lens))
    positions = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).to(torch.int32).cuda()
    row_req = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(torch.int32).cuda()
    src = _normal(g, T, (H + 2 * kv) * d)
    src[:, H * d:] += _normal(g, (2 * kv) * d, std=0.7)                      # a bias: some features lie off zero
    src[:, H * d + 5::37] *= 4.0                                              # ... and some reach far
    angle = positions.double()[:, None] * 1e6 ** (-torch.arange(0, c["rot"], 2, device="cuda").double() / max(c["rot"], 1))
    return {"src": src.to(DTYPES[c["dtype"]]), "q": torch.empty((T, H * d), dtype=DTYPES[c["dtype"]], device="cuda"),
            "cos_sin": torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous(), "positions": positions, "row_req": row_req, "table": table,
            "pool": _pool(c, g, pages, c["bounds"]), "values": torch.empty((T, 2, kv, d), dtype=torch.float32, device="cuda")}


def _attend_inputs(c, seed, bounds=0):
    g = _generator(seed)
    lengths = torch.randint(c["lo"], c["hi"] + 1, (c["rows"],), generator=torch.Generator().manual_seed(int(seed) * 7919 + 13)).tolist()
    table, pages = _tables(lengths, c["page"], seed)
    q = _normal(g, c["rows"], c["heads"] * c["dim"], std=1.2, dtype=DTYPES[c["dtype"]])
    return {"q": q, "pool": _pool(c, g, pages, bounds), "table": table, "positions": torch.tensor(lengths, dtype=torch.int32).cuda() - 1,
            "longest": max(lengths), "sink": _normal(g, c["heads"], std=2.0) if c.get("sink") else None, "scale": 1.0 / math.sqrt(c["dim"]),
            "out": torch.empty_like(q)}


def _sparse_inputs(c, seed):
    s = _attend_inputs(c, seed, bounds=1)
    return s | {"pages": torch.empty((c["rows"], c["kv_heads"], c["top"]), dtype=torch.int32, device="cuda")}


def _portion_inputs(c, seed):
    g = _generator(seed)
    parts = [tuple(int(v) for v in p.split(":")) for p in c["requests"].split(",")]
    table, pages = _tables([n + start for n, start in parts], c["page"], seed)
    T = sum(n for n, _ in parts)
    q = _normal(g, T, c["heads"] * c["dim"], std=1.2, dtype=DTYPES[c["dtype"]])
    positions = torch.cat([torch.arange(start, start + n) for n, start in parts]).to(torch.int32).cuda()
    return {"q": q, "pool": _pool(c, g, pages, 0), "table": table, "positions": positions, "parts": parts, "longest": max(n + s for n, s in parts),
            "scale": 1.0 / math.sqrt(c["dim"]), "out": torch.empty_like(q)}


_INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "portion": _portion_inputs, "sparse": _sparse_inputs}


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    state["case"], state["status"] = case, torch.zeros(1, dtype=torch.int32, device="cuda")
    if own and case["kind"] == "portion":
        from beglin_b200.csrc import ops
        state["plan"] = ops.packed_plan([n for n, _ in state["parts"]], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]],
                                        page_size=case["page"], device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state)
    return _PLAIN[state["case"]["kind"]](state)


def _own_append(s):
    from beglin_b200.csrc import ops
    c = s["case"]
    ops.packed_append(s["src"], s["q"], c["heads"], c["kv_heads"], c["dim"], c["rot"], bool(c["interleaved"]), s["cos_sin"] if c["rot"] else None,
                      s["positions"], s["row_req"], s["table"], s["pool"], c["page"], s["status"])
    if c["bounds"]:
        ops.packed_bounds(s["pool"], s["positions"], s["row_req"], s["table"], c["dim"], c["page"], s["status"])
    ops.packed_rows(s["pool"], s["positions"], s["row_req"], s["table"], c["dim"], c["page"], s["values"], s["status"])
    return {"q": s["q"], "values": s["values"]} | ({"bounds": _bounds(c, s["pool"])} if c["bounds"] else {})


def _own_attend(s, **more):
    from beglin_b200.csrc import ops
    c = s["case"]
    ops.packed_attention(s["q"], s["pool"], s["table"], s["positions"], c["heads"], c["kv_heads"], c["dim"], c["page"], s["longest"] - 1, s["scale"], s["out"],
                         s["status"], **more)
    return s["out"]


def _own_alone(s):
    c = s["case"]
    return _own_attend(s, window=c["window"], softcap=c["cap"], sink_weight=s["sink"])


def _own_portion(s):
    return _own_attend(s, plan=s["plan"])


def _own_sparse(s):
    from beglin_b200.csrc import ops
    c = s["case"]
    ops.packed_select(s["q"], s["pool"], s["table"], s["positions"], c["heads"], c["kv_heads"], c["dim"], c["page"], s["longest"] - 1, s["pages"], s["status"],
                      first=c["first"], recent=c["recent"])
    return {"out": _own_attend(s, pages=s["pages"]), "pages": s["pages"]}


_OWN = {"append": _own_append, "attend": _own_alone, "portion": _own_portion, "sparse": _own_sparse}


def _bounds(c, pool):
    """The smallest and largest value of every feature of the pages' keys, [pages, kv heads, 2, features]."""
    return pool[:, :, _sizes(c)[3]:].view(torch.bfloat16).unflatten(2, (2, c["dim"]))


def _orders(c):
    """Where the codes stand: for a position's key the feature of every nibble of its bytes (the low one first), and for a tile's values the position
    times features plus feature of every nibble."""
    d, groups = c["dim"], c["dim"] // GROUP
    at = torch.arange(GROUP).view(4, 2, 4, 2)                                  # a quarter, a word, its pairs of features
    key = at.transpose(2, 3)[:, None] + GROUP * torch.arange(groups).view(1, -1, 1, 1, 1)        # quarter, group, word, odd, pair
    lane = torch.arange(32)
    pos = 2 * (lane % 4)[:, None] + torch.tensor([0, 1, 8, 9])
    value = pos[:, :, None, None] * d + (GROUP * torch.arange(groups))[:, None] + (8 * (lane // 4))[:, None, None, None] + torch.arange(8)
    if groups == 2:                                                            # lane, position, group, feature: two positions at a time
        value = value.unflatten(1, (2, 2)).transpose(0, 1)
    return key.flatten(), value.flatten()


def _nibbles(x):
    return torch.stack([x & 15, x >> 4], dim=-1).flatten(-2)


def _values(c, pages):
    """Keys and values [..., positions, features] in 32 bits of the tiles [..., bytes] of one kv head."""
    groups, codes, tile, _ = _sizes(c)
    t = pages.unflatten(-1, (-1, tile))
    key, value = (torch.argsort(o).to(pages.device) for o in _orders(c))
    k = _nibbles(t[..., :codes]).unflatten(-1, (TILE, c["dim"]))[..., key]
    v = _nibbles(t[..., codes:2 * codes])[..., value].unflatten(-1, (TILE, c["dim"]))
    pair = t[..., 2 * codes:].contiguous().view(torch.bfloat16).float().unflatten(-1, (TILE, 2, groups, 2))

    def scaled(u, p):
        return (u.unflatten(-1, (groups, GROUP)).float() * p[..., 0:1] + p[..., 1:2]).flatten(-2).flatten(-3, -2)
    return scaled(k, pair[..., 0, :, :]), scaled(v, pair[..., 1, :, :])


def _rotate(x, cos_sin, rot, interleaved):
    """Rows [T, heads, features] with their first `rot` features rotated."""
    if not rot:
        return x
    cos, sin = cos_sin[:, None, :, 0].to(x.dtype), cos_sin[:, None, :, 1].to(x.dtype)
    front = x[..., :rot]
    a, b = (front[..., 0::2], front[..., 1::2]) if interleaved else (front[..., :rot // 2], front[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    front = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([front, x[..., rot:]], dim=-1)


def _code(x):
    """Codes, steps and lowest values of rows [..., groups, 64]."""
    lowest = x.amin(-1, keepdim=True).to(torch.bfloat16).to(x.dtype)
    step = ((x.amax(-1, keepdim=True) - lowest) / 15.0).to(torch.bfloat16).to(x.dtype)
    u = torch.round((x - lowest) / torch.where(step > 0, step, torch.ones_like(step))).clamp(0, 15)
    return u.to(torch.uint8), step[..., 0], lowest[..., 0]


def _plain_append(s):
    c = s["case"]
    groups, codes, tile, tiles = _sizes(c)
    H, kv, d, T = c["heads"], c["kv_heads"], c["dim"], s["src"].shape[0]
    x = s["src"].double().view(T, H + 2 * kv, d)                              # (in 64 bits: a value next to the border of two codes gets the nearer one)
    turned = _rotate(x[:, :H + kv], s["cos_sin"], c["rot"], c["interleaved"])
    s["q"].copy_(turned[:, :H].reshape(T, H * d))
    rows = torch.stack([turned[:, H:], x[:, H + kv:]], dim=1)                  # T, keys and values, kv heads, features
    u, step, lowest = _code(rows.unflatten(-1, (groups, GROUP)))
    u = u.flatten(-2)
    pos = s["positions"].long()
    page = s["table"][s["row_req"].long(), pos // c["page"]].long()
    at, slot = pos % c["page"] // TILE * tile, pos % TILE
    key, value = (o.to(pos.device) for o in _orders(c))
    heads = torch.arange(kv, device=pos.device)[None, :, None]

    def put(offset, data):
        s["pool"][page[:, None, None], heads, offset[:, None, :]] = data

    pair = u[:, 0][..., key].unflatten(-1, (-1, 2))
    put((at + slot * (d // 2))[:, None] + torch.arange(d // 2, device=pos.device), pair[..., 0] | pair[..., 1] << 4)
    place = torch.argsort(value).view(TILE, d)[slot]                          # the nibble of every feature of a row's value
    pair = u[:, 1].unflatten(-1, (-1, 2))
    put((at + codes)[:, None] + place[:, 0::2] // 2, pair[..., 0] | pair[..., 1] << 4)
    both = torch.stack([step, lowest], dim=-1).to(torch.bfloat16).transpose(1, 2).flatten(2).contiguous().view(torch.uint8)
    put((at + 2 * codes + slot * 8 * groups)[:, None] + torch.arange(8 * groups, device=pos.device), both)
    if c["bounds"]:
        full = page[pos % c["page"] == c["page"] - 1]
        k, _ = _values(c, s["pool"][full][:, :, :tiles])
        _bounds(c, s["pool"])[full] = torch.stack([k.amin(2), k.amax(2)], dim=2).to(torch.bfloat16)
    one = s["pool"][page[:, None], torch.arange(kv, device=pos.device)[None], :tiles].unflatten(-1, (-1, tile))
    k, v = _values(c, one[torch.arange(T, device=pos.device), :, pos % c["page"] // TILE])
    every = torch.arange(T, device=pos.device)
    s["values"].copy_(torch.stack([k[every, :, slot], v[every, :, slot]], dim=1))
    return {"q": s["q"], "values": s["values"]} | ({"bounds": _bounds(c, s["pool"])} if c["bounds"] else {})


def _weigh(q, k, v, ok, scale, cap=0.0, sink=None):
    """Queries [..., m, d] over keys [..., n, d] that `ok` [..., 1 or m, n] lets them see; a learned score that has no value joins the sum."""
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    if cap > 0.0:
        x = cap * torch.tanh(x / cap)
    x = torch.where(ok, x, torch.full_like(x, -math.inf))
    m = x.amax(-1, keepdim=True)
    if sink is not None:
        m = torch.maximum(m, sink)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - m)
    return torch.matmul(p, v) / total


def _gathered(c, s, pages):
    """Keys and values [rows, kv heads, positions, features] of the page indexes [rows, kv heads, pages] of each row's request."""
    rows, heads = torch.arange(pages.shape[0], device=pages.device), torch.arange(c["kv_heads"], device=pages.device)
    real = s["table"][rows[:, None, None], pages].long().clamp(min=0)
    return _values(c, s["pool"][real, heads[None, :, None]][..., :_sizes(c)[3]].flatten(2))


def _plain_attend(s):
    c = s["case"]
    R, kv, H, d, pos = c["rows"], c["kv_heads"], c["heads"], c["dim"], s["positions"].long()
    n = -(-s["longest"] // c["page"])
    k, v = _gathered(c, s, torch.arange(n, device=pos.device).expand(R, kv, n))
    at = torch.arange(n * c["page"], device=pos.device)
    ok = at <= pos[:, None]
    if c["window"]:
        ok = ok & (at > pos[:, None] - c["window"])
    sink = None if s["sink"] is None else s["sink"].view(kv, -1, 1)
    s["out"].copy_(_weigh(s["q"].float().view(R, kv, -1, d), k, v, ok[:, None, None], s["scale"], c["cap"], sink).reshape(R, -1))
    return s["out"]


def _plain_portion(s):
    c, row = s["case"], 0
    kv, d = c["kv_heads"], c["dim"]
    for i, (n, start) in enumerate(s["parts"]):                                # a request at a time: the scores of all together take too much room
        pages = s["table"][i, :-(-(start + n) // c["page"])].long()
        k, v = _values(c, s["pool"][pages][..., :_sizes(c)[3]])
        k, v = (t.transpose(0, 1).flatten(1, 2)[:, None, :start + n] for t in (k, v))
        q = s["q"][row:row + n].float().view(n, kv, -1, d).permute(1, 2, 0, 3)
        ok = torch.arange(start + n, device=q.device) <= torch.arange(start, start + n, device=q.device)[:, None]
        s["out"][row:row + n] = _weigh(q, k, v, ok, s["scale"]).permute(2, 0, 1, 3).reshape(n, -1)
        row += n
    return s["out"]


def _plain_sparse(s):
    c = s["case"]
    R, kv, d, top, pos = c["rows"], c["kv_heads"], c["dim"], c["top"], s["positions"].long()
    n = max(top, -(-s["longest"] // c["page"]))
    index = torch.arange(n, device=pos.device)
    table = torch.nn.functional.pad(s["table"], (0, max(0, n - s["table"].shape[1])), value=-1)[:, :n].long().clamp(min=0)
    ends = _bounds(c, s["pool"])[table].double().permute(3, 0, 2, 4, 1)        # smallest and largest, row, kv head, feature, page
    q = s["q"].double().view(R, kv, -1, d)
    # (in 64 bits, where the sums are exact: pages whose scores lie side by side come out in one order)
    score = (torch.matmul(q.clamp(max=0.0), ends[0]) + torch.matmul(q.clamp(min=0.0), ends[1])).float().amax(2)
    last = (pos // c["page"])[:, None, None]
    always = (index < c["first"]) | (index > last - c["recent"])
    score = torch.where(always, torch.full_like(score, math.inf), score)
    score = torch.where(index <= last, score, torch.full_like(score, -math.inf))
    pick = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    pick = torch.where(pick <= last, pick, n).sort(-1).values
    s["pages"].copy_(torch.where(pick < n, pick, -1))
    k, v = _gathered(c, s | {"table": torch.nn.functional.pad(table, (0, 1))}, pick)
    at = (pick[..., None] * c["page"] + torch.arange(c["page"], device=pos.device)).flatten(2)
    ok = at <= pos[:, None, None]
    s["out"].copy_(_weigh(q.float(), k, v, ok[:, :, None], s["scale"]).reshape(R, -1))
    return {"out": s["out"], "pages": s["pages"]}


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "portion": _plain_portion, "sparse": _plain_sparse}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    H, kv, d, size = c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]].itemsize
    held = kv * _sizes(c)[2] / TILE                                            # bytes that the cache holds of a position
    if c["kind"] == "append":
        lens = _requests(c["rows"])
        T = sum(lens)
        ends = sum(n / c["page"] for n in lens) * 4 * kv * d if c["bounds"] else 0
        return {"bytes": int(T * ((H + 2 * kv) * d * size + H * d * size + held + 8 * kv * d + 4 * c["rot"]) + ends), "flops": int(T * (6 * (H + kv) + 8 * kv) * d)}
    if c["kind"] == "portion":
        parts = [tuple(int(v) for v in p.split(":")) for p in c["requests"].split(",")]
        pairs = sum(n * start + n * (n + 1) // 2 for n, start in parts)
        return {"bytes": int(sum(n + s for n, s in parts) * held + 2 * sum(n for n, _ in parts) * H * d * size), "flops": int(4 * pairs * H * d)}
    mean = (c["lo"] + c["hi"]) / 2
    if c["kind"] == "attend":
        read = c["rows"] * (min(mean, c["window"]) if c["window"] else mean)
        return {"bytes": int(read * held + 2 * c["rows"] * H * d * size), "flops": int(4 * read * H * d)}
    read, pages = c["rows"] * min(mean, c["top"] * c["page"]), c["rows"] * mean / c["page"]
    return {"bytes": int(read * held + pages * 4 * kv * d + c["rows"] * (2 * H * d * size + 4 * kv * c["top"])), "flops": int(4 * read * H * d + 2 * pages * H * d)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](case, _INPUTS[case["kind"]](case, seed))


def _held(c, pool, page, head, slot):
    """Key and value [n, features] in 64 bits of positions `slot` of pages `page`, one by one from where their codes stand."""
    groups, codes, tile, _ = _sizes(c)
    f = torch.arange(c["dim"], device=pool.device)
    group, r = f // GROUP, f % GROUP
    base, p = (slot // TILE * tile)[:, None], (slot % TILE)[:, None]
    nib = r % 8 // 2 + 4 * (r % 2)
    key = base + p * (c["dim"] // 2) + (r // 16 * groups + group) * 8 + r % 16 // 8 * 4 + nib // 2
    lane = r // 8 * 4 + p % 8 // 2
    if groups == 2:
        value = base + codes + p // 8 * 512 + lane * 16 + p % 2 * 8 + group * 4 + r % 8 // 2
    else:
        value = base + codes + lane * 16 + (p // 8 * 2 + p % 2) * 4 + r % 8 // 2
    out = []
    for kind, (at, shift) in enumerate(((key, nib % 2 * 4), (value, r % 2 * 4))):
        u = pool[page[:, None], head, at].int() >> shift & 15
        pair = (base + 2 * codes + p * 8 * groups + (kind * groups + group) * 4)[..., None] + torch.arange(4, device=pool.device)
        pair = pool[page[:, None, None], head, pair].view(torch.bfloat16).double()
        out.append(pair[..., 1] + pair[..., 0] * u.double())
    return out


def _softmaxed(q, k, v, scale, cap=0.0, sink=None):
    score = q @ k.T * scale
    if cap > 0.0:
        score = cap * torch.tanh(score / cap)
    if sink is not None:
        score = torch.cat([score, sink[:, None]], dim=1)
    return torch.softmax(score, dim=1)[:, :k.shape[0]] @ v


def _exact_append(c, s):
    H, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["src"].double().view(-1, H + 2 * kv, d).clone()
    half = c["rot"] // 2
    i = torch.arange(half, device=x.device)
    one, two = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    cos, sin = s["cos_sin"].double()[:, None, :, 0], s["cos_sin"].double()[:, None, :, 1]
    a, b = x[:, :H + kv, one], x[:, :H + kv, two]
    if half:
        x[:, :H + kv, one], x[:, :H + kv, two] = a * cos - b * sin, a * sin + b * cos
    result = torch.empty((x.shape[0], 2, kv, d), dtype=torch.float64, device=x.device)
    for g in range(d // GROUP):
        part = torch.stack([x[:, H:H + kv], x[:, H + kv:]], dim=1)[..., g * GROUP:(g + 1) * GROUP]
        lowest = part.min(-1, keepdim=True).values.to(torch.bfloat16).double()
        step = ((part.max(-1, keepdim=True).values - lowest) / 15).to(torch.bfloat16).double()
        u = ((part - lowest) / step.clamp(min=1e-300)).round().clamp(0, 15)
        result[..., g * GROUP:(g + 1) * GROUP] = lowest + step * u
    # (a page's bounds take in positions that the pages held before: their values are compared with the plain form's alone)
    return {"q": x[:, :H].reshape(x.shape[0], -1), "values": result} | ({"bounds": None} if c["bounds"] else {})


def _exact_attend(c, s, pick=None):
    H, kv, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    result = torch.empty((c["rows"], H, d), dtype=torch.float64, device="cuda")
    per = H // kv
    for r, last in enumerate(s["positions"].tolist()):
        for h in range(kv):
            if pick is None:
                at = torch.arange(max(0, last + 1 - c["window"]) if c["window"] else 0, last + 1, device="cuda")
            else:
                at = (pick[r][h][:, None] * ps + torch.arange(ps, device="cuda")).flatten()
                at = at[at <= last]
            k, v = _held(c, s["pool"], s["table"][r].long()[at // ps], h, at % ps)
            heads = slice(h * per, (h + 1) * per)
            result[r, heads] = _softmaxed(s["q"][r].double().view(H, d)[heads], k, v, s["scale"], c.get("cap", 0.0),
                                          None if s["sink"] is None else s["sink"].double()[heads])
    return result.view(c["rows"], -1)


def _exact_portion(c, s):
    H, kv, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    result, row = torch.empty((s["q"].shape[0], H, d), dtype=torch.float64, device="cuda"), 0
    for i, (n, start) in enumerate(s["parts"]):
        at = torch.arange(start + n, device="cuda")
        later = at[None] > torch.arange(start, start + n, device="cuda")[:, None]
        for h in range(H):
            if h % (H // kv) == 0:
                k, v = _held(c, s["pool"], s["table"][i].long()[at // ps], h // (H // kv), at % ps)
            score = (s["q"][row:row + n, h * d:(h + 1) * d].double() @ k.T * s["scale"]).masked_fill_(later, -math.inf)
            result[row:row + n, h] = torch.softmax(score, dim=1) @ v
        row += n
    return result.view(-1, H * d)


def _exact_sparse(c, s):
    """Page by page from the definition: the score of a page is the largest, over the heads that share it, of the most that q k can be."""
    kv, d, top = c["kv_heads"], c["dim"], c["top"]
    listed_pages = torch.full((c["rows"], kv, top), -1, dtype=torch.int32, device="cuda")
    picks = []
    for r, last in enumerate((s["positions"] // c["page"]).tolist()):
        picks.append([])
        for h in range(kv):
            index = torch.arange(last + 1, device="cuda")
            if last + 1 > top:
                ends = _bounds(c, s["pool"])[s["table"][r, :last + 1].long(), h].double()
                q = s["q"][r].double().view(kv, -1, d)[h]
                score = torch.stack([torch.maximum(one * ends[:, 0], one * ends[:, 1]).sum(-1) for one in q]).amax(0).float()
                middle = index[c["first"]:last + 1 - c["recent"]]
                best = middle[torch.sort(score[middle], descending=True, stable=True).indices[:top - c["first"] - c["recent"]]]
                index = torch.cat([index[:c["first"]], best, index[last + 1 - c["recent"]:]]).sort().values
            picks[r].append(index)
            listed_pages[r, h, :index.numel()] = index.int()
    return {"out": _exact_attend(c, s, picks), "pages": listed_pages}


_EXACT = {"append": _exact_append, "attend": _exact_attend, "portion": _exact_portion, "sparse": _exact_sparse}
