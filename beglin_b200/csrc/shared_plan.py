"""How the attention of a step of single tokens is cut where requests share their first positions: what a CTA takes, as the lists that the kernels read.
Pure host code on numpy, tested without a GPU; `shared` is a `cache.shared.SharedPrefix`.
"""
from __future__ import annotations

from typing import Sequence, Tuple

import numpy as np

MOST = 0x7fffffff
TILE = 64                  # positions of a tile of the tensor-core kernel: ranges begin on whole tiles


def shared_blocks(shared, bq: int, split: int, room: int):
    """For kernels whose splits lie at multiples of `split`: (blocks int32 [room, 8], rows int32 [2 n]).  Up to `bq` rows of a group take the
    group's whole splits together; every row takes the splits behind them by itself."""
    n = shared.n_rows
    rows = np.arange(2 * n, dtype=np.int32) % max(n, 1)
    first, blocks, at = np.zeros(n, dtype=np.int32), [], 0
    for group, positions in shared.groups:
        whole = positions // split
        rows[at:at + len(group)] = group
        if whole > 0:
            first[list(group)] = whole
            for b in range(0, len(group), bq):
                blocks.append((group[0], at + b, min(bq, len(group) - b), 0, whole, whole * split - 1, 0, 0))
        at += len(group)
    blocks += [(r, n + r, 1, int(first[r]), MOST, MOST, 0, 0) for r in range(n)]
    if len(blocks) > room:
        raise ValueError(f"{len(blocks)} blocks, room for {room}")
    out = np.zeros((room, 8), dtype=np.int32)
    out[:len(blocks)] = blocks
    return out, rows


def blocks_room(n_rows: int) -> int:
    """The most blocks that `shared_blocks` makes of n rows (a group has two rows at least)."""
    return n_rows + n_rows // 2 + 1 if n_rows > 1 else 1


# What a range costs beside its positions, in positions: measured as the time of a CTA that takes one tile.
RANGE_COST = 320


def range_length(tiles: Sequence[Tuple[int, int]], nkv: int, sms: int, most: int) -> int:
    """Positions of a range, a multiple of TILE, for blocks of rows `tiles` = [(blocks, positions of their group)]: the length for which the CTAs, `sms` of
    them at once, are done first, each taking its positions and RANGE_COST.  No more than `most` ranges a group."""
    longest = max(p for _, p in tiles)
    best, best_cost = None, None
    floor = -(-longest // most)
    for n in range(1, most + 1):
        length = -(-max(-(-longest // n), TILE) // TILE) * TILE
        if length < floor:
            break
        ctas = nkv * sum(b * -(-p // length) for b, p in tiles)
        cost = -(-ctas // sms) * (length + RANGE_COST)
        if best is None or cost < best_cost:
            best, best_cost = length, cost
    return best


def shared_items(shared, bq: int, nkv: int, sms: int, room: int, most: int):
    """For the tensor-core kernel: (items int32 [room, 8], rows int32 [n], first position of its own of every row int32 [n], results of every row over what it
    shares int32 [n]).  A group's rows are cut into blocks of `bq`, its positions into ranges of one length for all groups."""
    n = shared.n_rows
    rows, first, parts = np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.int32)
    items, at = [], 0
    if shared.groups:
        tiles = [(-(-len(g) // bq), p) for g, p in shared.groups]
        length = range_length(tiles, nkv, sms, min(most, max(1, room // sum(b for b, _ in tiles))))
        for group, positions in shared.groups:
            rows[at:at + len(group)] = group
            first[list(group)] = positions
            ranges = -(-positions // length)
            parts[list(group)] = ranges
            for b in range(0, len(group), bq):
                items += [(group[0], at + b, min(bq, len(group) - b), s * length, min(positions, (s + 1) * length), s, 0, 0) for s in range(ranges)]
            at += len(group)
    if len(items) > room:
        raise ValueError(f"{len(items)} items, room for {room}")
    out = np.zeros((room, 8), dtype=np.int32)
    out[:len(items)] = np.asarray(items, dtype=np.int32).reshape(-1, 8)
    return out, rows, first, parts


def items_room(n_rows: int, bq: int, nkv: int, sms: int) -> int:
    """Room for the items of any groups of n rows: two waves of CTAs, or a range for every block."""
    return max(-(-2 * sms // nkv), n_rows // 2 + 1)
