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


def blocks_room(n_rows: int, bq: int = 3) -> int:
    """The most blocks that `shared_blocks` makes of n rows: one for each, and those of the groups, of two rows and more: k rows in blocks of `bq` are k blocks
    where bq is 1, at most 2 k / 3 where it is 2 (three rows), and at most k / 2 else."""
    return n_rows + (n_rows if bq == 1 else 2 * n_rows // 3 if bq == 2 else n_rows // 2) + 1 if n_rows > 1 else 1


# What the tensor-core kernels take, in microseconds, measured on B200 with heads of 128 features (64 do not differ much: these are latencies).  The shared
# positions' kernel: a CTA beside its tiles, a tile of 64 positions for up to 128 rows and for up to 256; one more range is one more result to join.
CTA_US, TILE_US, PAIR_US, RANGE_US = 6.0, 0.52, 1.03, 0.05
# The rows' own positions and the joining of results behind it: the two kernels, a position in a CTA, bytes a microsecond of many CTAs, and what more it is
# where the shared positions' kernel leaves them no SMs to begin on.
BEHIND_US, OWN_POSITION_US, OWN_RATE, CROWDED_US = 0.4, 0.0135, 4.5e6, 3.6
OWN_GUESS = 256            # positions that a request is taken to hold behind those that it shares
# Every row by itself over all of its positions: beside the CTAs, beside a CTA's positions, a position (pages that several rows hold come from the L2) and
# what more it is for every page of 64 positions where pages are smaller; CTAs that come to an SM behind others begin under those.  (Against 220 steps of 2 to
# 256 rows the choices that follow from these numbers take 0.6 % longer than the better of both ways would.)
ALONE_US, ALONE_CTA_US, ALONE_POSITION_US, ALONE_PAGE_US, ALONE_BEHIND = 1.5, 4.5, 0.0058, 0.001, 0.7


def _up(n: int, unit: int) -> int:
    return -(-n // unit) * unit


def _done(ctas: int, longest: float, total: float, sms: int) -> float:
    """About when CTAs are through, the longest first."""
    return longest if ctas <= sms else max(longest, total / sms + longest / 2)


def cut_ranges(groups: Sequence[Tuple[int, int]], nkv: int, sms: int, room: int, most: int, streams: int = 0) -> Tuple[int, int, float]:
    """(rows of a block, positions of a range, microseconds) for groups = [(rows of a kv head, positions)]: blocks of 128 or of 256 rows, and ranges, a multiple
    of TILE and of one length for all groups, at most `most` a group, that are through first.  No more than `room` items.  Of the SMs those that the step's
    `streams` (rows x kv heads) have use for by themselves are left to them, where they are few (two streams an SM)."""
    longest = max(p for _, p in groups)
    left = sms - -(-streams // 2) if -(-streams // 2) <= sms // 4 else 0
    best = None
    for block in (128, 256):
        if block > 128 and all(r <= 128 for r, _ in groups):
            break
        n, last = 1, 0
        while n <= most:
            length = _up(max(-(-longest // n), TILE), TILE)
            if length != last:
                total, slowest, items = 0.0, 0.0, 0
                for r, p in groups:
                    ranges, tiles = -(-p // length), min(length, p) / TILE
                    for rows, count in ((block, r // block), (r % block, 1)):
                        if rows and count:
                            one = CTA_US + tiles * (PAIR_US if rows > 128 else TILE_US)
                            items += ranges * count
                            total += nkv * ranges * count * one
                            slowest = max(slowest, one)
                if items > room:
                    break
                done = _done(nkv * items, slowest, total, sms) + RANGE_US * -(-longest // length) + (CROWDED_US if nkv * items > left else 0.0)
                if best is None or done < best[2]:
                    best = block, length, done
            last = length
            n += 1 if n < 16 else 4
    return best or (256, _up(longest, TILE), 0.0)


def own_us(longest: int, total: int, n_rows: int, nkv: int, ranges, row_bytes: int) -> float:
    """About what the rows' own positions take behind the shared ones, `total` in all; `ranges`(streams, positions) is how a stream is cut (in whole multiples of
    256 positions)."""
    one = _up(-(-longest // ranges(n_rows * nkv, longest)), 256) * OWN_POSITION_US
    return BEHIND_US + max(total * nkv * row_bytes / OWN_RATE, one)


def alone_us(longest: int, total: int, n_rows: int, nkv: int, ranges, sms: int, row_bytes: int, page_size: int) -> float:
    """About what a step takes whose rows are read by themselves, the longest of `longest` positions, `total` in all."""
    streams, at_once = n_rows * nkv, sms * (1 if row_bytes > 256 else 3)
    cut = ranges(streams, longest)
    ctas, each = streams * cut, ALONE_POSITION_US + (ALONE_PAGE_US * 64 / page_size if page_size < 64 else 0.0)
    one = ALONE_CTA_US + _up(-(-longest // cut), 256) * each
    if ctas <= at_once:
        return ALONE_US + one
    return ALONE_US + max(one, ALONE_BEHIND * ctas / at_once * (ALONE_CTA_US + total * nkv / ctas * each) + one / 2)


def worth_sharing(shared, group_heads: int, nkv: int, sms: int, room: int, most: int, own_ranges, alone_ranges, row_bytes: int,
                  page_size: int = 64):
    """The groups of `shared` whose sharing is expected to pay, those that save most first: few rows of few positions are read from the L2 again sooner than they
    are split off and joined, and a long request beside a family is walked by fewer CTAs where its rows' own positions are cut by themselves.  A row is taken to
    hold OWN_GUESS positions behind what it shares, or what `shared.lengths` says where that is more (63 rows of 8,192 shared positions and one request of 16,384
    alone, 4 kv heads: 181 us row by row, 249 with sharing; with 2 kv heads 103 and 95).  own_ranges, alone_ranges(streams, positions): how a stream is cut with
    sharing and without; `row_bytes`: of a key and a value of one kv head."""
    order = sorted(shared.groups, key=lambda g: -(len(g[0]) - 1) * g[1])
    n, streams = shared.n_rows, shared.n_rows * nkv
    before = np.zeros(n, dtype=np.int64)
    for rows, p in order:
        before[list(rows)] = p
    own = np.full(n, OWN_GUESS) if shared.lengths is None else np.maximum(np.asarray(shared.lengths, dtype=np.int64) - before, OWN_GUESS)
    walked = before + own                      # by the rows themselves
    best, kept = alone_us(int(walked.max(initial=OWN_GUESS)), int(walked.sum()), n, nkv, alone_ranges, sms, row_bytes, page_size), 0
    for k in sorted({1, 2, len(order) // 2, len(order)} & set(range(1, len(order) + 1))):
        walked = before + own
        for rows, p in order[:k]:              # (groups that are left alone are walked by their rows)
            walked[list(rows)] -= p
        us = own_us(int(walked.max()), int(walked.sum()), n, nkv, own_ranges, row_bytes)
        us += cut_ranges([(len(g) * group_heads, p) for g, p in order[:k]], nkv, sms, room, most, streams)[2]
        if us < best:
            best, kept = us, k
    return order[:kept]


def shared_items(shared, group_heads: int, nkv: int, sms: int, room: int, most: int):
    """For the tensor-core kernel: (items int32 [room, 8], rows int32 [n], first position of its own of every row int32 [n], results of every row over what it
    shares int32 [n]).  A group's rows (requests x query heads of a kv head) are cut into blocks, its positions into ranges."""
    n = shared.n_rows
    rows, first, parts = np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.int32)
    items, at = [], 0
    if shared.groups:
        block, length, _ = cut_ranges([(len(g) * group_heads, p) for g, p in shared.groups], nkv, sms, room, most, n * nkv)
        for group, positions in shared.groups:
            rows[at:at + len(group)] = group
            first[list(group)] = positions
            ranges, count = -(-positions // length), len(group) * group_heads
            parts[list(group)] = ranges
            for b in range(0, count, block):
                items += [(group[0], at * group_heads + b, min(block, count - b), s * length, min(positions, (s + 1) * length), s, 0, 0) for s in range(ranges)]
            at += len(group)
    if len(items) > room:
        raise ValueError(f"{len(items)} items, room for {room}")
    # those that take longest come first (they are begun in this order)
    items.sort(key=lambda i: -(i[4] - i[3]) * (2 if i[2] > 128 else 1))
    out = np.zeros((room, 8), dtype=np.int32)
    out[:len(items)] = np.asarray(items, dtype=np.int32).reshape(-1, 8)
    return out, rows, first, parts


def items_room(n_rows: int, group_heads: int, nkv: int, sms: int, fixed: bool = False) -> int:
    """Room for the items of any groups of n rows: three waves of CTAs (one, where the launch always has as many), or a range for every block of every group
    (a group has two rows at least)."""
    return max(-(-(1 if fixed else 3) * sms // nkv), n_rows // 2 + -(-n_rows * group_heads // 256) + 1)
