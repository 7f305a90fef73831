"""Which rows of a step of single tokens share the first positions of their requests (requests that go on from one text hold its pages together,
`CacheManager.fork`)."""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple


class SharedPrefix:
    """`groups` = [(rows, positions)]: the requests of these rows (row r is request r) hold their first `positions` positions in the same pages.
    A row is in one group at most; a row in none shares nothing.  `lengths`: about how many positions every row's request holds in all, which whether
    sharing pays hangs on (None: not known); prefixes of the same groups are equal whatever their lengths."""

    def __init__(self, n_rows: int, groups: Sequence[Tuple[Sequence[int], int]], lengths: Optional[Sequence[int]] = None):
        self.n_rows = int(n_rows)
        self.lengths = None if lengths is None else tuple(int(n) for n in lengths)
        if self.lengths is not None and (len(self.lengths) != self.n_rows or min(self.lengths, default=0) < 0):
            raise ValueError(f"{self.n_rows} rows have as many lengths, none of them negative")
        self.groups: List[Tuple[Tuple[int, ...], int]] = []
        seen = set()
        for rows, positions in groups:
            rows, positions = tuple(int(r) for r in rows), int(positions)
            if positions < 0:
                raise ValueError(f"a group shares {positions} positions")
            for r in rows:
                if not 0 <= r < self.n_rows:
                    raise ValueError(f"row {r} is outside the {self.n_rows} rows")
                if r in seen:
                    raise ValueError(f"row {r} is named twice")
                seen.add(r)
            if len(rows) > 1 and positions > 0:
                self.groups.append((rows, positions))

    def key(self) -> tuple:
        return self.n_rows, tuple(self.groups)

    def __eq__(self, other) -> bool:
        return isinstance(other, SharedPrefix) and self.key() == other.key()

    def __hash__(self) -> int:
        return hash(self.key())

    def most_shared(self) -> int:
        return max((p for _, p in self.groups), default=0)
