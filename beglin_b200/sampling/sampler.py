"""Choosing the next token from a row of logits.

Greedy is the reference's only sampler: the index of the first maximum (qwen_infer.c:2152-2155).
Temperature sampling is added: p = softmax(logits / T) in float, inverted in index order at a
uniform number u.  u comes from a counter-based generator keyed by (seed, request, number of tokens
the request has generated), so a request's draws do not depend on what else is in its batch or on
how its steps were cut.  T = 0 means greedy.
"""
from __future__ import annotations

import zlib
from dataclasses import dataclass
from typing import Hashable, List, Optional, Sequence

import numpy as np
import torch

from ..csrc import ops
from .rules import RuleTables

_MASK = (1 << 64) - 1


def _splitmix64(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    z = x
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    return z ^ (z >> 31)


def request_key(rid: Hashable) -> int:
    if isinstance(rid, int) and not isinstance(rid, bool):
        return rid & _MASK
    return zlib.crc32(repr(rid).encode())


def uniform(seed: int, rid: Hashable, step: int) -> float:
    """A number in [0, 1) with 24 random bits, a pure function of its three arguments."""
    z = _splitmix64(seed & _MASK)
    z = _splitmix64(z ^ request_key(rid))
    z = _splitmix64(z ^ (step & _MASK))
    return (z >> 40) / float(1 << 24)


@dataclass
class SamplingParams:
    temperature: float = 0.0
    seed: int = 0


class Sampler:
    def __init__(self, device, status: Optional[torch.Tensor] = None):
        """`status`: the word in which kernels record what is wrong, for whoever looks at it (`ops.raise_on_status`); without one `sample` looks itself."""
        self.device, self.status = torch.device(device), status

    def sample(self, logits: torch.Tensor, temperatures: Sequence[float], uniforms: Sequence[float], rules: Optional[Sequence] = None) -> List[int]:
        """One token per row of float logits [n, V]; rows with temperature <= 0 are greedy.  `rules`: (LogitRules or None, prompt, generated tokens) of every row;
        the logits are changed by them."""
        n = logits.shape[0]
        if rules is not None and any(r is not None and not r.plain for r, _, _ in rules):
            lengths = [len(prompt) + len(made) for _, prompt, made in rules]
            tables = RuleTables(n, logits.shape[1], max(lengths), logits.device)
            tables.load(rules)
            tables.load_masks(rules)
            status = self.status if self.status is not None else ops.new_status(logits.device)
            tables.apply(logits, torch.tensor(lengths, dtype=torch.int32).to(logits.device), None, status, tables.masked)
            if self.status is None:
                ops.raise_on_status(status)
        out = torch.empty(n, dtype=torch.int32, device=logits.device)
        if any(t > 0.0 for t in temperatures):
            t = torch.from_numpy(np.asarray(temperatures, dtype=np.float32)).to(logits.device)
            u = torch.from_numpy(np.asarray(uniforms, dtype=np.float32)).to(logits.device)
            ops.sample(logits, t, u, out)
        else:
            ops.sample(logits, None, None, out)
        return out.tolist()

    def greedy(self, logits: torch.Tensor) -> torch.Tensor:
        """Device int32 [n]: the first maximum of every row, without a host round trip."""
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
        ops.sample(logits, None, None, out)
        return out
