"""What a request may ask of the choice of its tokens: penalties for tokens that it holds already, biases of single tokens, and a mask of the tokens that
may come next (a grammar's, say), on the logits before the sampler sees them.

With x a token's logit: where the token occurs in the request's text, x / `repetition` if x > 0, else x `repetition`; where it occurs among the generated
tokens, c times, x - `frequency` c - `presence`; then x + `bias`; and -inf where `allowed` leaves it out.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Callable, List, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch

from ..csrc import ops


MOST_BIASES = 512          # biased tokens of a request


class Biases(dict):
    """Token -> bias, as given: replayed steps keep what they have loaded for as long as the rules are the same."""

    def _stay(self, *args, **kw):
        raise TypeError("the biases of rules stay as they are: make new rules")

    __setitem__ = __delitem__ = __ior__ = update = pop = popitem = clear = setdefault = _stay

    def __reduce__(self):
        return Biases, (dict(self),)


@dataclass(frozen=True)
class LogitRules:
    """`allowed` is called before every token with the tokens that the request has generated so far and returns which may come next: token ids, truth
    values [vocab] (a bool array), those packed as bits already (a uint32 array: bit v % 32 of word v / 32 is token v's), or None for all."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: Mapping[int, float] = field(default_factory=dict)
    allowed: Optional[Callable[[Sequence[int]], Optional[Sequence[int]]]] = None

    def __post_init__(self):
        object.__setattr__(self, "bias", Biases(self.bias))    # (the caller's own may change)

    def check(self, vocab: int) -> None:
        if not (self.repetition > 0.0 and math.isfinite(self.repetition)):
            raise ValueError(f"repetition={self.repetition} must be positive and finite (1: none)")
        if not (math.isfinite(self.frequency) and math.isfinite(self.presence)):
            raise ValueError(f"frequency={self.frequency} and presence={self.presence} must be finite")
        if len(self.bias) > MOST_BIASES:
            raise ValueError(f"{len(self.bias)} biased tokens, at most {MOST_BIASES}")
        for token, value in self.bias.items():
            if not 0 <= int(token) < vocab:
                raise ValueError(f"biased token {token} is outside the vocabulary [0, {vocab})")
            if math.isnan(value):
                raise ValueError(f"the bias of token {token} is not a number")

    @property
    def plain(self) -> bool:
        """Whether the logits stay as they are."""
        return self.repetition == 1.0 and self.frequency == 0.0 and self.presence == 0.0 and not self.bias and self.allowed is None

    def mask(self, generated: Sequence[int], vocab: int) -> Optional[np.ndarray]:
        """The tokens that may come next, packed: int32 words, bit v % 32 of word v / 32; or None."""
        if self.allowed is None:
            return None
        given = self.allowed(list(generated))
        if given is None:
            return None
        given = np.asarray(given)
        if given.dtype == np.uint32:
            if given.shape != (-(-vocab // 32),):
                raise ValueError(f"allowed: packed bits of {given.shape}, expected ({-(-vocab // 32)},)")
            words = np.ascontiguousarray(given)
            if not (words[:-1].any() or int(words[-1]) & ((1 << (vocab - 1) % 32 + 1) - 1)):
                raise ValueError("allowed: no token may come next")
            return words.view(np.int32)
        if given.dtype == np.bool_:
            if given.shape != (vocab,):
                raise ValueError(f"allowed: truth values of {given.shape}, expected ({vocab},)")
            bits = given
        else:
            if given.size and given.dtype.kind not in "iu":
                raise ValueError(f"allowed: token ids are whole numbers, got {given.dtype}")
            ids = given.astype(np.int64).reshape(-1)
            if ids.size and (ids.min() < 0 or ids.max() >= vocab):
                raise ValueError(f"allowed: token {int(ids[(ids < 0) | (ids >= vocab)][0])} is outside the vocabulary [0, {vocab})")
            bits = np.zeros(vocab, dtype=np.bool_)
            bits[ids] = True
        if not bits.any():
            raise ValueError("allowed: no token may come next")
        packed = np.zeros(-(-vocab // 32) * 4, dtype=np.uint8)
        packed[:-(-vocab // 8)] = np.packbits(bits, bitorder="little")
        return packed.view(np.int32)


# One row of a step: a request's rules, its prompt and the tokens that it has generated so far.
RuledRow = Tuple[Optional[LogitRules], Sequence[int], Sequence[int]]


class RuleTables:
    """The rules of a step's rows on the device, as `ops.adjust_logits` reads them.  Of a fixed number of rows and with room for `room` tokens of text each, so
    that a captured step reads them too; the newest token of every row is the step's input, which the kernel adds to the text."""

    def __init__(self, n: int, vocab: int, room: int, device):
        i32, f32 = dict(dtype=torch.int32, device=device), dict(dtype=torch.float32, device=device)
        self.n, self.vocab, self.room = n, vocab, room
        self.history = torch.zeros((n, max(room, 1)), **i32)
        self.prompts = torch.zeros(n, **i32)
        self.penalties = torch.zeros((3, n), **f32)
        self.bias_ids, self.bias_values, self.begins = torch.zeros(n * MOST_BIASES, **i32), torch.zeros(n * MOST_BIASES, **f32), torch.zeros(n + 1, **i32)
        self.allowed, self.allowed_row = torch.zeros((n, -(-vocab // 32)), **i32), torch.full((n,), -1, **i32)
        self._masked = False
        self._staged: List[torch.Tensor] = []

    def _copy(self, dst: torch.Tensor, src: np.ndarray) -> int:
        host = torch.from_numpy(np.ascontiguousarray(src))
        if dst.is_cuda:
            host = host.pin_memory()
            self._staged.append(host)                      # (kept while the copy may be under way)
            del self._staged[:-64]
        dst.copy_(host, non_blocking=True)
        return host.numel() * host.element_size()

    def load(self, rows: Sequence[RuledRow]) -> int:
        """The rules and texts of the step's rows; rows behind them have none.  The newest token of a text is left to the step.  Returns the bytes sent."""
        n = self.n
        prompts, pen = np.zeros(n, dtype=np.int32), np.zeros((3, n), dtype=np.float32)
        pen[0] = 1.0
        texts = [list(prompt) + list(made) for _, prompt, made in rows]
        width = max((len(t) for t in texts), default=0)
        if width > self.room:
            raise ValueError(f"a text of {width} tokens, room for {self.room}")
        history, ids, values, begins = np.zeros((len(rows), width), dtype=np.int32), [], [], [0]
        for r, ((rules, prompt, _), text) in enumerate(zip(rows, texts)):
            prompts[r] = len(prompt)
            tokens = np.asarray(text, dtype=np.int64)
            if len(text) and (tokens.min() < 0 or tokens.max() >= self.vocab):
                raise ValueError(f"row {r}: token {int(tokens[(tokens < 0) | (tokens >= self.vocab)][0])} of its text is outside the vocabulary [0, {self.vocab})")
            history[r, :len(text)] = tokens
            if rules is not None:
                rules.check(self.vocab)
                pen[:, r] = rules.repetition, rules.frequency, rules.presence
                for token in sorted(rules.bias):
                    ids.append(int(token)); values.append(float(rules.bias[token]))
            begins.append(len(ids))
        begins += [len(ids)] * (n + 1 - len(begins))
        sent = self._copy(self.prompts, prompts) + self._copy(self.penalties, pen) + self._copy(self.begins, np.asarray(begins, dtype=np.int32))
        if width:
            sent += self._copy(self.history[:len(rows), :width], history)
        if ids:
            sent += self._copy(self.bias_ids[:len(ids)], np.asarray(ids, dtype=np.int32)) + self._copy(self.bias_values[:len(ids)], np.asarray(values, dtype=np.float32))
        return sent

    def load_masks(self, rows: Sequence[RuledRow]) -> int:
        """What every row's grammar leaves for the next token.  Returns the bytes sent."""
        masks, where = [], np.full(self.n, -1, dtype=np.int32)
        for r, (rules, _, made) in enumerate(rows):
            words = None if rules is None else rules.mask(made, self.vocab)
            if words is not None:
                where[r] = len(masks)
                masks.append(words)
        if not masks and not self._masked:
            return 0
        self._masked = bool(masks)
        sent = self._copy(self.allowed_row, where)
        if masks:
            sent += self._copy(self.allowed[:len(masks)], np.stack(masks))
        return sent

    @property
    def masked(self) -> bool:
        """Whether any of the rows' grammars leaves tokens out."""
        return self._masked

    def apply(self, logits: torch.Tensor, lengths: torch.Tensor, newest: Optional[torch.Tensor], status: Optional[torch.Tensor], masked: bool) -> None:
        """The logits [n, vocab] under the rules, in place.  lengths: of the texts in front of the newest tokens."""
        ops.adjust_logits(logits, logits, history=self.history, lengths=lengths, prompts=self.prompts, newest=newest, repetition=self.penalties[0],
                          frequency=self.penalties[1], presence=self.penalties[2], bias=(self.bias_ids, self.bias_values, self.begins), allowed=self.allowed if masked else None,
                          allowed_row=self.allowed_row if masked else None, status=status)
