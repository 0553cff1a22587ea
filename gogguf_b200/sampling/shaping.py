"""What is done to a row's logits before an id is drawn: penalties for ids that repeat, biases, and the ids that a grammar
allows.  With c the number of times id v stands among a sequence's last `last_n` ids (prompt included):

    z = x_v ; where c > 0: z = z / repeat (z > 0) or z * repeat, then z -= frequency c + presence
    z += bias of v ; where the grammar does not allow v: z = -inf

The repeat penalty is the reference's (pkg/sampler/penalties.go:5-32), which has none of the others.  On the device all of it is
one kernel (`csrc.kernels.shape_logits`) over the state that `ShapingState` keeps there, so that the loop stays a step ahead of
the host; `shape_host` is the same on one row in numpy."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .grammar import TokenGrammar


def _finite(x: float) -> bool:
    """Is x a finite number, and does it stay one in 32 bits?"""
    return abs(x) <= float(np.finfo(np.float32).max)


@dataclass(frozen=True)
class LogitShaping:
    repeat: float
    last_n: int
    frequency: float
    presence: float
    bias: Tuple[Tuple[int, float], ...]
    grammar: Optional[TokenGrammar]

    @classmethod
    def of(cls, params, vocab_size: int) -> Optional["LogitShaping"]:
        """What a request's parameters ask for beyond the repeat penalty alone, or None."""
        frequency, presence = float(params.frequency_penalty), float(params.presence_penalty)
        if not (_finite(frequency) and _finite(presence)):
            raise ValueError("frequency_penalty and presence_penalty must be finite (as float32 numbers)")
        bias = []
        for t, b in (params.logit_bias or {}).items():
            b = float(b)
            if not 0 <= int(t) < vocab_size or int(t) != t:
                raise ValueError(f"logit_bias: id {t} is outside the vocabulary (0..{vocab_size - 1})")
            if math.isnan(b) or b == math.inf or not (b == -math.inf or _finite(b)):
                raise ValueError(f"logit_bias: {b} for id {t} is not a number that a logit takes")
            if b != 0:
                bias.append((int(t), b))
        grammar = params.grammar
        if grammar is not None and grammar.vocab_size != vocab_size:
            raise ValueError(f"the grammar is over {grammar.vocab_size} ids, the model's vocabulary has {vocab_size}")
        if frequency == 0 and presence == 0 and not bias and grammar is None:
            return None
        repeat = float(params.repeat_penalty)
        if repeat > 0 and not (_finite(repeat) and np.float32(repeat) > 0):
            raise ValueError("repeat_penalty must be finite and no less than 2^-149 (as a float32 number)")
        return cls(repeat if repeat > 0 else 1.0, int(params.repeat_last_n) if params.repeat_last_n else 64, frequency, presence,
                   tuple(sorted(bias)), grammar)

    @property
    def counts(self) -> bool:
        """Do the last ids matter?"""
        return self.repeat != 1 or self.frequency != 0 or self.presence != 0

    def window(self, history: Sequence[int]) -> Sequence[int]:
        return history[-self.last_n:] if 0 < self.last_n < len(history) else history

    def state_of(self, generated: Sequence[int]) -> int:
        return self.grammar.walk(generated) if self.grammar is not None else -1


class GrammarWalks:
    """The states of a sampler's rows, from one step to the next: where a stream's ids begin with those of its last step, only what
    came after them is walked."""

    def __init__(self, grammar: Optional[TokenGrammar]):
        self.grammar = grammar
        self._at: Dict[int, Tuple[List[int], int]] = {}          # stream -> (the ids walked, the state behind them)

    def states(self, streams: Sequence[int], made: Sequence[List[int]]) -> List[int]:
        """A state per row (-1 without a grammar, or where the row has left it)."""
        if self.grammar is None:
            return [-1] * len(made)
        was, self._at, out = self._at, {}, []
        for stream, ids in zip(streams, made):
            known, state = was.get(stream, ([], self.grammar.start))
            if ids[:len(known)] != known:
                known, state = [], self.grammar.start
            state = self.grammar.walk(ids[len(known):], state)
            self._at[stream] = (ids, state)
            out.append(state)
        return out

    def keep(self, states: Sequence[int], tokens: Sequence[int]) -> List[int]:
        """`tokens` drawn in `states`, -1 in the place of one that is not allowed."""
        if self.grammar is None:
            return list(tokens)
        return [t if self.grammar.step(s, int(t)) >= 0 else -1 for s, t in zip(states, tokens)]


def shape_host(row: np.ndarray, shaping: LogitShaping, history: Sequence[int], generated: Sequence[int], state: Optional[int] = None) -> None:
    """One row of float32 logits, in place; `history` is prompt and generated ids; `state`: the grammar's behind `generated`, where it is
    known."""
    if shaping.counts:
        ids, times = np.unique(np.asarray(list(shaping.window(history)), dtype=np.int64), return_counts=True)
        inside = (ids >= 0) & (ids < row.size)
        ids, times = ids[inside], times[inside].astype(np.float32)
        z = row[ids]
        if shaping.repeat != 1:
            z = np.where(z > 0, z / np.float32(shaping.repeat), z * np.float32(shaping.repeat))
        row[ids] = z - (np.float32(shaping.frequency) * times + np.float32(shaping.presence))
    for t, b in shaping.bias:
        row[t] += np.float32(b)
    if shaping.grammar is not None:
        row[~shaping.grammar.allowed(shaping.state_of(generated) if state is None else state)] = -np.inf


class ShapingState:
    """The requests' last ids, biases and grammar states on the device."""

    @staticmethod
    def advances(shaping: LogitShaping) -> bool:
        """Can a state follow the drawn ids on the device?  Not where the window has no end."""
        return shaping.last_n > 0 or not shaping.counts

    def __init__(self, shaping: LogitShaping, histories: Sequence[Sequence[int]], generated: Sequence[Sequence[int]], device,
                 most: Optional[int] = 0, states: Optional[Sequence[int]] = None, bias=None):
        """`most`: ids that may still join a request's history by `advance` (0: the state is made for a step; None: any number);
        `states`: the grammar's behind `generated`, where they are known; `bias`: that of a state for as many requests."""
        self.shaping = shaping
        # (a window is no longer than what it can hold, and one below one is the whole history)
        rows, n = len(histories), shaping.last_n
        if n < 1 or most is not None:
            held = max([1] + [len(h) + (most or 0) for h in histories])
            n = held if n < 1 else min(n, held)
        self.hist = self.hist_len = self.hist_pos = None
        if shaping.counts:
            hist = np.full((rows, n), -1, dtype=np.int32)
            lens = np.zeros(rows, dtype=np.int32)
            for r, h in enumerate(histories):
                tail = list(shaping.window(h))
                hist[r, :len(tail)] = tail
                lens[r] = len(tail)
            self.hist, self.hist_len, self.hist_pos = (torch.from_numpy(a).to(device) for a in (hist, lens, lens % n))
        self.bias = bias
        if shaping.bias and bias is None:
            nb = len(shaping.bias)
            ids, values = zip(*shaping.bias)
            self.bias = (torch.arange(rows + 1, dtype=torch.int32, device=device) * nb,
                         torch.tensor(ids, dtype=torch.int32, device=device).repeat(rows),
                         torch.tensor(values, dtype=torch.float32, device=device).repeat(rows))
        self.masks = self.classes = self.next = self.states = None
        if shaping.grammar is not None:
            self.masks, self.classes, self.next = shaping.grammar.on(device)
            # (a sequence that has left the grammar is where nothing is allowed: beyond the table)
            at = [shaping.state_of(g) for g in generated] if states is None else states
            self.states = torch.tensor([s if s >= 0 else shaping.grammar.states for s in at], dtype=torch.int32, device=device)

    def apply(self, logits: torch.Tensor, ring_rows: Optional[torch.Tensor], rows: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        from ..csrc import kernels as K
        s = self.shaping
        return K.shape_logits(logits, out, hist=self.hist, hist_len=self.hist_len, ring_rows=ring_rows, repeat=s.repeat, frequency=s.frequency,
                              presence=s.presence, bias=self.bias, masks=self.masks, mask_rows=self.states, rows=rows)

    def advance(self, tokens: torch.Tensor, ring_rows: torch.Tensor, rows: int) -> None:
        """tokens[r] was drawn for request ring_rows[r]: it joins the last ids and moves the grammar's state; one that the grammar
        does not allow (nothing was) becomes -1, which ends its sequence."""
        from ..csrc import kernels as K
        K.shape_advance(tokens, ring_rows, rows, hist=self.hist, hist_len=self.hist_len, hist_pos=self.hist_pos, states=self.states,
                        classes=self.classes, next=self.next)
