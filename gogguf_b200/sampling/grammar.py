"""Which ids a sequence may go on with: a deterministic automaton over token ids.

The ids are sorted into classes, and a table says which state follows a state and a class (-1: such an id is not allowed
there), so that the automaton itself stays small: the vocabulary is kept once, not once per state.  The masks of
allowed ids that the logits take (`csrc.kernels.shape_logits`) are made from it, one row of bits per state: on a device a grammar
keeps a bit for every id and state while it lives (10,000 states of 151,936 ids: 190 MB).  What builds an
automaton from a schema or a context-free grammar is outside this library; `from_rows` and `choices` build small ones."""
from __future__ import annotations

from typing import Dict, Iterable, List, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch


class TokenGrammar:
    """`classes` [vocabulary]: the class of every id; `next` [states][classes]: the state that follows, -1 where an id of the
    class is not allowed; `start`: the state of a sequence that has made no id yet."""

    def __init__(self, classes: Sequence[int], next: Sequence[Sequence[int]], start: int = 0):
        self.classes = np.array(classes, dtype=np.int32, order="C")          # (copies that nobody writes to: `on` keeps others)
        self.next = np.array(next, dtype=np.int32, order="C")
        self.classes.flags.writeable = self.next.flags.writeable = False
        self.start = int(start)
        if self.classes.ndim != 1 or self.classes.size == 0 or self.next.ndim != 2 or self.next.size == 0:
            raise ValueError("a grammar has a class per id and a row of classes per state")
        states, n = self.next.shape
        if self.classes.min() < 0 or self.classes.max() >= n:
            raise ValueError(f"a grammar's classes lie in 0..{n - 1}")
        if self.next.min() < -1 or self.next.max() >= states or not 0 <= self.start < states:
            raise ValueError(f"a grammar's states lie in 0..{states - 1}")
        self._on: Dict[torch.device, Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = {}

    @property
    def vocab_size(self) -> int:
        return int(self.classes.size)

    @property
    def states(self) -> int:
        return int(self.next.shape[0])

    @classmethod
    def from_rows(cls, vocab_size: int, rows: Sequence[Mapping[Optional[int], int]], start: int = 0) -> "TokenGrammar":
        """`rows[state]` maps an id to the state that follows; under None stands what follows all ids that it does not list (not
        there: they are not allowed)."""
        named = sorted({t for row in rows for t in row if t is not None})
        if named and not (0 <= named[0] and named[-1] < vocab_size):
            raise ValueError(f"a grammar names ids outside the vocabulary (0..{vocab_size - 1})")
        columns: Dict[Tuple[int, ...], int] = {}

        def class_of(t: Optional[int]) -> int:
            column = tuple(int(row.get(t, row.get(None, -1))) for row in rows)
            return columns.setdefault(column, len(columns))

        classes = np.full(vocab_size, class_of(None), dtype=np.int32)
        for t in named:
            classes[t] = class_of(t)
        return cls(classes, np.array(list(columns), dtype=np.int32).T.reshape(len(rows), len(columns)), start)

    @classmethod
    def choices(cls, vocab_size: int, sequences: Iterable[Sequence[int]], end: Sequence[int]) -> "TokenGrammar":
        """One of the given sequences of ids, then one of the `end` ids (a model's stop ids)."""
        rows: List[Dict[Optional[int], int]] = [{}, {}]          # 0: the start, 1: behind the end, where nothing goes on
        for seq in sequences:
            at = 0
            if not len(seq):
                raise ValueError("a choice has at least one id")
            for t in seq:
                if t in rows[at] and rows[at][t] != 1:
                    at = rows[at][t]
                    continue
                rows.append({})
                rows[at][int(t)] = len(rows) - 1
                at = len(rows) - 1
            for t in end:
                rows[at].setdefault(int(t), 1)
        if not rows[0]:
            raise ValueError("a grammar of choices needs at least one")
        return cls.from_rows(vocab_size, rows)

    def step(self, state: int, token: int) -> int:
        """The state after `token`, or -1 where it is not allowed (no id, an id outside the vocabulary, or after a -1)."""
        if state < 0 or not 0 <= token < self.classes.size:
            return -1
        return int(self.next[state, self.classes[token]])

    def walk(self, tokens: Sequence[int], state: Optional[int] = None) -> int:
        """The state after all of `tokens` (-1: one of them was not allowed)."""
        at = self.start if state is None else state
        for t in tokens:
            at = self.step(at, int(t))
        return at

    def allowed(self, state: int) -> np.ndarray:
        """One truth value per id."""
        if state < 0:
            return np.zeros(self.classes.size, dtype=bool)
        return self.next[state][self.classes] >= 0

    def masks(self) -> np.ndarray:
        """[states, words] int32: bit v % 32 of word v / 32 is set where id v is allowed."""
        words = -(-self.classes.size // 32)
        packed = np.zeros((self.states, words * 4), dtype=np.uint8)
        for s in range(self.states):
            row = np.packbits(self.allowed(s), bitorder="little")
            packed[s, :row.size] = row
        return packed.view(np.int32)

    def on(self, device) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(masks, classes, next) on a device, made at the first call."""
        device = torch.device(device)
        if device not in self._on:
            self._on[device] = tuple(torch.from_numpy(a if a.flags.writeable else np.array(a)).to(device)
                                     for a in (self.masks(), self.classes, self.next))
        return self._on[device]
