"""Steps of sequences that share pages: whether sharing pays is decided once (no GPU)."""
import types

import pytest
import torch

from gogguf_b200.cache import KVRequest, SequenceCache
from gogguf_b200.csrc import fast_attention as A
from gogguf_b200.engine.graphs import GraphStepper
from gogguf_b200.engine.step import StepEntry, StepLayout

NQ, NKV = 32, 8


class Model:
    """As much of a model as a stepper asks for its decisions."""
    rt = types.SimpleNamespace(fast=True, dtype=torch.bfloat16, device=torch.device("cpu"))

    def __init__(self, heads=((NQ, NKV),)):
        self.heads = heads

    def parts(self):
        for nq, nkv in self.heads:
            yield types.SimpleNamespace(nq=nq, nkv=nkv, _fast=object())
        yield types.SimpleNamespace()


class Recorded(GraphStepper):
    """Captures and replays nothing, keeps what it would have captured."""

    def __init__(self, cache, **kw):
        super().__init__(Model(**kw), cache)
        self.captured = []

    def _capture(self, entries, bucket, width, prefixes=None):
        self.captured.append((bucket, width, prefixes))
        lay = StepLayout(bucket, bucket, bucket, [width], sorted(prefixes.groups) if prefixes else ())
        event = types.SimpleNamespace(synchronize=lambda: None, record=lambda: None)
        return types.SimpleNamespace(graph=types.SimpleNamespace(replay=lambda: None), host=None, host2=None, dev=None, ws=None, turn=0,
                                     copied=[event, event], layout=lay, kernels=0, logits=torch.zeros(bucket, 1))

    def build_context(self, entries, **kw):
        self.now = kw["prefixes"]

    def decode(self, slots):
        self._enqueue_decode([StepEntry(s, [0], want=[0]) for s in slots], None, None)
        return self.now


def forks(n, tokens, pages=2000):
    c = SequenceCache([KVRequest(NKV, 8)], [None], 64 * pages, dtype=torch.bfloat16, device="cpu", max_slots=80)
    a = c.open()
    c.plan([a], [tokens])
    c.commit([a], [tokens])
    return c, [a] + [c.fork(a) for _ in range(n - 1)]


def plan_of(stepper, prefixes, rows):
    lay = StepLayout(rows, rows, rows, [1], sorted(prefixes.groups))
    return stepper.prefix_plans(lay, torch.zeros(lay.total, dtype=torch.int32), prefixes)[0]


@pytest.mark.parametrize("rows, bucket", [(5, 8), (9, 16), (3, 4), (33, 64)])
def test_the_decision_is_made_once(rows, bucket):
    """A step that is found to be worth sharing is read together, whatever rows its graph is filled up to."""
    pages = next(p for p in range(1, 600) if A.prefix_pays([(rows, p)], rows, NKV))
    c, slots = forks(rows, 64 * pages)
    st = Recorded(c)
    prefixes = st.decode(slots)
    assert prefixes is not None and st.captured[0][0] == bucket
    assert plan_of(st, prefixes, bucket).pays(NKV)
    c, slots = forks(rows, 64 * (pages - 1))
    assert Recorded(c).decode(slots) is None
