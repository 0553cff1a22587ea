"""Steps of sequences that share pages: whether sharing pays is decided once, and a captured step is found by what its launches
depend on (no GPU)."""
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


def test_captures_of_answers_that_grow():
    """64 answers of 500 tokens to a prompt of 2,048: a graph for each width of the table."""
    c, slots = forks(64, 2048)
    st = Recorded(c)
    widths = set()
    for _ in range(500):
        assert st.decode(slots) is not None
        widths.add(st._width_bucket(slots))
    assert len(st.captured) == len(widths) == 1, [(b, w, p.own_pages) for b, w, p in st.captured]


def test_a_graph_serves_the_launch_it_was_captured_for():
    """Steps that are answered by one graph have the same launches, and those are what their plans ask for."""
    seen = {}
    for rows, pages in ((5, 60), (5, 100), (7, 64), (8, 70), (6, 130), (8, 256)):
        c, slots = forks(rows, 64 * pages)
        st = Recorded(c)
        for k in range(1200):
            prefixes = st.decode(slots)
            if prefixes is None or k % 37:
                continue
            plan = plan_of(st, prefixes, 8)
            key, launch = st.prefix_key(prefixes, 8), plan.launch(NQ, NKV, 512)
            assert (8, st._width_bucket(slots), key) in st._graphs and seen.setdefault(key, launch) == launch
            assert 1 <= launch[0] <= A.SHARED_RUNS and 1 <= launch[1] <= A.SHARED_SHARES
    assert len(set(seen.values())) == len(seen)


def test_layers_with_other_numbers_of_heads():
    """The key holds the launches of every number of query heads on a group's kv heads, and of no other."""
    c, slots = forks(64, 64 * 12)
    one, two, other = (Recorded(c, heads=h) for h in (((32, NKV),), ((32, NKV), (128, NKV)), ((32, NKV), (32, 4))))
    prefixes = one.shared_prefixes(slots)
    a, b, o = (st.prefix_key(prefixes, 64) for st in (one, two, other))
    assert a == o and a != b
    # 64 members are two tiles of 128 rows with four heads each, eight with sixteen: 192 and 768 pages of (tile, kv head), four a run
    assert A.step_launch([(64, 12)], 1, 64, 32, NKV)[0] == 64 and A.step_launch([(64, 12)], 1, 64, 128, NKV)[0] == A.SHARED_RUNS // 2


def test_heads_inside_a_mixer_of_mixers_and_heads_that_are_not_known():
    """Attention that stands beside other mixers in one part counts as any other; where no part says its heads, steps are told apart by
    the weight of their groups and their own pages."""
    c, slots = forks(64, 64 * 12)
    flat = Recorded(c)
    inner = types.SimpleNamespace(nq=NQ, nkv=NKV, _fast=object())
    other = types.SimpleNamespace(_fast=object())
    nested = Recorded(c)
    nested.model.parts = lambda: iter([types.SimpleNamespace(members=[(other, 1.0, True), (inner, 0.5, None)]), other])
    GraphStepper.__init__(nested, nested.model, c)
    prefixes = flat.shared_prefixes(slots)
    assert nested._heads == flat._heads == [(NQ, NKV)] and nested.prefix_key(prefixes, 64) == flat.prefix_key(prefixes, 64)
    unknown = Recorded(c, heads=())
    c2, slots2 = forks(64, 64 * 48)
    few, many = unknown.prefix_key(prefixes, 64), Recorded(c2, heads=()).prefix_key(Recorded(c2).shared_prefixes(slots2), 64)
    assert few != many
