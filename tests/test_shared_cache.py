"""Sequences that go on from the same tokens: pages held by several slots, copied when one writes to them (no GPU)."""
import random

import pytest
import torch

from gogguf_b200.cache import CacheError, CacheFull, KVRequest, SequenceCache, StateRequest
from gogguf_b200.cache.sequence_cache import LatentRequest, PagedStore
from gogguf_b200.engine.generate import GenerateParams, Generator, plan_shared_batches
from gogguf_b200.sampling import SamplerConfig, TokenGrammar


def make(max_tokens=64 * 12, window=None, state=False, latent=False, max_slots=None):
    reqs = [KVRequest(2, 8)]
    if window:
        reqs.append(KVRequest(2, 8, window=window))
    if state:
        reqs.append(StateRequest((3,), torch.float32))
    if latent:
        reqs.append(LatentRequest(12))
    return SequenceCache(reqs, [None] * len(reqs), max_tokens, dtype=torch.float32, device="cpu", max_slots=max_slots)


def write(c, slot, n, mark):
    """A step of n tokens that writes `mark` at its positions, as the kernels would."""
    c.plan([slot], [n])
    for p in range(c.length(slot), c.length(slot) + n):
        for st in c.stores:
            if not st.paged:
                st.state[slot] += mark
                continue
            page = st.seq_pages[slot][p // 64]
            if hasattr(st, "pool"):
                st.pool[:, page, p % 64] = mark
            else:
                st.k[:, page, :, p % 64] = mark
                st.v[:, page, :, p % 64] = -mark
    c.commit([slot], [n])
    c.check()


def tokens(c, slot, group=0):
    g = c.groups[group]
    return [float(g.k[0, g.seq_pages[slot][p // 64], 0, p % 64, 0]) for p in range(c.length(slot)) if g.seq_pages[slot][p // 64] >= 0]


def test_a_fork_shares_pages_until_it_writes():
    c = make(state=True, latent=True)
    a = c.open()
    write(c, a, 100, 1.0)
    held = c.groups[0].pages.held_count
    b = c.fork(a)
    assert c.groups[0].pages.held_count == held == 2 and c.length(b) == 100 and c.groups[0].shared
    assert torch.equal(c.view(1).state[a], c.view(1).state[b])
    write(c, b, 1, 2.0)                                  # the second page is half full: copied before b writes to it
    assert c.groups[0].pages.held_count == 3
    assert c.groups[0].seq_pages[a][0] == c.groups[0].seq_pages[b][0] and c.groups[0].seq_pages[a][1] != c.groups[0].seq_pages[b][1]
    write(c, a, 1, 3.0)                                  # its own by now
    assert c.groups[0].pages.held_count == 3
    assert tokens(c, a) == [1.0] * 100 + [3.0] and tokens(c, b) == [1.0] * 100 + [2.0]
    pool = c.view(2).pool
    pages = c.groups[1].seq_pages
    assert float(pool[pages[a][1], 36, 0]) == 3.0 and float(pool[pages[b][1], 36, 0]) == 2.0 and float(pool[pages[b][1], 35, 0]) == 1.0
    c.close(a)
    assert c.groups[0].pages.held_count == 2 and not c.groups[0].shared
    assert tokens(c, b) == [1.0] * 100 + [2.0]
    c.close(b)
    c.check()
    assert c.groups[0].pages.held_count == 0


def test_a_fork_at_a_page_border_copies_nothing():
    c = make()
    a = c.open()
    write(c, a, 128, 1.0)
    b = c.fork(a)
    write(c, a, 1, 2.0)
    write(c, b, 1, 3.0)
    assert c.groups[0].pages.held_count == 4
    assert tokens(c, a)[-2:] == [1.0, 2.0] and tokens(c, b)[-2:] == [1.0, 3.0]


def test_the_last_holder_writes_in_place_and_the_count_says_so():
    c = make(max_tokens=64 * 3)
    a = c.open()
    write(c, a, 10, 1.0)
    b, d = c.fork(a), c.fork(a)
    assert c.groups[0].copies_needed([a, b, d], [10, 10, 10]) == 2 and c.groups[0].copies_needed([b], [10]) == 1
    c.plan([a, b, d], [1, 1, 1])                         # three pages: two copies, one written in place
    c.commit([a, b, d], [1, 1, 1])
    c.check()
    assert c.groups[0].pages.free_count == 0
    for s in (a, b, d):
        c.close(s)
    a = c.open()
    write(c, a, 70, 1.0)
    b, d = c.fork(a), c.fork(a)
    with pytest.raises(CacheFull):
        c.plan([a, b, d], [1, 1, 1])                     # two copies, one page free
    c.check()
    assert c.pages_short([a, b, d], [1, 1, 1]) == 1 and c.pages_short([a], [1]) == 0
    c.close(d)
    write(c, a, 1, 2.0)
    write(c, b, 1, 3.0)


def test_a_cut_back_fork_leaves_the_others_tokens():
    c = make()
    a = c.open()
    write(c, a, 200, 1.0)
    b = c.fork(a)
    assert c.truncate(b, 70)
    write(c, b, 20, 2.0)                                 # into page 1, which a holds too
    assert tokens(c, a) == [1.0] * 200 and tokens(c, b) == [1.0] * 70 + [2.0] * 20
    c.restart(b)
    assert c.length(b) == 0 and tokens(c, a) == [1.0] * 200
    c.close(a)
    c.check()


def test_windowed_groups_and_unplanned_steps():
    c = make(window=70)
    a = c.open()
    write(c, a, 200, 1.0)
    b = c.fork(a)
    for s, mark in ((a, 2.0), (b, 3.0)):
        write(c, s, 100, mark)
    full, win = c.groups
    assert all(p < 0 for p in win.seq_pages[a][:3]) and tokens(c, a) == [1.0] * 200 + [2.0] * 100
    d = c.fork(b)
    c.plan([d], [5])
    c.unplan([d])
    c.check()
    assert tokens(c, d) == tokens(c, b)
    for s in (a, b, d):
        c.close(s)
    c.check()
    assert full.pages.held_count == win.pages.held_count == 0


def test_refusals():
    c = make(max_slots=2)
    with pytest.raises(CacheError):
        c.fork(0)                                        # not open
    a = c.open()
    c.fork(a)
    with pytest.raises(CacheFull):
        c.fork(a)                                        # no slot
    c.check()

    class Bare(PagedStore):
        pass
    bare = Bare(None, [0], 4, 64)
    assert not bare.can_fork
    with pytest.raises(CacheError):
        bare.fork(0, 1)


def test_random_forks_keep_the_books():
    rng = random.Random(3)
    c = make(max_tokens=64 * 20, window=100, state=True, max_slots=8)
    want = {}
    for k in range(600):
        do = rng.random()
        if do < 0.1 and len(want) < 8:
            want[c.open()] = []
        elif do < 0.3 and want and len(want) < 8:
            s = rng.choice(list(want))
            want[c.fork(s)] = list(want[s])
        elif do < 0.4 and want:
            s = rng.choice(list(want))
            c.close(s)
            del want[s]
        elif want:
            s, n, mark = rng.choice(list(want)), rng.choice([1, 1, 1, 7, 64, 65]), float(k + 1)
            if c.pages_short([s], [n]) <= 0:
                write(c, s, n, mark)
                want[s] += [mark] * n
            else:
                with pytest.raises(CacheFull):
                    c.plan([s], [n])
        c.check()
        for s, t in want.items():
            assert tokens(c, s) == t, k


V = 16


class ScriptedStepper:
    """The next token of a sequence is (last token + 1) % V."""

    def __init__(self, max_tokens=64 * 8, **kw):
        self.cache = make(max_tokens, **kw)
        self.steps = []

    def step(self, entries):
        slots, counts = [e.slot for e in entries], [len(e.tokens) for e in entries]
        self.cache.plan(slots, counts)
        self.steps.append([len(e.tokens) for e in entries])
        rows = [torch.nn.functional.one_hot(torch.tensor((e.tokens[w] + 1) % V), V).float() * 5 for e in entries for w in e.want]
        self.cache.commit(slots, counts)
        self.cache.check()
        return torch.stack(rows) if rows else None


def test_several_answers_run_the_prompt_once():
    st = ScriptedStepper()
    out = Generator(st, V, 1000).generate([[1, 2, 3], [7]], GenerateParams(max_tokens=3, answers=3))
    assert [r.tokens for r in out] == [[4, 5, 6]] * 3 + [[8, 9, 10]] * 3
    assert st.steps == [[3, 1], [1] * 6, [1] * 6] and st.cache.live_slots == 0
    # every answer draws as the request that it is: the first one's numbers do not depend on how many there are
    hot = GenerateParams(max_tokens=5, sampler=SamplerConfig(temp=5.0, seed=3))
    one = Generator(ScriptedStepper(), V, 1000).generate([[1]], hot)
    many = Generator(ScriptedStepper(), V, 1000).generate([[1]], GenerateParams(max_tokens=5, sampler=SamplerConfig(temp=5.0, seed=3), answers=6))
    assert many[0].tokens == one[0].tokens and len({tuple(r.tokens) for r in many}) > 1


def test_answers_that_do_not_fit_together_run_in_batches():
    st = ScriptedStepper(max_tokens=64 * 4, max_slots=4)
    out = Generator(st, V, 1000, max_batch=3).generate([list(range(10)) * 7], GenerateParams(max_tokens=4, answers=5))
    assert len(out) == 5 and all(r.tokens == [10, 11, 12, 13] for r in out) and st.cache.live_slots == 0
    assert [s for s in st.steps if s[0] == 70] == [[70], [70]]
    assert plan_shared_batches([130, 130, 130, 5], [0, 0, 0, 3], 10, 8, 64 * 5, 64, 1000) == [[0, 1, 2], [3]]
    assert plan_shared_batches([130] * 3, [0, 1, 2], 10, 8, 64 * 5, 64, 1000, prefix_tokens=128) == [[0, 1, 2]]
    with pytest.raises(ValueError):
        plan_shared_batches([400], [0], 10, 8, 64 * 5, 64, 1000)


def test_a_prefix_is_run_once_and_stays():
    st = ScriptedStepper(max_tokens=64 * 10)
    g = Generator(st, V, 1000)
    slot = st.cache.open()
    from gogguf_b200.engine.step import StepEntry
    prefix = [k % V for k in range(100)]
    st.step([StepEntry(slot, prefix)])
    out = g.generate([prefix + [5], prefix + [9, 10]], GenerateParams(max_tokens=2, answers=2), prefix=slot)
    assert [r.tokens for r in out] == [[6, 7]] * 2 + [[11, 12]] * 2 and [r.prompt_tokens for r in out] == [101, 101, 102, 102]
    assert st.steps == [[100], [1, 2], [1] * 4] and st.cache.live_slots == 1 and st.cache.length(slot) == 100
    # a prompt that is the prefix alone gives its last token back first
    out = g.generate([prefix], GenerateParams(max_tokens=1), prefix=slot)
    assert out[0].tokens == [(prefix[-1] + 1) % V] and st.cache.length(slot) == 100
    st.cache.close(slot)
    st.cache.check()


def test_storage_that_cannot_fork_runs_every_answer(monkeypatch):
    st = ScriptedStepper()
    monkeypatch.setattr(type(st.cache), "can_fork", property(lambda self: False))
    out = Generator(st, V, 1000).generate([[1, 2, 3]], GenerateParams(max_tokens=2, answers=2))
    assert [r.tokens for r in out] == [[4, 5]] * 2 and st.steps[0] == [3, 3]


def test_answers_refusals():
    g = Generator(ScriptedStepper(), V, 1000)
    with pytest.raises(ValueError):
        g.generate([[1]], GenerateParams(answers=0))
    slot = g.cache.open()
    with pytest.raises(ValueError):
        g.generate([[1]], GenerateParams(answers=2), held={0: slot})


def test_answers_to_a_prompt_as_long_as_the_context():
    """They add no page to the prompt's, and are planned in batches that the slots hold all the same."""
    g = Generator(ScriptedStepper(max_tokens=64 * 4), V, 64)
    res = g.generate([[1] * 64], GenerateParams(max_tokens=5, answers=11, stop_token_ids=[]))
    assert [r.tokens for r in res] == [[2]] * 11 and g.cache.live_slots == 0
    g.cache.check()


def test_windows_without_an_end():
    """repeat_last_n below zero is the whole history; a repeat penalty joins the others."""
    run = lambda **kw: [r.tokens for r in Generator(ScriptedStepper(), V, 1000).generate([[7, 5, 1]], GenerateParams(max_tokens=4, stop_token_ids=[0], **kw))]
    assert run(presence_penalty=9.0, logit_bias={9: 4.0}, repeat_last_n=-1) == [[2, 3, 4, 9]]
    assert run(presence_penalty=9.0, logit_bias={9: 4.0}, repeat_last_n=2) == [[2, 3, 4, 5]]
    with pytest.raises(ValueError):
        run(presence_penalty=9.0, repeat_penalty=float("inf"))


def test_penalties_biases_and_a_grammar_in_the_loop():
    run = lambda **kw: [r.tokens for r in Generator(ScriptedStepper(), V, 1000).generate([[1]], GenerateParams(max_tokens=4, stop_token_ids=[0], **kw))]
    assert run() == [[2, 3, 4, 5]]
    assert run(logit_bias={3: -10.0, 9: 1.0}) == [[2, 9, 10, 11]]
    assert run(logit_bias={2: float("-inf")}) == [[]]    # id 0, the first of equals, is the stop id
    g = TokenGrammar.from_rows(V, [{2: 1}, {3: 2, 7: 2}, {9: 3}, {}])
    assert run(grammar=g) == [[2, 3, 9]]                 # then nothing is allowed: the answer ends
    r = Generator(ScriptedStepper(), V, 1000).generate([[1]], GenerateParams(max_tokens=9, grammar=g))[0]
    assert r.finish_reason == "stop"
    assert run(frequency_penalty=9.0, logit_bias={7: 4.0}) == [[2, 3, 4, 5]]
    # an id of the prompt is penalised, too: 2 stands in it
    out = Generator(ScriptedStepper(), V, 1000).generate([[2, 1]], GenerateParams(max_tokens=1, presence_penalty=9.0, logit_bias={7: 4.0}))
    assert out[0].tokens == [7]
    with pytest.raises(ValueError):
        run(logit_bias={V: 1.0})
    with pytest.raises(ValueError):
        run(logit_bias={1: float("nan")})
    with pytest.raises(ValueError):
        run(presence_penalty=float("inf"))
    with pytest.raises(ValueError):
        run(grammar=TokenGrammar.from_rows(V + 1, [{0: 0}]))


def test_answers_beyond_one_batch_share_in_every_batch():
    """A prompt counts once in every batch that holds answers to it, not only in the one with its first answer."""
    plan = plan_shared_batches([2048] * 128, [0] * 128, 64, 64, 200 * 64, 64, 40960)
    assert [len(b) for b in plan] == [64, 64]
    # two prompts in turn: the second batch begins in the middle of one
    plan = plan_shared_batches([640] * 8, [0] * 4 + [4] * 4, 10, 3, 64 * 25, 64, 1000)
    assert plan == [[0, 1, 2], [3, 4, 5], [6, 7]]
    st = ScriptedStepper(max_tokens=64 * 20, max_slots=8)
    out = Generator(st, V, 1000, max_batch=4).generate([list(range(10)) * 64], GenerateParams(max_tokens=4, answers=12))
    assert len(out) == 12 and all(r.tokens == [10, 11, 12, 13] for r in out)
    assert [s for s in st.steps if s[0] == 640] == [[640]] * 3 and st.cache.live_slots == 0


@pytest.mark.parametrize("answers", [1, 2])
def test_prompts_that_are_a_prefix_of_whole_pages(answers):
    """They give their last token back, and write it to a page of their own: it is counted."""
    st = ScriptedStepper(max_tokens=64 * 6)
    g = Generator(st, V, 1000)
    from gogguf_b200.engine.step import StepEntry
    slot = st.cache.open()
    prefix = [k % V for k in range(128)]
    st.step([StepEntry(slot, prefix)])
    out = g.generate([list(prefix) for _ in range(4)], GenerateParams(max_tokens=10, answers=answers, stop_token_ids=[]), prefix=slot)
    assert [r.tokens for r in out] == [[(prefix[-1] + 1 + k) % V for k in range(10)]] * (4 * answers)
    assert st.cache.live_slots == 1 and st.cache.length(slot) == 128 and tuple(st.cache.groups[0].more_holders) == ()
    # one of its own for the last token, one for what follows
    assert plan_shared_batches([128] * 4, [0, 1, 2, 3], 10, 8, 64 * 4, 64, 1000, prefix_tokens=128) == [[0, 1], [2, 3]]
    assert plan_shared_batches([129] * 4, [0, 1, 2, 3], 10, 8, 64 * 4, 64, 1000, prefix_tokens=128) == [[0, 1, 2, 3]]


def test_a_prefix_that_cannot_be_cut_back_is_run_again_by_prompts_that_are_it():
    """A state in which all tokens are folded together cannot give the last one back: such a prompt shares nothing, and is planned so."""
    st = ScriptedStepper(max_tokens=64 * 6, state=True)
    g = Generator(st, V, 1000)
    from gogguf_b200.engine.step import StepEntry
    slot = st.cache.open()
    prefix = [k % V for k in range(128)]
    st.step([StepEntry(slot, prefix)])
    run = dict(params=GenerateParams(max_tokens=10, stop_token_ids=[]), prefix=slot)
    out = g.generate([list(prefix) for _ in range(3)], **run)
    assert [r.tokens for r in out] == [[(prefix[-1] + 1 + k) % V for k in range(10)]] * 3
    assert [s for s in st.steps if s[0] == 128] == [[128]] * 4
    # prompts that go on from it do share it
    out = g.generate([prefix + [k] for k in range(3)], **run)
    assert [r.tokens[0] for r in out] == [1, 2, 3] and [1, 1, 1] in st.steps and st.cache.live_slots == 1
    with pytest.raises(CacheError):
        st.cache.can_truncate(slot, 129)
    assert st.cache.can_truncate(slot, 128) and not st.cache.can_truncate(slot, 127) and st.cache.length(slot) == 128
