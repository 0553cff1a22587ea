"""Several answers to one prompt, prompts behind a held prefix, penalties, biases and grammars, through the entry point."""
import math

import numpy as np
import pytest
import torch

from helpers import TOL_BF16, make_folder, random_tokens, rel_err

pytestmark = pytest.mark.gpu

LONG = 64 * 20 + 17          # positions of a prompt that is worth sharing


def engine(tmp_path_factory, name, dtype="bfloat16", **kw):
    import gogguf_b200 as gg
    folder = make_folder(tmp_path_factory.getbasetemp(), name, "bfloat16" if dtype == "bfloat16" else "float32", scale=4.0)
    return gg.load(folder, gg.LoadOptions(dtype=dtype, max_tokens=64 * 300, **kw))


@pytest.fixture
def always_shares(monkeypatch):
    """Prefixes are read together whatever it saves (the models here are small)."""
    from gogguf_b200.csrc import fast_attention as A
    monkeypatch.setattr(A, "prefix_pays", lambda groups, n_tokens, nkv: True)


def counted(monkeypatch):
    from gogguf_b200.csrc import fast_attention as A
    calls = []
    was = A.attn_decode_shared

    def count(*a, **kw):
        calls.append(1)
        return was(*a, **kw)
    monkeypatch.setattr(A, "attn_decode_shared", count)
    return calls


@pytest.mark.parametrize("name, dtype, graphs", [("L", "bfloat16", True), ("L", "bfloat16", False), ("M", "bfloat16", True), ("A", "float32", True)])
def test_steps_of_answers_are_the_steps_of_sequences_alone(tmp_path_factory, name, dtype, graphs, always_shares, monkeypatch):
    """The logits of forked sequences that go different ways, beside those of sequences that ran the whole text alone."""
    from gogguf_b200.engine.step import StepEntry
    calls = counted(monkeypatch)
    eng = engine(tmp_path_factory, name, dtype, graphs=graphs)
    n = min(LONG, eng.context_length() - 40)
    V = eng.model.spec.vocab_size
    ctx = eng.new_context()
    c, st = ctx.cache, ctx.stepper
    prompt, other = random_tokens(V, n, 1), random_tokens(V, 150, 2)
    a = c.open()
    st.step([StepEntry(a, prompt)])
    o = c.open()
    st.step([StepEntry(o, other)])
    forks = [a] + [c.fork(a) for _ in range(4)] + [o, c.fork(o)]
    texts = [list(prompt) for _ in range(5)] + [list(other) for _ in range(2)]
    worst = 0.0
    steps = 12
    kept = []
    for k in range(steps):
        new = random_tokens(V, len(forks), 100 + k)
        if k == 7:                                   # one leaves: its pages stay the others'
            c.close(forks.pop(2))
            texts.pop(2)
        out = st.step([StepEntry(s, [t], want=[0]) for s, t in zip(forks, new)])
        for text, t in zip(texts, new):
            text.append(t)
        kept.append(out.clone())
        c.check()
    for r, text in enumerate(texts):
        s = c.open()
        alone = st.step([StepEntry(s, text, want=[len(text) - 1])])
        c.close(s)
        worst = max(worst, rel_err(kept[-1][r], alone[0]))
    assert worst < (TOL_BF16 if dtype == "bfloat16" else 2e-5), worst
    assert bool(calls) == (dtype == "bfloat16")
    for s in forks:
        c.close(s)
    c.check()


def test_several_answers_and_a_prefix_through_the_entry_point(tmp_path_factory, always_shares, monkeypatch):
    import gogguf_b200 as gg
    calls = counted(monkeypatch)
    eng = engine(tmp_path_factory, "L")
    ctx = eng.new_context()
    V = eng.model.spec.vocab_size
    prompt = random_tokens(V, LONG, 5)
    hot = gg.SamplerConfig(temp=1.5, top_k=50, seed=11)
    one = ctx.generate(prompt, gg.GenerateParams(max_tokens=24, sampler=hot, stop_token_ids=[]))
    assert not calls
    many = ctx.generate(prompt, gg.GenerateParams(max_tokens=24, sampler=hot, stop_token_ids=[], answers=6))
    assert len(many) == 6 and calls and ctx.cache.live_slots == 0
    assert len({tuple(r.tokens) for r in many}) == 6 and all(len(r.tokens) == 24 for r in many)
    # the first token is drawn from the same logits in either call
    assert many[0].tokens[0] == one.tokens[0]
    with ctx.new_prefix(prompt[:-30]) as prefix:
        tail = prompt[-30:]
        again = ctx.generate([tail, tail[:9]], gg.GenerateParams(max_tokens=6, sampler=hot, stop_token_ids=[], answers=3), prefix=prefix)
        assert len(again) == 6 and [r.prompt_tokens for r in again] == [LONG] * 3 + [LONG - 21] * 3
        assert ctx.cache.live_slots == 1 and ctx.cache.length(prefix._slot) == LONG - 30
        greedy = gg.GenerateParams(max_tokens=1, stop_token_ids=[])
        got, want = ctx.generate(tail, greedy, prefix=prefix), ctx.generate(prompt, greedy)
        assert got.tokens == want.tokens
        with pytest.raises(ValueError):
            eng.new_context(max_tokens=640).generate(tail, greedy, prefix=prefix)
    with pytest.raises(ValueError):
        ctx.generate(tail, greedy, prefix=prefix)
    ctx.cache.check()
    assert ctx.cache.live_slots == 0


@pytest.mark.parametrize("name", ["gigopel", "sokirax", "felolorn", "dinuzen", "kulesun", "niresun"])
def test_other_architectures_answer_several_times(name):
    """Latent caches, windows, chunks and states per sequence: forked sequences against ones that ran the text alone."""
    import importlib
    import gogguf_b200 as gg
    from gogguf_b200.engine.step import StepEntry
    cases = importlib.import_module(f"{name}_cases")
    cfg = next(iter(cases.CASES.values()))[0]
    eng = gg.load_random(cfg, seed=3, options=gg.LoadOptions(dtype="float32", max_tokens=64 * 24))
    ctx = eng.new_context()
    c, st = ctx.cache, ctx.stepper
    if not c.can_fork:
        pytest.skip("a store of this configuration cannot be shared")
    V = eng.model.spec.vocab_size
    prompt = random_tokens(V, 90, 1)
    a = c.open()
    st.step([StepEntry(a, prompt)])
    forks = [a, c.fork(a), c.fork(a)]
    texts = [list(prompt) for _ in forks]
    for k in range(5):
        new = random_tokens(V, 3, 50 + k)
        out = st.step([StepEntry(s, [t], want=[0]) for s, t in zip(forks, new)]).clone()
        for text, t in zip(texts, new):
            text.append(t)
    for r, text in enumerate(texts):
        s = c.open()
        alone = st.step([StepEntry(s, text, want=[len(text) - 1])])
        c.close(s)
        # (recurrences that fold tokens one by one or in chunks differ by the rounding of their sums)
        assert rel_err(out[r], alone[0]) < 2e-4, (name, r)
    c.check()


def follow(row, shaping, history, made):
    from gogguf_b200.sampling import shape_host
    row = row.numpy().copy()
    shape_host(row, shaping, history, made)
    return row


@pytest.mark.parametrize("sampler", [dict(), dict(temp=0.9, seed=5), dict(temp=1.2, top_k=20, top_p=0.9, seed=6), dict(temp=1.1, top_p=0.8, seed=7)])
def test_a_step_ahead_of_the_host_draws_what_the_host_draws(tmp_path_factory, sampler):
    """Penalties, biases and a grammar: the loop that stays a step ahead, the one that waits for every id (kept logits), and the
    host's own arithmetic on the kept rows agree."""
    import gogguf_b200 as gg
    from gogguf_b200.sampling import LogitShaping, sample_host, uniform01
    eng = engine(tmp_path_factory, "L", "float32")
    ctx = eng.new_context()
    V = eng.model.spec.vocab_size
    prompts = [random_tokens(V, n, n) for n in (7, 30, 1)]
    g = gg.TokenGrammar.from_rows(V, [{None: 0, 5: 1, 6: -1, 7: -1}, {t: 0 if t % 3 else 1 for t in range(10, 60)}])
    kw = dict(max_tokens=14, sampler=gg.SamplerConfig(**sampler), stop_token_ids=[], repeat_penalty=1.3, repeat_last_n=9, frequency_penalty=0.4,
              presence_penalty=0.2, logit_bias={5: 3.0, 8: -math.inf, 12: 1.0}, grammar=g)
    ahead = ctx.generate(prompts, gg.GenerateParams(**kw))
    waited = ctx.generate(prompts, gg.GenerateParams(keep_logits=True, **kw))
    assert [r.tokens for r in ahead] == [r.tokens for r in waited]
    shaping = LogitShaping.of(gg.GenerateParams(**kw), V)
    cfg = gg.SamplerConfig(**sampler)
    for i, (p, r) in enumerate(zip(prompts, waited)):
        assert g.walk(r.tokens) >= 0 and 8 not in r.tokens and len(r.tokens) == 14
        for k, t in enumerate(r.tokens):
            row = follow(r.logits[k], shaping, list(p) + r.tokens[:k], r.tokens[:k])
            assert t == sample_host(row, cfg, uniform01(cfg.seed, i, k)), (i, k)


def test_a_window_without_an_end(tmp_path_factory):
    """repeat_last_n below zero: all of prompt and answer count, step by step."""
    import gogguf_b200 as gg
    from gogguf_b200.sampling import LogitShaping
    eng = engine(tmp_path_factory, "L", "float32")
    ctx = eng.new_context()
    prompts = [random_tokens(eng.model.spec.vocab_size, n, n) for n in (80, 2)]
    kw = dict(max_tokens=9, stop_token_ids=[], repeat_penalty=1.2, repeat_last_n=-1, frequency_penalty=2.0, logit_bias={4: 1.0})
    shaping = LogitShaping.of(gg.GenerateParams(**kw), eng.model.spec.vocab_size)
    out = ctx.generate(prompts, gg.GenerateParams(keep_logits=True, **kw))
    for p, r in zip(prompts, out):
        for k, t in enumerate(r.tokens):
            assert t == int(follow(r.logits[k], shaping, list(p) + r.tokens[:k], r.tokens[:k]).argmax())
    assert [r.tokens for r in ctx.generate(prompts, gg.GenerateParams(**kw))] == [r.tokens for r in out]


def test_an_answer_that_the_grammar_ends(tmp_path_factory):
    """A state in which nothing is allowed ends that answer, in the loop that is a step ahead and in the one that is not; the others go on."""
    import gogguf_b200 as gg
    eng = engine(tmp_path_factory, "L")
    ctx = eng.new_context()
    V = eng.model.spec.vocab_size
    g = gg.TokenGrammar.choices(V, [[3, 4, 5], [9] * 7, [11, 12]], end=[0])
    for keep in (False, True):
        for kw in (dict(), dict(sampler=gg.SamplerConfig(temp=2.0, seed=4)), dict(sampler=gg.SamplerConfig(temp=2.0, top_k=5, seed=4))):
            out = ctx.generate([[1, 2], [7]], gg.GenerateParams(max_tokens=12, grammar=g, stop_token_ids=[], answers=8, keep_logits=keep, **kw))
            for r in out:
                assert r.finish_reason == "stop" and r.tokens[-1] == 0 and r.tokens[:-1] in ([3, 4, 5], [9] * 7, [11, 12])
            out = ctx.generate([[1, 2]], gg.GenerateParams(max_tokens=12, grammar=g, stop_token_ids=[0], keep_logits=keep, **kw))
            assert out[0].tokens in ([3, 4, 5], [9] * 7, [11, 12]) and out[0].finish_reason == "stop"
    assert ctx.cache.live_slots == 0


def test_a_session_with_penalties_and_a_grammar(tmp_path_factory):
    import gogguf_b200 as gg
    eng = engine(tmp_path_factory, "L")
    ctx = eng.new_context()
    V = eng.model.spec.vocab_size
    prompts = [random_tokens(V, 12, 3), random_tokens(V, 4, 4)]
    g = gg.TokenGrammar.from_rows(V, [{None: 0, 3: -1}])
    params = gg.GenerateParams(max_tokens=8, frequency_penalty=0.7, presence_penalty=0.1, logit_bias={9: 0.5}, grammar=g, stop_token_ids=[])
    want = ctx.generate(prompts, params)
    with ctx.start_generation(prompts, stop_token_ids=[]) as sess:
        for _ in range(8):
            sess.decode_step(params)
        assert [sess.generated_tokens(i) for i in range(2)] == [r.tokens for r in want]
    with ctx.start_generation(prompts) as sess:
        with pytest.raises(ValueError):
            sess.decode_step(gg.GenerateParams(answers=2))


def test_advance_on_the_device():
    from gogguf_b200.csrc import kernels as K
    from gogguf_b200.sampling import TokenGrammar
    dev = dict(dtype=torch.int32, device="cuda")
    g = TokenGrammar.from_rows(40, [{3: 1, 39: 0}, {None: 0}])
    masks, classes, nxt = g.on("cuda")
    tokens = torch.tensor([3, 5, 39, 7, -1, 40, 39], **dev)
    rings = torch.tensor([6, 5, 4, 3, 2, 1, 0], **dev)
    states = torch.tensor([-1, 0, 0, 1, 0, 0, 0], **dev)              # ring 0 has no grammar
    hist, hlen, hpos = torch.full((7, 3), -1, **dev), torch.tensor([3, 0, 0, 2, 0, 0, 1], **dev), torch.tensor([1, 0, 0, 2, 0, 0, 1], **dev)
    K.shape_advance(tokens, rings, 7, hist=hist, hist_len=hlen, hist_pos=hpos, states=states, classes=classes, next=nxt)
    assert tokens.tolist() == [3, -1, 39, 7, -1, -1, 39]
    assert states.tolist() == [-1, 0, 0, 0, 0, 0, 1]
    assert hlen.tolist() == [3, 0, 0, 3, 1, 0, 2] and hpos.tolist() == [2, 0, 0, 0, 1, 0, 2]
    assert hist[0].tolist() == [-1, 39, -1] and hist[3].tolist() == [-1, -1, 7] and hist[4, 0] == 39 and hist[6, 1] == 3
    from gogguf_b200.csrc.build import KernelError
    with pytest.raises(KernelError):
        K.shape_advance(tokens, rings, 8, states=states, classes=classes, next=nxt)
    with pytest.raises(KernelError):
        K.shape_advance(tokens, rings, 7, states=states)
