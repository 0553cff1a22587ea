"""Captured steps of sequences that share pages, by the rule that chooses how they are read."""
import pytest
import torch

from helpers import TINY_L, TOL_BF16, random_tokens, rel_err

pytestmark = pytest.mark.gpu


def test_rows_that_do_not_fill_their_bucket_are_read_together_and_captured_once(monkeypatch):
    """Five sequences (a bucket of eight) that share 60 pages: read together, by one graph while they grow, as sequences alone."""
    import gogguf_b200 as gg
    from gogguf_b200.csrc import fast_attention as A
    from gogguf_b200.engine.step import StepEntry
    together = []
    was = A.attn_decode_tma
    monkeypatch.setattr(A, "attn_decode_tma", lambda *a, **kw: (together.append(0), was(*a, **kw))[1])
    cfg = dict(TINY_L, num_attention_heads=32, num_key_value_heads=8, max_position_embeddings=8192)
    eng = gg.load_random(cfg, 3, gg.LoadOptions(max_tokens=64 * 200))
    ctx = eng.new_context()
    c, st, V = ctx.cache, ctx.stepper, cfg["vocab_size"]
    prompt = random_tokens(V, 64 * 60, 1)
    a = c.open()
    st.step([StepEntry(a, prompt)])
    slots = [a] + [c.fork(a) for _ in range(4)]
    texts = [list(prompt) for _ in slots]
    for k in range(64 * 4):
        new = random_tokens(V, 5, 50 + k)
        out = st.step([StepEntry(s, [t], want=[0]) for s, t in zip(slots, new)])
        for text, t in zip(texts, new):
            text.append(t)
    assert not together
    # a graph for each number of CTAs that share a row's own pages: 1, then 2 (from four pages on)
    assert len(st._graphs) == 2 and all(len(key) == 3 for key in st._graphs)
    last = out.clone()
    for r in (0, 3):
        s = c.open()
        alone = st.step([StepEntry(s, texts[r], want=[len(texts[r]) - 1])])
        c.close(s)
        assert rel_err(last[r], alone[0]) < TOL_BF16
    for s in slots:
        c.close(s)
    c.check()
