"""Grammars over token ids and the shaping of a row of logits on the host (no GPU)."""
import numpy as np
import pytest

from gogguf_b200.engine.generate import GenerateParams
from gogguf_b200.sampling import LogitShaping, TokenGrammar, shape_host


def test_rows_make_classes():
    g = TokenGrammar.from_rows(100, [{5: 1, None: 0}, {7: 0, 8: 0}])
    assert g.next.shape[1] == 3 and g.states == 2 and g.vocab_size == 100          # the rest, 5, and 7 with 8
    assert g.step(0, 5) == 1 and g.step(0, 99) == 0 and g.step(1, 7) == 0 and g.step(1, 5) == -1 and g.step(1, 100) == -1 and g.step(-1, 5) == -1
    assert g.walk([1, 2, 5, 8, 5]) == 1 and g.walk([5, 5]) == -1 and g.walk([5, 5, 7]) == -1
    assert g.allowed(0).all() and list(np.flatnonzero(g.allowed(1))) == [7, 8] and not g.allowed(-1).any()


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100])
def test_masks_are_the_allowed_ids(vocab):
    rng = np.random.default_rng(vocab)
    classes = rng.integers(0, 4, vocab)
    g = TokenGrammar(classes, rng.integers(-1, 3, (3, 4)))
    m = g.masks()
    assert m.shape == (3, -(-vocab // 32)) and m.dtype == np.int32
    for s in range(3):
        assert [bool(m[s, v // 32] >> (v % 32) & 1) for v in range(vocab)] == g.allowed(s).tolist()
        for v in range(vocab):
            assert g.allowed(s)[v] == (g.step(s, v) >= 0)


def test_choices():
    g = TokenGrammar.choices(50, [[1, 2, 3], [1, 4], [9]], end=[0])
    for seq in ([1, 2, 3, 0], [1, 4, 0], [9, 0]):
        assert g.walk(seq) >= 0
    for seq in ([1, 0], [2], [1, 2, 3, 4], [9, 9], [0], [9, 0, 0]):
        assert g.walk(seq) == -1
    both = TokenGrammar.choices(50, [[1], [1, 2]], end=[0])
    assert both.walk([1, 0]) >= 0 and both.walk([1, 2, 0]) >= 0
    with pytest.raises(ValueError):
        TokenGrammar.choices(50, [[]], end=[0])
    with pytest.raises(ValueError):
        TokenGrammar.choices(50, [], end=[0])


@pytest.mark.parametrize("bad", [dict(classes=[0, 2], next=[[0, 0]]), dict(classes=[0], next=[[1]]), dict(classes=[0], next=[[-2]]),
                                 dict(classes=[], next=[[0]]), dict(classes=[0], next=[]), dict(classes=[-1], next=[[0]]),
                                 dict(classes=[0], next=[[0]], start=1)])
def test_refusals(bad):
    with pytest.raises(ValueError):
        TokenGrammar(**bad)


def test_a_grammar_does_not_change_with_what_it_was_made_from():
    classes, rows = np.zeros(4, dtype=np.int32), np.zeros((1, 1), dtype=np.int32)
    g = TokenGrammar(classes, rows)
    classes[:], rows[:] = 1, -1
    assert g.step(0, 3) == 0 and g.on("cpu")[1].tolist() == [0] * 4
    with pytest.raises(ValueError):
        g.next[0, 0] = -1


def test_ids_outside_the_vocabulary_are_refused():
    with pytest.raises(ValueError):
        TokenGrammar.from_rows(10, [{10: 0}])


def test_shaping_of_a_row():
    g = TokenGrammar.from_rows(6, [{0: 0, 1: 0, 2: 0, 3: 0, 5: 0}])
    s = LogitShaping.of(GenerateParams(repeat_penalty=2.0, repeat_last_n=4, frequency_penalty=0.25, presence_penalty=0.5,
                                       logit_bias={3: 1.5, 2: 0.0}, grammar=g), 6)
    assert s.bias == ((3, 1.5),)
    row = np.array([4.0, -4.0, 1.0, 0.0, 9.0, 2.0], dtype=np.float32)
    shape_host(row, s, [5, 0, 0, 1, 99], [0])            # the last four: 0 twice, 1, and an id that is not in the vocabulary
    assert row.tolist() == [4 / 2 - 0.5 - 0.5, -8 - 0.25 - 0.5, 1.0, 1.5, -np.inf, 2.0]
    shape_host(row, s, [5], [4])                         # a sequence that has left the grammar
    assert (row == -np.inf).all()
    assert LogitShaping.of(GenerateParams(repeat_penalty=1.3), 6) is None      # the repeat penalty alone keeps its own path
