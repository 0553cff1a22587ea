"""What the shaping of logits keeps for a step or an answer: no more than the histories hold (no GPU)."""
import pytest
import torch

from gogguf_b200.sampling import LogitShaping, Sampler, SamplerConfig, TokenGrammar, make_sampler
from gogguf_b200.sampling.shaping import ShapingState


def shaping(last_n, grammar=None, bias=()):
    return LogitShaping(1.1, last_n, 0.2, 0.1, tuple(bias), grammar)


def test_a_states_window_is_no_longer_than_the_histories():
    for last_n, want in ((1_000_000, 7), (5, 5), (7, 7), (-1, 7)):
        st = ShapingState(shaping(last_n), [[1, 2, 3], [4, 5, 6, 7, 8, 9, 10]], [[], []], "cpu")
        assert st.hist.shape == (2, want)
        assert st.hist[0].tolist() == [1, 2, 3] + [-1] * (want - 3) and st.hist[1].tolist() == list(range(11 - want, 11))
        assert st.hist_len.tolist() == [3, want] and st.hist_pos.tolist() == [3 % want, 0]
    # no history at all
    assert ShapingState(shaping(100), [[]], [[]], "cpu").hist.shape == (1, 1)
    # a state that follows answers has room for the ids that are still to come
    for last_n, most, want in ((1_000_000, 20, 27), (10, 20, 10), (25, 20, 25), (64, 0, 7)):
        st = ShapingState(shaping(last_n), [[1, 2, 3], [4, 5, 6, 7, 8, 9, 10]], [[], []], "cpu", most=most)
        assert st.hist.shape == (2, want) and st.hist_len.tolist() == [3, min(want, 7)]


def test_a_sampler_begins_with_what_its_requests_may_make(monkeypatch):
    monkeypatch.setattr(Sampler, "_ring_pairs", staticmethod(lambda rows, device: None))
    s = Sampler(SamplerConfig(temp=0.0), 1.0, 1_000_000, 16, shaping(1_000_000))
    s.begin([0, 1], [[1, 2], [3]], "cpu", 30)
    assert s._state.hist.shape == (2, 32) and s.device_only
    s.begin([0, 1], [[1, 2], [3]], "cpu")                   # not told: the window as it is asked for
    assert s._state.hist.shape == (2, 1_000_000)


class CountedGrammar(TokenGrammar):
    steps = 0

    def step(self, state, token):
        CountedGrammar.steps += 1
        return super().step(state, token)


def counting(v):
    """Only v, v + 1, ... in turn, from 0 on, and back."""
    return CountedGrammar.from_rows(v, [{t: (t + 1) % v} for t in range(v)])


@pytest.mark.parametrize("kind", ["chain", "function"])
def test_a_waiting_loop_walks_each_id_once(kind):
    """The grammar's state goes on from where the last step left it: steps of the automaton grow with the ids, not with their square."""
    v, n = 7, 200
    cfg = SamplerConfig(temp=0.0) if kind == "chain" else (lambda row: int(row.argmax()))
    s = make_sampler(cfg, 1.0, 64, v, shaping(3, counting(v)))
    made = [[], []]
    CountedGrammar.steps = 0
    for k in range(n):
        got = s.sample(torch.zeros(2, v), [4, 9], [k, k], [[5, 5] + made[0], [1] + made[1]])
        for m, t in zip(made, got):
            m.append(t)
    assert made == [[k % v for k in range(n)]] * 2
    assert CountedGrammar.steps <= 2 * 2 * n


@pytest.mark.parametrize("kind", ["chain", "function"])
def test_a_walk_begins_again_where_the_ids_are_others(kind):
    """What a caller gives is what counts: other ids for a stream, fewer of them, streams in another order or in a second batch."""
    v = 7
    cfg = SamplerConfig(temp=0.0) if kind == "chain" else (lambda row: int(row.argmax()))
    s = make_sampler(cfg, 1.0, 64, v, shaping(3, counting(v)))
    one = lambda streams, made: s.sample(torch.zeros(len(made), v), streams, [len(m) for m in made], [[6] + m for m in made])
    assert one([0, 1], [[0, 1, 2], [0]]) == [3, 1]
    assert one([1, 0], [[0, 1], [0, 1, 2, 3]]) == [2, 4]
    assert one([0], [[0]]) == [1]
    assert one([0], [[0, 1, 3]]) == [-1]                    # left the grammar: nothing is allowed
    assert one([0], [[0, 1, 3, 4]]) == [-1]
    assert one([0], [[0, 1, 2]]) == [3]
    assert one([0, 0], [[0, 1, 2, 3], [0, 1]]) == [4, 2]    # a stream twice


def test_what_does_not_change_is_made_once():
    """Biases of a waiting loop's rows are on the device once for a number of rows."""
    sh = shaping(3, bias=[(2, 1.5), (5, -1.0)])
    a = ShapingState(sh, [[1], [2]], [[], []], "cpu")
    b = ShapingState(sh, [[1, 1], [2, 3]], [[], []], "cpu", bias=a.bias)
    assert all(x is y for x, y in zip(a.bias, b.bias)) and a.bias[0].tolist() == [0, 2, 4] and a.bias[1].tolist() == [2, 5, 2, 5]
