"""What the shaping of logits keeps for a step or an answer: no more than the histories hold (no GPU)."""
from gogguf_b200.sampling import LogitShaping, Sampler, SamplerConfig
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
