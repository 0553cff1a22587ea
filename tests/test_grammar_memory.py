"""What the masks of a grammar take on the host (no GPU)."""
import tracemalloc

import numpy as np
import pytest

from gogguf_b200.sampling import TokenGrammar


@pytest.mark.parametrize("v", [1, 31, 32, 33, 1000])
def test_masks_are_the_allowed_ids(v):
    rng = np.random.default_rng(v)
    g = TokenGrammar(rng.integers(0, 5, size=v), rng.integers(-1, 9, size=(9, 5)))
    masks = g.masks()
    assert masks.dtype == np.int32 and masks.shape == (9, -(-v // 32)) and masks.flags.c_contiguous
    for s in range(9):
        bits = (masks[s, np.arange(masks.shape[1] * 32) // 32].view(np.uint32) >> (np.arange(masks.shape[1] * 32) % 32).astype(np.uint32)) & 1
        assert (bits[:v].astype(bool) == g.allowed(s)).all() and not bits[v:].any()


def test_masks_take_a_bit_for_an_id_and_state():
    """The table itself and a few rows of one state (8 bytes an id at most, twice), not a byte for every id and state."""
    states, v = 2000, 16000
    rng = np.random.default_rng(0)
    g = TokenGrammar(rng.integers(0, 5, size=v), rng.integers(-1, states, size=(states, 5)))
    tracemalloc.start()
    masks = g.masks()
    peak = tracemalloc.get_traced_memory()[1]
    tracemalloc.stop()
    assert masks.nbytes == states * v // 8 and peak < masks.nbytes + 16 * v + 100_000
