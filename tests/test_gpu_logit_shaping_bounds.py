"""Numbers on the device that lie outside what they index: the shaping of logits reads nothing there."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BIG = 2 ** 31 - 1


@pytest.mark.parametrize("in_place", [False, True])
def test_lists_of_biases_that_begin_or_end_outside(in_place):
    """A request's list is what of start[q]..start[q + 1] - 1 there is; nothing where it begins beyond the list, or ends before it begins."""
    from gogguf_b200.csrc import kernels as K
    dev = dict(dtype=torch.int32, device="cuda")
    ids, values = torch.tensor([3, 4, 5, 6], **dev), torch.tensor([1.0, 2.0, 4.0, 8.0], device="cuda")
    for pair, want in (((BIG, BIG), {}), ((5, BIG), {}), ((4, BIG), {}), ((2, BIG), {5: 4.0, 6: 8.0}), ((-BIG - 1, 1), {3: 1.0}), ((-7, -3), {}),
                       ((3, 1), {}), ((BIG, 0), {}), ((BIG - 200, BIG), {})):
        x = torch.zeros(1, 5000, device="cuda")
        out = x if in_place else torch.empty_like(x)
        got = K.shape_logits(x, out, bias=(torch.tensor(pair, **dev), ids, values)).cpu()[0]
        assert {int(i): float(got[i]) for i in got.nonzero()} == want, pair


def test_windows_and_states_outside():
    from gogguf_b200.csrc import kernels as K
    dev = dict(dtype=torch.int32, device="cuda")
    hist = torch.tensor([[1, 2, 3], [4, -5, BIG]], **dev)
    for length, want in (((-BIG - 1, 2), {(1, 4)}), ((BIG, 0), {(0, 1), (0, 2), (0, 3)}), ((1, BIG), {(0, 1), (1, 4)})):
        got = K.shape_logits(torch.zeros(2, 40, device="cuda"), hist=hist, hist_len=torch.tensor(length, **dev), presence=1.0).cpu()
        assert {tuple(i.tolist()) for i in got.nonzero()} == want
    got = K.shape_logits(torch.zeros(3, 40, device="cuda"), ring_rows=torch.tensor([BIG, -1, 1], **dev), hist=hist, hist_len=torch.tensor([3, 1], **dev),
                         presence=1.0, masks=torch.zeros(1, 2, **dev), mask_rows=torch.tensor([BIG, -BIG], **dev)).cpu()
    assert {tuple(i.tolist()) for i in got.nonzero()} == {(2, 4)}
