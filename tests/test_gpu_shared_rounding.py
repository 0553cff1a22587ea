"""How the parts of a shared prefix are rounded: one key that outweighs all others gives back its value, to the bit.

Every head of a row looks along one direction u (elements +-2 in the key that it finds, +-c in q, 1 <= c < 1.5): that key's score is
2 c 128 / sqrt(128), 22.6 c, in units of e.  All other keys are normal numbers: their scores c sqrt(128) N / sqrt(128) = c N, and
2,304 of them weigh at most 2304 e^(6 c) / e^(22.6 c) < 2304 e^-16.6 = 1.5e-4 together even if every one stood at N = 6; as they are
(mean weight e^(c^2 / 2)) below 2304 e^(1.2 - 22.6) < 2e-6.  Their values are below 2 in size and so is the found one's, at least 1:
what they add moves the result by less than 4e-6 of itself, and the sums are 32-bit (2,304 terms, 2^-24 each and a weight: below 2e-4
of the others' 2e-6, and 2^-23 of the found one's).  The found value, a bfloat16 number, is 2^-9 of itself or more from the middle
to a neighbour, so the rounded result is it, provided that the weight's own rounding to bfloat16 (up to 2^-8 of it) is in the
denominator, too: the key's weight is some 2^25 to 2^49 against the maximum of the run's first page, which is the one in use."""
import math

import pytest
import torch

from test_gpu_shared_attention import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d, nq, nkv, groups, where", [(128, 32, 8, [8], 5), (128, 32, 8, [40], 31), (128, 12, 4, [3, 9], 17), (128, 32, 2, [12], 30)])
@pytest.mark.parametrize("how", [dict(together=True), dict(together=True, runs=3), dict(together=True, runs=296), dict(together=False)])
def test_one_key_that_outweighs_all_gives_back_its_value(d, nq, nkv, groups, where, how):
    s = Setup(groups, [32] * len(groups), (1, 200), nq, nkv, d, seed=7)
    g = torch.Generator(device="cuda").manual_seed(8)
    G = nq // nkv
    u = torch.where(torch.rand(nkv, d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    c = (1 + torch.rand(s.T, nq, generator=g, device="cuda") / 2).to(torch.bfloat16).float().clamp(max=1.4921875)
    s.q = (c[:, :, None] * u.repeat_interleave(G, 0)[None]).reshape(s.T, nq * d).to(torch.bfloat16)
    m = torch.randint(0, 128, s.v.shape, generator=g, device="cuda").float()
    s.v = ((1 + m / 128) * torch.where(torch.rand(s.v.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)).to(torch.bfloat16)
    want = torch.empty(s.T, nq * d, dtype=torch.bfloat16, device="cuda")
    for r, pages in enumerate(s.lists):
        s.k[pages[where], :, 41] = (2 * u).to(torch.bfloat16)
        want[r] = s.v[pages[where], :, 41].repeat_interleave(G, 0).reshape(-1)
    assert torch.equal(s.run(**how), want)


def test_the_error_of_steep_rows_is_that_of_rows_alone():
    """Scores of standard deviation 6: the weights of a row read together are rounded as they are summed, so that it is no further from
    the formula than twice a row alone (both hold the weights in bfloat16; a row alone rounds them below its maximum so far)."""
    s = Setup([16], [36], (1, 200), 32, 8, 128, seed=9, size=6.0)
    out, _ = s.want()
    off = {how: float((s.run(together=how).double() - out).norm() / out.norm()) for how in (True, False)}
    # the result's own rounding: half a step, 2^-8 of each number at most
    assert off[True] < min(2.0 ** -8, 2 * off[False]), off
    assert math.isfinite(off[True])
