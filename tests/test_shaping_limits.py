"""Penalties and biases that are no numbers in 32 bits are refused before a kernel divides by them (no GPU)."""
import math

import pytest
import torch

from gogguf_b200.csrc import kernels as K
from gogguf_b200.csrc.build import KernelError
from gogguf_b200.engine.generate import GenerateParams
from gogguf_b200.sampling import LogitShaping

MOST = (2 - 2.0 ** -23) * 2.0 ** 127            # of float32
LEAST = 2.0 ** -149


@pytest.mark.parametrize("kw", [dict(repeat=1e-46), dict(repeat=1e39), dict(repeat=-1.0), dict(repeat=math.nan), dict(frequency=1e39),
                                dict(frequency=-math.inf), dict(presence=-4e38), dict(presence=math.nan)])
def test_shape_logits_refuses(kw):
    with pytest.raises(KernelError, match="as float32 numbers"):
        K.shape_logits(torch.zeros(2, 9), **kw)


@pytest.mark.parametrize("kw", [dict(repeat=LEAST), dict(repeat=MOST), dict(frequency=-MOST), dict(presence=MOST)])
def test_shape_logits_takes_what_32_bits_hold(kw):
    with pytest.raises(KernelError, match="on the current CUDA device"):        # the next thing that is wrong here
        K.shape_logits(torch.zeros(2, 9), **kw)


@pytest.mark.parametrize("kw", [dict(repeat_penalty=1e-46, presence_penalty=1.0), dict(repeat_penalty=1e39, presence_penalty=1.0),
                                dict(repeat_penalty=math.inf, presence_penalty=1.0), dict(frequency_penalty=1e39), dict(presence_penalty=-1e39),
                                dict(frequency_penalty=math.nan), dict(logit_bias={1: 1e39}), dict(logit_bias={1: -1e39}), dict(logit_bias={1: math.inf})])
def test_parameters_are_refused(kw):
    with pytest.raises(ValueError):
        LogitShaping.of(GenerateParams(**kw), 16)


def test_parameters_that_stay():
    s = LogitShaping.of(GenerateParams(repeat_penalty=LEAST, frequency_penalty=-MOST, logit_bias={1: -math.inf, 2: MOST}), 16)
    assert s.repeat == LEAST and s.bias == ((1, -math.inf), (2, MOST))
    for off in (0.0, -3.0, math.nan):                    # no repeat penalty, as where it stands alone
        assert LogitShaping.of(GenerateParams(repeat_penalty=off, presence_penalty=1.0), 16).repeat == 1.0
