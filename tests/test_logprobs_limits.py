"""Token log probabilities at the limits of their arithmetic, of their kernels and of what a call may be given.

Oracle and tolerances are those of ``test_logprobs.py``, which derives them.
"""
import math

import pytest
import torch

from weightbridge_b200 import token_logprobs

from .test_logprobs import DTYPES, _bounds, _check, _check_grad, _close, _inputs, _oracle, gpu


@gpu
@pytest.mark.parametrize("temperature", [1.0, 0.01, 2.0 ** -20])
@pytest.mark.parametrize("rows,vocab", [(3, 40000), (1000, 2048), (2, 131072)])
def test_references_near_their_limit(rows, vocab, temperature):
    """Rows whose first columns lie just below 2^20 (or -2^20) in units of ln 2 and whose last ones lie
    0 to 40 nats higher, for the kernels of a warp, a CTA and a cluster a row."""
    x = torch.empty(rows, vocab, device="cuda")
    step = torch.arange(rows, device="cuda", dtype=torch.float64)
    for sign in (1.0, -1.0):
        for below in (-3.0, 0.1, 3.0, 17.0, 30.0):
            x[:] = (sign * 2.0 ** 20 * math.log(2.0) - below) * temperature
            x[:, -1] = ((sign * 2.0 ** 20 * math.log(2.0) - below + 10.0 * (1 + step % 3) + step % 11) * temperature).float()
            t = torch.full((rows,), vocab - 1, device="cuda")
            t[1::2] = 5
            _check(x, t, temperature=temperature)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1000, 20000, 60001])
def test_no_log_probability_above_0_and_no_entropy_below(dtype, vocab):
    """One column holds nearly all of the probability: both results are 0 but for their rounding, whose sign is known."""
    x, t = _inputs(400, vocab, dtype, seed=14, std=1.0)
    x[:, -3] = torch.linspace(12, 40, 400, device="cuda").to(dtype)
    t[:] = vocab - 3
    for part in (slice(0, 400), slice(0, 7)):
        out = _check(x[part], t[part], top_k=2, grad=part.stop == 7)
        assert not bool((out.logprobs > 0).any()) and not bool((out.top_logprobs > 0).any()) and not bool((out.entropy < 0).any())
    out = _check(x, t)
    assert not bool((out.logprobs > 0).any()) and not bool((out.entropy < 0).any())
