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


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [500, 501])
@pytest.mark.parametrize("temperature,scale", [(1e-4, 2.0 ** 17), (1e-6, 2.0 ** 16), (1e-9, 1.0), (1e-12, 1.0), (1e-20, 1.0), (1e-30, 1.0), (1e-30, 1e6)])
def test_gradient_at_small_temperatures(dtype, vocab, temperature, scale):
    """Columns without any probability get no gradient, however large 1 / temperature and the incoming gradients are."""
    x, t = _inputs(6, vocab, dtype, seed=15)
    x[0, ::2] = -math.inf
    x[1, 3:] = torch.finfo(dtype).min
    x[2, 5] = x[2, 7] = 30.0                                     # two largest
    x[3] = 0.0
    x[3, 4] = -math.inf
    t[2], t[4] = 7, int(x[4].argmax())
    x = x[:, :vocab].detach().requires_grad_()
    out = token_logprobs(x, t, temperature=temperature)
    lp, h, logp, keep, z, p = _oracle(x, t, vocab, temperature)
    tol_lp, tol_h = _bounds(z, p, lp, vocab)
    g = torch.Generator(device="cuda").manual_seed(1)
    g1, g2 = (torch.randn(6, device="cuda", generator=g) * scale for _ in range(2))
    d, = torch.autograd.grad((out.logprobs, out.entropy), x, (g1, g2))
    assert bool(d.isfinite().all())
    _check_grad(d, g1, g2, lp, h, logp, p, keep, t, vocab, temperature, tol_lp, tol_h)


def test_forward_mode_derivatives_are_refused():
    """They would be lost: the results would come out as constants."""
    import torch.autograd.forward_ad as forward_ad
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)

    def refused(match, logits, tokens=t):
        with pytest.raises(ValueError, match=match):
            token_logprobs(logits, tokens)

    with forward_ad.dual_level():
        refused("forward mode", forward_ad.make_dual(x, torch.ones_like(x)))
        refused("forward mode", forward_ad.make_dual(x, torch.ones_like(x)).clone().requires_grad_())
        refused("forward mode", forward_ad.make_dual(torch.randn(5, 10), torch.ones(5, 10))[1:])


def test_lazily_negated_tensors_are_refused():
    """Their memory holds other values than they do."""
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)
    for logits, tokens in ((torch._neg_view(x), t), (torch.complex(x, x).conj().imag, t), (x, torch._neg_view(t))):
        with pytest.raises(ValueError, match="resolve_neg"):
            token_logprobs(logits, tokens)


@gpu
def test_lazily_negated_gradient():
    x, t = _inputs(5, 300, torch.float32)
    x.requires_grad_()
    out = token_logprobs(x, t)
    g = torch.randn(5, device="cuda")
    lazy = torch.complex(g, g).conj().imag                       # -g, with g's values in memory
    assert lazy.is_neg()
    for o in (out.logprobs, out.entropy):
        d, = torch.autograd.grad(o, x, lazy, retain_graph=True)
        want, = torch.autograd.grad(o, x, -g, retain_graph=True)
        assert torch.equal(d, want)


def test_tensors_of_transforms_are_refused():
    """What torch.func hands to a function has no memory of its own (an address of 0 for some)."""
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match="wrapper"):
        token_logprobs(torch._efficientzerotensor((4, 10)), t)
    for transform in (torch.func.functionalize, torch.func.grad, torch.vmap):
        with pytest.raises(ValueError, match="wrapper"):
            transform(lambda y: token_logprobs(y, t if y.dim() == 2 else t[0]).logprobs.sum())(x)
        with pytest.raises(ValueError, match="wrapper"):
            transform(lambda y: token_logprobs(x, y).logprobs.sum())(t.float() if transform is torch.func.grad else t)
