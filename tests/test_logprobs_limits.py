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


def _warp_a_row(rows, vocab, dtype):
    """Whether the rows are many and short enough for a warp each (the rule of the launch)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = 1024 // dtype.itemsize
    tiles = (vocab + n - 1) // n + 1
    return tiles <= 65 and tiles * sms * 2 <= rows * 3


def _mixed(rows, vocab, dtype, seed, pad=0, start=0):
    """Rows of every kind, as a view of rows that are `pad` columns longer; (logits, tokens, rows without NaN)."""
    x, t = _inputs(rows, vocab + pad, dtype, seed=seed, vocab=vocab)
    x = x[:, start:start + vocab]
    at = torch.arange(rows, device="cuda") % 23
    low = torch.finfo(dtype).min
    x[at == 3] = -math.inf                                       # empty
    half = torch.arange(vocab, device="cuda") % 2 == 0
    x[(at == 5)[:, None] & half] = -math.inf
    x[(at == 7)[:, None] & half] = low
    x[at == 9] = low
    x[at == 11, -1] = 60.0
    x[at == 13, 0] = math.nan
    x[at == 15, vocab // 2] = math.inf
    t[at == 17] = vocab                                          # no such token
    t[at == 19] = -1
    t[at == 21] = -100
    return x, t, (at != 13) & (at != 15) & (at != 17) & (at != 19)


def _check_mixed(x, t, good, temperature=1.0):
    vocab = x.shape[1]
    leaf = x.detach().requires_grad_()
    out = token_logprobs(leaf, t, temperature=temperature)
    live = t != -100
    bad = ~good & live
    assert bool(out.logprobs[bad].isnan().all()) and not bool(out.logprobs[~bad].isnan().any())
    g = torch.Generator(device="cuda").manual_seed(2)
    g1, g2 = (torch.randn(t.shape, device="cuda", generator=g) for _ in range(2))
    d, = torch.autograd.grad((out.logprobs, out.entropy), leaf, (g1, g2))
    assert bool(d[bad & ~torch.isneginf(x).all(1)].isnan().all())
    keep_rows = good | ~live
    xs, ts = x[keep_rows], t[keep_rows]
    lp, h, logp, keep, z, p = _oracle(xs, ts, vocab, temperature)
    tol_lp, tol_h = _bounds(z, p, lp, vocab)
    _close(out.logprobs[keep_rows], lp, tol_lp, "logprobs")
    _close(out.entropy[keep_rows], h, tol_h, "entropy")
    _check_grad(d[keep_rows], g1[keep_rows], g2[keep_rows], lp, h, logp, p, keep, ts, vocab, temperature, tol_lp, tol_h)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,pad,start", [(10000, 1, 0, 0), (9990, 33, 0, 0), (5001, 1000, 0, 0), (2400, 1501, 7, 3), (10007, 2049, 1, 1), (4096, 9001, 0, 0),
                                                  (4097, 4096, 8, 5)])
def test_a_warp_a_row(dtype, rows, vocab, pad, start):
    """More rows than the grid has warps, aligned and not, with ignored, masked, empty and NaN rows between the others."""
    assert _warp_a_row(rows, vocab, dtype)
    x, t, good = _mixed(rows, vocab, dtype, seed=rows, pad=pad, start=start)
    _check_mixed(x, t, good, temperature=0.8)
    t[0] = t[-1] = -100
    t[rows // 4:rows // 4 + min(4736, rows // 2)] = -100         # as many in a row as a B200's grid has warps
    _check_mixed(x, t, good)
    t[:] = -100
    leaf = x.detach().requires_grad_()
    out = token_logprobs(leaf, t)
    d, = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), leaf)
    assert not bool(out.logprobs.any()) and not bool(out.entropy.any()) and not bool(d.any())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tiles", [2, 9, 64, 65, 66])
def test_row_counts_around_the_warp_rule(dtype, tiles):
    vocab = (tiles - 1) * (1024 // dtype.itemsize)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    border = (tiles * sms * 2 + 2) // 3
    assert _warp_a_row(border, vocab, dtype) == (tiles <= 65) and not _warp_a_row(border - 1, vocab, dtype)
    for rows in (border - 1, border):
        x, t, good = _mixed(rows, vocab, dtype, seed=rows)
        _check_mixed(x, t, good)


@gpu
@pytest.mark.parametrize("rows,vocab", [(149, 131072 - 256), (149, 131073), (150, 140001), (2, 2 ** 21), (1, 2 ** 21 - 5), (300, 152000)])
@pytest.mark.parametrize("top_k", [1, 20, 32])
def test_alternatives_of_wide_rows(rows, vocab, top_k):
    """More tiles a CTA than two a thread: their maxima are selected by search instead of by counting."""
    x, t = _inputs(rows, vocab, torch.float32, seed=16)
    x[0] = x[0].round()                                          # many ties
    if rows > 8:
        x[1] = 0.25                                              # one value: the lowest ids
        x[2] = -math.inf
        x[3] = -math.inf
        x[3, vocab - 7] = 1.0                                    # one column, then ties of -inf
        x[4] = torch.arange(vocab, device="cuda").float()
        x[5] = -x[4]
        x[6] = -0.0
        x[6, ::3] = 0.0
        x[7] = x[7].bfloat16().float()
        t[2] = -100
    for part in (slice(0, 12), slice(rows - 1, rows)):           # the oracle sorts in 64 bits
        want = _check(x[part], t[part], top_k=top_k, grad=False)
        out = token_logprobs(x, t, top_k=top_k)
        assert torch.equal(out.top_ids[part], want.top_ids)


@gpu
def test_next_tokens_by_ignoring_the_last_position():
    """The whole logits with the last position ignored: what the shifted views give, to the bit."""
    full, _ = _inputs(4 * 65, 5003, torch.bfloat16, seed=17)
    full = full.view(4, 65, 5003).requires_grad_()
    ids = torch.randint(0, 5003, (4, 65), device="cuda")
    g = torch.randn(4, 65, device="cuda")
    view = token_logprobs(full[:, :-1], ids[:, 1:])
    whole = token_logprobs(full, torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100))
    for a, b in zip(view[:2], whole[:2]):
        assert torch.equal(a, b[:, :-1]) and not bool(b[:, -1].any())
    d, = torch.autograd.grad(view[:2], full, (g[:, :-1], g[:, :-1]))
    e, = torch.autograd.grad(whole[:2], full, (g, g))
    assert torch.equal(d, e)


def test_released_storage_is_refused():
    """A tensor whose storage was given back, whole (its address is 0) or in part, still has its sizes."""
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)
    for left in (0, 31):
        gone, no_tokens = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)
        for y in (gone, no_tokens):
            y.untyped_storage().resize_(left)
        for logits, tokens in ((gone, t), (x, no_tokens)):
            with pytest.raises(ValueError, match="storage"):
                token_logprobs(logits, tokens)
    with pytest.raises(ValueError, match="CUDA"):                # nothing to read: not refused for that
        token_logprobs(torch.randn(0, 10), torch.zeros(0, dtype=torch.long))


@gpu
def test_saved_tensors_that_hooks_replace():
    """What a hook gives back is checked again: kept on the host and returned packed it is fine, left there it is refused."""
    full, _ = _inputs(8, 703, torch.float32, seed=18)
    ids = torch.randint(0, 700, (8,), device="cuda")
    leaf = full[:, 3:].detach().requires_grad_()
    g = torch.randn(8, device="cuda")

    def grad():
        out = token_logprobs(leaf, ids)
        return torch.autograd.grad((out.logprobs, out.entropy), leaf, (g, g))[0]

    want = grad()
    with torch.autograd.graph.save_on_cpu():
        assert torch.allclose(grad(), want, rtol=1e-6, atol=0)   # rows at other alignments
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x.cpu(), lambda x: x):
        with pytest.raises(RuntimeError, match="hook"):
            grad()
    for change in (lambda x: x[:4] if x.dim() else x, lambda x: x.double() if x.is_floating_point() else x):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, change):
            with pytest.raises(RuntimeError, match="hook"):
                grad()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x.t().contiguous().t() if x.dim() == 2 else x):
        assert torch.allclose(grad(), want, rtol=1e-6, atol=0)   # the same values in another order of memory
    assert torch.equal(grad(), want)
