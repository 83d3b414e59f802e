"""AdamW and the gradient norm at the limits of their arithmetic, of their kernels and of what a call may be given.

Tolerances are those of ``test_optim.py``, which derives them.
"""
import math

import pytest
import torch

from weightbridge_b200 import AdamW, grad_norm

from .test_optim import _rand, _setup, _step_and_check, gpu


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
@pytest.mark.parametrize("shift", [0, 3])
def test_the_same_bits_every_time(states, shift):
    """Three steps, with another optimizer's steps between them and without: parameters, states and norms agree bit for bit."""
    sizes = [(1500001,), (300, 517), (70001,), (128,), (5,)]

    def make(seed=21):
        return _setup(sizes, torch.float32, shift=shift, seed=seed, states=states)

    a, ga, x = make()
    b, gb, y = make()
    c, gc, other = make(seed=40)
    for k in range(3):
        norms = x.step(ga, max_norm=None if k == 1 else 0.5), y.step(gb, max_norm=None if k == 1 else 0.5)
        other.step(gc)
        assert norms[0] is None and norms[1] is None or torch.equal(*norms)
    torch.cuda.synchronize()
    assert all(torch.equal(p, b[n]) for n, p in a.items())
    for p, q in zip(x.states().values(), y.states().values()):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


@gpu
def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as forward_ad
    p, g = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    opt = AdamW({"a": p})
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(g, torch.ones_like(g))
        for call in (lambda: AdamW({"a": dual}), lambda: opt.step({"a": dual}), lambda: grad_norm([dual])):
            with pytest.raises(ValueError, match="forward mode"):
                call()
    assert opt.step_count == 0 and bool((p == 1).all())


@gpu
def test_lazily_negated_tensors_are_refused():
    p, g = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    opt = AdamW({"a": p})
    for call in (lambda x: AdamW({"a": x}), lambda x: opt.step({"a": x}), lambda x: grad_norm([x])):
        with pytest.raises(ValueError, match="resolve_neg"):
            call(torch._neg_view(g))
    assert opt.step_count == 0 and bool((p == 1).all())


def test_tensors_of_transforms_are_refused():
    x = torch.ones(4)
    for transform in (torch.func.functionalize, torch.func.grad, torch.vmap):
        for call in (lambda y: AdamW({"a": y}), lambda y: grad_norm([y])):
            with pytest.raises(ValueError, match="wrapper"):
                transform(call)(x[0] if transform is torch.func.grad else x)
    with pytest.raises(ValueError, match="wrapper"):
        grad_norm([torch._efficientzerotensor((4,))])


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_captured_step_follows_rebound_parameters(states):
    params, grads, opt = _setup(states=states, seed=5, master=True)
    twin, _, ref = _setup(states=states, seed=5, master=True)
    for o in (opt, ref):
        o.step(grads, max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(grads, max_norm=1.0)
    first = {n: p.clone() for n, p in params.items()}
    moved = {n: p.clone() for n, p in params.items()}
    opt.rebind(moved)
    junk = [torch.full((1 << 12,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]      # takes what was given back
    for k in range(3):
        for i, g in enumerate(grads.values()):
            g.copy_(_rand(tuple(g.shape), g.dtype, 10 * k + i, 0.1))
        graph.replay()
        assert torch.equal(norm, ref.step(grads, max_norm=1.0))
    torch.cuda.synchronize()
    assert len(junk) == 64 and opt.step_count == ref.step_count == 4
    assert all(torch.equal(p, twin[n]) for n, p in moved.items())
    assert all(torch.equal(p, first[n]) for n, p in params.items())          # the old memory is left alone


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_optimizer_released_while_its_step_waits(states):
    """The step waits on a side stream behind other work; what the optimizer held is not given to anyone else before it ran."""
    params, grads, opt = _setup([(1 << 20,)], torch.bfloat16, states=states, master=True)
    twin, _, ref = _setup([(1 << 20,)], torch.bfloat16, states=states, master=True)
    ref.step(grads, max_norm=1.0)
    held = {t.data_ptr(): t.nbytes for t in opt.states().values()}
    sizes = sorted(held.values())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ran = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)                         # half a second
        opt.step(grads, max_norm=1.0)
        ran.record()
    del opt
    others = [torch.full((n,), 0x55, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
    assert not ran.query()                                       # else this test shows nothing
    for o in others:
        assert not any(a < o.data_ptr() + o.nbytes and o.data_ptr() < a + n for a, n in held.items())
    torch.cuda.synchronize()
    assert all(torch.equal(p, twin[n]) for n, p in params.items())


@gpu
def test_only_updated_parameters_change_their_version():
    """A graph that saved a frozen parameter is still good after a step."""
    p, q = (torch.nn.Parameter(_rand((40,), torch.float32, s)) for s in (1, 2))
    e = torch.nn.Parameter(torch.empty(0, device="cuda"))
    opt = AdamW({"p": p, "q": q, "e": e}, lr=0.1)
    kept = (q * q).sum()
    versions = q._version, p._version
    opt.step({"p": torch.ones_like(p), "q": None, "e": torch.empty(0, device="cuda")}, max_norm=1.0)
    assert q._version == versions[0] and p._version > versions[1]
    kept.backward()
    assert torch.equal(q.grad, 2 * q.detach())


def test_8_bit_second_moments_refuse_long_memories():
    p = {"a": torch.ones(4)}
    for beta2 in (0.951, 0.97, 0.99, 0.999):
        with pytest.raises(ValueError, match="beta2"):
            AdamW(p, betas=(0.9, beta2), states="fp8")
    with pytest.raises(ValueError, match="CUDA"):                # not refused for its betas
        AdamW(p, betas=(0.9, 0.95), states="fp8")
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(p, betas=(0.9, 0.999))


@gpu
def test_8_bit_second_moments_over_many_steps():
    """Normal gradients for 1200 steps at the largest beta2, then half of every block's a hundredth of
    before: the roots stay within half a step of the codes (2^-4) of those in 64 bits in the median, and
    98 of 100 between 3/4 and 3/2 of them (an emulation of the definition gives 0.86 to 1.28)."""
    n = 128 * 256
    params = {"p": torch.zeros(n, device="cuda")}
    opt = AdamW(params, lr=1e-3, weight_decay=0.0, states="fp8")
    assert opt.betas == (0.9, 0.95) and AdamW({"p": torch.zeros(4, device="cuda")}).betas == (0.9, 0.999)
    g = torch.Generator(device="cuda").manual_seed(3)
    v = torch.zeros(n, dtype=torch.float64, device="cuda")
    for step in range(1200):
        grad = torch.randn(n, device="cuda", generator=g)
        if step >= 600:
            grad[::2] *= 0.01
        opt.step({"p": grad})
        v = 0.95 * v + 0.05 * grad.double().square()
    st = opt.states()
    root = (st["rms"].float().view(-1, 128) * st["rms_scale"][:, None]).view(-1).double()
    ratio = root / v.sqrt()
    for part in (ratio[::2], ratio[1::2]):
        assert abs(math.log(float(part.median()))) <= math.log(1 + 2.0 ** -4)
        assert 0.75 < float(part.quantile(0.01)) and float(part.quantile(0.99)) < 1.5


def test_8_bit_first_moments_refuse_long_memories():
    p = {"a": torch.ones(4)}
    for beta1 in (0.981, 0.99, 0.999):
        with pytest.raises(ValueError, match="beta1"):
            AdamW(p, betas=(beta1, 0.95), states="fp8")
        with pytest.raises(ValueError, match="CUDA"):            # not refused for its betas
            AdamW(p, betas=(beta1, 0.95))
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(p, betas=(0.98, 0.95), states="fp8")


@gpu
@pytest.mark.parametrize("beta1,most", [(0.9, 0.09), (0.98, 0.2)])
def test_8_bit_first_moments_over_many_steps(beta1, most):
    """Normal gradients with means of a third of their size: what the codes' rounding adds up to (an
    emulation of the definition gives 0.059 and 0.134 of the moments)."""
    n = 128 * 256
    opt = AdamW({"p": torch.zeros(n, device="cuda")}, lr=1e-3, betas=(beta1, 0.95), weight_decay=0.0, states="fp8")
    g = torch.Generator(device="cuda").manual_seed(4)
    mean = 0.3 * torch.randn(n, device="cuda", generator=g)
    m = torch.zeros(n, dtype=torch.float64, device="cuda")
    for _ in range(1000):
        grad = torch.randn(n, device="cuda", generator=g) + mean
        opt.step({"p": grad})
        m = beta1 * m + (1 - beta1) * grad.double()
    st = opt.states()
    got = (st["exp_avg"].float().view(-1, 128) * st["exp_avg_scale"][:, None]).view(-1).double()
    assert float((got - m).norm() / m.norm()) < most


@gpu
def test_moments_that_are_not_numbers_stay_visible_in_8_bits():
    """The second moment of a NaN gradient is a NaN code, like the first; the block's others stay numbers."""
    params = {"p": torch.ones(256, device="cuda")}
    opt = AdamW(params, states="fp8")
    g = torch.ones(256, device="cuda")
    g[3] = math.nan
    for _ in range(2):
        opt.step({"p": g})
        g[3] = 1.0
        for key in ("exp_avg", "rms"):
            bad = opt.states()[key].float().isnan()
            assert bool(bad[3]) and int(bad.sum()) == 1
    assert int(params["p"].isnan().sum()) == 1


@gpu
@pytest.mark.parametrize("large", [2.0 ** 125, 2.0 ** 126, 1e38, 3.4e38])
def test_moments_near_the_largest_number_in_8_bits(large):
    """beta1 = 0: the first moment is the gradient; its block keeps it to half a step."""
    g = torch.full((256,), large, device="cuda")
    g[1] = -large / 2
    g[128:] = 1.0
    opt = AdamW({"p": torch.ones(256, device="cuda")}, betas=(0.0, 0.95), states="fp8")
    opt.step({"p": g})
    st = opt.states()
    got = st["exp_avg"].float().view(-1, 128).double() * st["exp_avg_scale"][:, None].double()
    assert bool(((got.view(-1) - g.double()).abs() <= g.double().abs() * 2.0 ** -4).all())


def test_eps_below_what_32_bits_can_hold_is_refused():
    p = {"a": torch.ones(4)}
    for eps in (0.0, 1e-40, 1e-30, 1e-20, 2.0 ** -51):
        with pytest.raises(ValueError, match="eps"):
            AdamW(p, eps=eps)
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(p, eps=2.0 ** -50)


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_small_gradients_take_small_steps(states):
    """Gradients down to 1e-40 at the smallest eps: a first step of g / (|g| + eps).  A second moment below
    2^-126 may count as 0: with beta2 = 0.95 that leaves out a root of at most 2^-63 / sqrt(0.05) < 2^-60.8
    beside eps, so 2^-10.8 of a step that is itself below 2^-10.8."""
    eps = 2.0 ** -50
    g = torch.logspace(-40, 0, 41, device="cuda", dtype=torch.float64).repeat_interleave(128)
    params = {"p": torch.zeros(g.numel(), device="cuda")}
    AdamW(params, lr=1.0, betas=(0.9, 0.95), weight_decay=0.0, eps=eps, states=states).step({"p": g.float()})
    want = -g / (g + eps)
    assert float((params["p"].double() - want).abs().max()) <= 2.0 ** -20


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_master_weights_reread_from_the_parameters(states):
    params, grads, opt = _setup(states=states, seed=9, master=True)
    opt.step(grads)
    for i, p in enumerate(params.values()):
        p.copy_(_rand(tuple(p.shape), p.dtype, 300 + i, 0.5))    # loaded from a checkpoint, say
    opt.read_master()
    for n, w in opt.slices(opt.states()["master"]).items():
        assert torch.equal(w, params[n].float())
    _step_and_check(params, grads, opt)
    moved = {n: (2 * p).clone() for n, p in params.items()}
    opt.rebind(moved)
    opt.read_master()
    _step_and_check(moved, grads, opt, max_norm=1.0)
    plain = _setup(states=states, seed=9)[2]
    with pytest.raises(ValueError, match="no master weights"):
        plain.read_master()


@gpu
@pytest.mark.parametrize("dtype,gdtype,master,elements", [
    (torch.bfloat16, None, False, 160_000_000), (torch.bfloat16, None, True, 160_000_000), (torch.bfloat16, torch.float32, True, 80_000_000),
    (torch.float32, None, False, 80_000_000)])
def test_8_bit_steps_whose_copies_run_ahead(dtype, gdtype, master, elements):
    """Enough elements for work items of several tiles, so that every warp fills its shared memory again
    and again, and every CTA takes several items; blocks of different size, ends of every kind."""
    sizes = [(elements // 2 + 12345,), (3, elements // 8 + 77), (elements // 16,), (5000,), (129,)]
    params, grads, opt = _setup(sizes, dtype, gdtype, seed=30, states="fp8", master=master)
    for k in range(2):
        for i, g in enumerate(grads.values()):
            flat = g.view(-1)
            g.copy_(_rand(tuple(g.shape), g.dtype, 500 + 10 * k + i, 1e-2))
            flat *= (1 + torch.arange(flat.numel(), device="cuda") // 128 % (37 + k)).to(flat.dtype)
        _step_and_check(params, grads, opt, max_norm=1.0 if k else None)


@gpu
@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("dtype,gdtype,master", [(torch.bfloat16, torch.float32, True), (torch.float32, None, False)])
def test_fp32_steps_of_several_items_a_block(dtype, gdtype, master, shift):
    params, grads, opt = _setup([(15_000_001,), (64,), (6_000_000,)], dtype, gdtype, shift=shift, seed=31, master=master)
    for k in range(2):
        _step_and_check(params, grads, opt, max_norm=1.0 if k else None)
        for i, g in enumerate(grads.values()):
            g.copy_(_rand(tuple(g.shape), g.dtype, 600 + i, 1e-3))


@gpu
def test_8_bit_steps_at_odd_addresses_of_several_items_a_block():
    params, grads, opt = _setup([(40_000_001,), (700_001,)], torch.bfloat16, shift=3, seed=32, states="fp8", master=True)
    for k in range(2):
        _step_and_check(params, grads, opt, max_norm=1.0 if k else None)
        for i, g in enumerate(grads.values()):
            g.copy_(_rand(tuple(g.shape), g.dtype, 700 + i, 1e-3))


def test_released_storage_is_refused():
    """A tensor whose storage was given back, whole (its address is 0) or in part, still has its sizes."""
    for left in (0, 15):
        x = torch.ones(4)
        x.untyped_storage().resize_(left)
        for call in (lambda: AdamW({"a": x}), lambda: grad_norm([x])):
            with pytest.raises(ValueError, match="storage"):
                call()


@gpu
def test_released_gradient_is_refused():
    p = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    opt = AdamW({"a": p})
    for dtype in (torch.bfloat16, torch.float32):
        g = torch.ones(64, dtype=dtype, device="cuda")
        g.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match="storage"):
            opt.step({"a": g})
    assert opt.step_count == 0 and bool((p == 1).all())


@gpu
def test_parameters_of_another_size_or_type_at_the_same_address():
    """`p.data` may be set to a part of itself: the address stays, the table's size is another."""
    for change in (lambda x: x[:5], lambda x: x.view(torch.bfloat16)):
        p = torch.nn.Parameter(torch.ones(64, device="cuda"))
        opt = AdamW({"a": p})
        address = p.data_ptr()
        p.data = change(p.data)
        assert p.data_ptr() == address
        with pytest.raises(RuntimeError, match="rebind"):
            opt.step({"a": torch.ones_like(p)})
        with pytest.raises(ValueError, match="another shape"):
            opt.rebind({"a": p})
        assert opt.step_count == 0
