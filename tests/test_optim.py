"""AdamW over many tensors and the gradient norm against the formulas in 64 bits.

Tolerances: u = 2^-24 is half a step of fp32.  m and v are two products and a sum of 32-bit
values (the clipping factor adds a rounding, squared in v): 8 u of the terms' sizes.  The update
lr m / (sqrt(v) + eps) adds a root, a quotient and three scalars rounded to fp32: 32 u of it, next
to 2 u of the parameter; a 16-bit parameter adds half a step of its type.  An e4m3 state is off by
at most half a step (2^-4 of the value, 2^-10 of the scale near zero).
"""
import math
import multiprocessing as mp
import os
import socket

import pytest
import torch

from weightbridge_b200 import AdamW, grad_norm

gpu = pytest.mark.gpu
U = 2.0 ** -24
SIZES = [(1,), (3, 5), (127,), (128,), (129,), (64, 300), (8192,), (8193,), (5, 7, 401), (0,), (70001,)]


def _rand(shape, dtype, seed, std=1.0, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = math.prod(shape)
    flat = torch.empty(n + shift, dtype=dtype, device="cuda")[shift:]
    flat.copy_(torch.randn(n, device="cuda", generator=g) * std)
    return flat.view(shape)


def _setup(sizes=SIZES, dtype=torch.bfloat16, gdtype=None, shift=0, seed=0, gstd=1e-2, **kw):
    params = {f"p{i}": _rand(s, dtype, seed + i, 0.05, shift) for i, s in enumerate(sizes)}
    grads = {f"p{i}": _rand(s, gdtype or dtype, 1000 + seed + i, gstd, shift) for i, s in enumerate(sizes)}
    return params, grads, AdamW(params, **{**dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1), **kw})


def _values(opt):
    """Per parameter: (start value, m, v) in 64 bits."""
    st = opt.states()
    if opt.state_bits == "fp8":
        wide = [st[k].float().view(-1, 128).double() * st[s][:, None].double() for k, s in (("exp_avg", "exp_avg_scale"), ("rms", "rms_scale"))]
        m, v = wide[0].view(-1), wide[1].view(-1) ** 2
    else:
        m, v = st["exp_avg"].double(), st["exp_avg_sq"].double()
    m, v = opt.slices(m), opt.slices(v)
    w = opt.slices(st["master"].double()) if "master" in st else None
    return m, v, w


def _step_and_check(params, grads, opt, lr=1e-2, max_norm=None, wd=0.1, no_decay=(), **kw):
    t = opt.step_count + 1
    m0, v0, w0 = _values(opt)
    before = {n: p.detach().double().clone() for n, p in params.items()}
    m0, v0 = ({n: x.clone() for n, x in d.items()} for d in (m0, v0))
    w0 = {n: x.clone() if params[n].dtype != torch.float32 else before[n] for n, x in w0.items()} if w0 else before
    norm = opt.step(grads, max_norm=max_norm, **kw)
    (b1, b2), eps = opt.betas, opt.eps
    c, live = 1.0, {n: g for n, g in grads.items() if g is not None}
    if max_norm is not None:
        total = math.sqrt(sum(float(g.double().square().sum()) for g in live.values()))
        assert abs(float(norm) - total) <= 64 * U * total          # at most 64 squares in a row in 32 bits, the rest in 64
        c = min(1.0, max_norm / (total + 1e-6))
    else:
        assert norm is None
    assert opt.step_count == t
    m1, v1, w1 = _values(opt)
    scales = {k: s for k, s in opt.states().items() if k.endswith("scale")}
    for n, p in params.items():
        if n not in live:
            assert torch.equal(p.double(), before[n]) and torch.equal(m1[n], m0[n]) and torch.equal(v1[n], v0[n])
            continue
        g = live[n].double() * c
        m, v = b1 * m0[n] + (1 - b1) * g, b2 * v0[n] + (1 - b2) * g * g
        slack = 64 * U if max_norm is not None else 0.0
        tol_m = (8 * U + slack) * (b1 * m0[n].abs() + (1 - b1) * g.abs())
        tol_v = (8 * U + 2 * slack) * v
        upd = lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
        upd_size = lr / (1 - b1 ** t) * (b1 * m0[n].abs() + (1 - b1) * g.abs()) / ((v / (1 - b2 ** t)).sqrt() + eps)
        decay = 0.0 if n in no_decay else wd
        want = w0[n] * (1 - lr * decay) - upd
        tol = 4 * U * w0[n].abs() + (32 * U + 2 * slack) * upd_size + 1e-45
        if w1 is not None and p.dtype != torch.float32:
            assert bool(((w1[n] - want).abs() <= tol).all())
            assert torch.equal(p, w1[n].to(p.dtype))
        tol = tol + torch.finfo(p.dtype).eps / 2 * want.abs() * 1.01 + torch.finfo(p.dtype).tiny * torch.finfo(p.dtype).eps
        assert bool(((p.double() - want).abs() <= tol).all()), (n, float(((p.double() - want).abs() - tol).max()))
        if not scales:
            assert bool(((m1[n] - m).abs() <= tol_m + 1e-45).all()) and bool(((v1[n] - v).abs() <= tol_v + 1e-45).all())
            continue
        if not p.numel():
            continue
        for got, x, tol_x, key in ((m1[n], m, tol_m, "exp_avg_scale"), (v1[n].sqrt(), v.sqrt(), tol_v / (2 * v.sqrt() + 1e-300), "rms_scale")):
            order = lambda y: torch.as_strided(y, (y.numel(),), (1,)) if y.is_contiguous() else y.transpose(-1, -2).reshape(-1)  # noqa: E731
            x, got, tol_x = order(x), order(got), order(tol_x)
            pad = (-x.numel()) % 128
            blocks = torch.nn.functional.pad(x, (0, pad)).view(-1, 128)
            amax = blocks.abs().amax(1)
            want_s = torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -126), 0.0)    # a scale is a normal number
            scale = want_s.repeat_interleave(128)[:x.numel()]
            tiny = (x.abs() < scale * 2.0 ** -9) & (x.abs() > 0)
            half = x.abs() * 2.0 ** -4 + scale * 2.0 ** -10
            if key == "rms_scale":      # a positive root keeps the smallest code; squares below 2^-126 may count as 0
                pos = x > 2.0 ** -63
                assert bool((got[pos] >= scale[pos] * 2.0 ** -9 * (1 - 1e-5)).all())
                half = torch.where(tiny, scale * 2.0 ** -9, half)
            least = 2.0 ** -63 if key == "rms_scale" else 1e-45     # roots of what 32 bits do not hold as normal numbers
            bad = (got - x).abs() > half * 1.0001 + tol_x + least
            assert not bool(bad.any()), (n, key, int(bad.sum()))
            assert bool((got[x == 0] == 0).all())
    return norm


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
@pytest.mark.parametrize("shift", [0, 1, 3, 4, 8])
@pytest.mark.parametrize("dtype,gdtype,master", [
    (torch.float32, None, False), (torch.bfloat16, None, False), (torch.bfloat16, torch.float32, True), (torch.bfloat16, torch.float32, False),
    (torch.float16, None, True), (torch.float16, torch.float32, False)])
def test_steps_match_the_formula(states, shift, dtype, gdtype, master):
    params, grads, opt = _setup(dtype=dtype, gdtype=gdtype, shift=shift, states=states, master=master)
    for k in range(4):
        _step_and_check(params, grads, opt, max_norm=[None, 1.0, 1e4, 0.01][k])
        for i, g in enumerate(grads.values()):
            g.copy_(_rand(tuple(g.shape), g.dtype, 77 * k + i, 10.0 ** -(k + 1)))


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_mixed_types_decay_and_missing_gradients(states):
    shapes = [(300, 5), (700,), (4096,), (33,), (9000,)]
    types = [torch.bfloat16, torch.float32, torch.float16, torch.float32, torch.bfloat16]
    params = {f"w{i}": _rand(s, d, i, 0.1) for i, (s, d) in enumerate(zip(shapes, types))}
    opt = AdamW(params, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, states=states, master=True, no_decay=["w1", "w3"])
    grads = {n: _rand(tuple(p.shape), torch.float32 if n == "w4" else p.dtype, 50 + i, 0.1) for i, (n, p) in enumerate(params.items())}
    _step_and_check(params, grads, opt, no_decay=("w1", "w3"))
    _step_and_check(params, {**grads, "w2": None}, opt, max_norm=0.5, no_decay=("w1", "w3"))
    _step_and_check(params, {n: g for n, g in grads.items() if n != "w0"}, opt, no_decay=("w1", "w3"))
    before = {n: p.clone() for n, p in params.items()}
    opt.step({}, max_norm=1.0)                                   # nothing to do; the step counts
    assert all(torch.equal(p, before[n]) for n, p in params.items()) and opt.step_count == 4
    by_rule = AdamW({n: p.clone() for n, p in params.items()}, no_decay=lambda n: n.endswith("1"))
    assert by_rule.names == list(params)


@gpu
def test_parameters_own_gradients_and_versions():
    p = torch.nn.Parameter(_rand((40, 30), torch.float32, 1))
    q = torch.nn.Parameter(_rand((17,), torch.float32, 2))
    opt = AdamW({"p": p, "q": q}, lr=0.1)
    loss = (p.square().sum() + q.sum())
    kept = (p * p).sum()
    loss.backward()
    start, version = p.detach().clone(), p._version
    opt.step()
    assert p._version > version and not torch.equal(p, start)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    q.grad = None
    held = q.detach().clone()
    opt.step(lr=0.05)
    assert torch.equal(q.detach(), held)


@gpu
def test_inference_tensors_and_no_elements():
    with torch.inference_mode():
        p = {"p": torch.ones(300, device="cuda")}
        AdamW(p, lr=0.5, weight_decay=0.0).step({"p": torch.ones(300, device="cuda")})
        assert float((p["p"] - 0.5).abs().max()) < 1e-6
    for states in ("fp32", "fp8"):
        opt = AdamW({"e": torch.empty(0, 5, device="cuda")}, states=states)
        assert float(opt.step({"e": torch.empty(0, 5, device="cuda")}, max_norm=1.0)) == 0.0 and opt.step_count == 1


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_transposed_parameters(states):
    base = _rand((130, 257), torch.float32, 3)
    params = {"t": base.t()}
    opt = AdamW(params, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, states=states)
    grads = {"t": _rand((130, 257), torch.float32, 4).t()}
    _step_and_check(params, grads, opt)
    _step_and_check(params, grads, opt, max_norm=1.0)
    with pytest.raises(ValueError, match="memory layout"):
        opt.step({"t": grads["t"].contiguous()})


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_a_step_on_gradients_that_are_not_finite_changes_nothing(states):
    for value in (math.inf, -math.inf, math.nan):
        params, grads, opt = _setup(states=states, dtype=torch.float32)
        opt.step(grads, max_norm=1.0)
        grads["p6"][77] = value
        before = {n: p.clone() for n, p in params.items()}
        st = {k: s.float().clone() for k, s in opt.states().items()}
        norm = opt.step(grads, max_norm=1.0)
        assert not math.isfinite(float(norm)) and opt.step_count == 1
        assert all(torch.equal(p, before[n]) for n, p in params.items())
        assert all(torch.equal(s.float(), st[k]) for k, s in opt.states().items())
        grads["p6"][77] = 0.5
        _step_and_check(params, grads, opt, max_norm=1.0)


@gpu
def test_extreme_gradients_in_8_bit_blocks():
    """Blocks of zeros, of subnormal numbers, and with one large value among small ones."""
    g = torch.zeros(6 * 128, device="cuda")
    g[128:256] = 1e-39
    g[256:384] = 1e-6
    g[300] = 1e3
    g[384:512] = 1e18
    g[512:640] = torch.logspace(-12, 0, 128, device="cuda")
    params = {"p": torch.ones(6 * 128, device="cuda")}
    opt = AdamW(params, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, states="fp8")
    for _ in range(3):
        _step_and_check(params, {"p": g}, opt)
    st = opt.states()
    assert all(bool(s.float().isfinite().all()) for s in st.values()) and bool(params["p"].isfinite().all())
    assert bool((st["exp_avg_scale"] > 0).all()) and bool((st["rms"].float()[256:384] > 0).all())
    assert bool((params["p"] < 1).all())                        # even the zeros decayed, and nothing blew up
    assert float((params["p"] - 1).abs().max()) < 0.5


@gpu
def test_infinite_gradients_without_clipping_stay_visible():
    """No norm, no check: the parameter turns NaN as in 32 bits, and the block's moments do not turn into numbers again."""
    for states in ("fp32", "fp8"):
        params = {"p": torch.ones(256, device="cuda")}
        opt = AdamW(params, states=states)
        g = torch.ones(256, device="cuda")
        g[3] = math.inf
        opt.step({"p": g})
        g[3] = 1.0
        opt.step({"p": g})
        p = params["p"]
        assert not math.isfinite(float(p[3])) and bool(p[128:].isfinite().all())
        assert not bool(opt.states()["exp_avg_scale" if states == "fp8" else "exp_avg"][:128].isfinite().all())


@gpu
def test_second_moment_keeps_up_in_8_bits():
    """Steady gradients of one size: the 8-bit optimizer takes the steps of the 32-bit one to the
    accuracy of its codes: m and r are each off by at most 2^-4, so an update by 2^-3 + 2^-8."""
    a = {"p": torch.zeros(4096, device="cuda")}
    b = {"p": torch.zeros(4096, device="cuda")}
    x, y = AdamW(a, lr=1e-2, weight_decay=0.0, betas=(0.9, 0.95)), AdamW(b, lr=1e-2, weight_decay=0.0, betas=(0.9, 0.95), states="fp8")
    g = {"p": _rand((4096,), torch.float32, 5).sign() * 1e-3}
    for _ in range(20):
        x.step(g)
        y.step(g)
    assert float((a["p"] - b["p"]).abs().max()) <= float(a["p"].abs().max()) * (2.0 ** -3 + 2.0 ** -8)


@gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_elements_beyond_32_bit_offsets(shift):
    """2^31 + 333 parameters in one tensor: the first step is lr along the gradient's sign, at both ends."""
    n = 2 ** 31 + 333
    flat, grad = (torch.zeros(n + shift, dtype=torch.bfloat16, device="cuda")[shift:] for _ in range(2))
    grad[:1000] = 2.0 ** -10
    grad[-1000:] = -2.0 ** -10
    opt = AdamW({"p": flat}, lr=0.25, weight_decay=0.0, states="fp8")
    norm = opt.step({"p": grad}, max_norm=1e9)
    assert abs(float(norm) - 2.0 ** -10 * math.sqrt(2000)) < 1e-6
    assert abs(float(grad_norm([grad])) - float(norm)) < 1e-9
    for part, want in ((flat[:1000], -0.25), (flat[-1000:], 0.25), (flat[1000:2000], 0.0), (flat[2 ** 31 - 5000:2 ** 31 - 4000], 0.0)):
        assert float((part.float() - want).abs().max()) < 1e-3       # half a step of bf16 at 0.25 is 2^-11
    assert int((flat != 0).sum()) == 2000


@gpu
def test_thousands_of_tensors_take_several_launches():
    n = 4100
    params = {f"p{i}": _rand((1 + i % 13,), torch.float32, i) for i in range(n)}
    grads = {k: torch.full_like(p, 0.25) for k, p in params.items()}
    flat = torch.cat(list(params.values())).double()
    opt = AdamW(params, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.0)
    norm = opt.step(grads, max_norm=1.0)
    want = 0.25 * math.sqrt(flat.numel())
    assert abs(float(norm) - want) < 1e-5 * want and opt.step_count == 1
    got = torch.cat(list(params.values())).double()
    assert float((got - (flat - 1e-2)).abs().max()) < 1e-6       # the first step is lr along the gradient's sign
    opt.step(grads)
    assert opt.step_count == 2


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_captured_step_replays_with_its_own_clock_and_rate(states):
    params, grads, opt = _setup(states=states, seed=5, master=True)
    twin, _, ref = _setup(states=states, seed=5, master=True)
    lr = torch.tensor(1e-2, device="cuda")
    opt.step(grads, lr=lr, max_norm=1.0)
    ref.step(grads, lr=1e-2, max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(grads, lr=lr, max_norm=1.0)
    for k in range(3):
        lr.fill_(1e-2 / (k + 1))
        for i, (n, g) in enumerate(grads.items()):
            g.copy_(_rand(tuple(g.shape), g.dtype, 10 * k + i, 0.1))
        graph.replay()
        want = ref.step(grads, lr=float(lr), max_norm=1.0)
        assert torch.equal(norm, want)
    assert opt.step_count == ref.step_count == 4
    assert all(torch.equal(p, twin[n]) for n, p in params.items())
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(opt.states().values(), ref.states().values()))
    with pytest.raises(ValueError, match="lr is a number"):
        opt.step(grads, lr=torch.tensor([1.0, 2.0], device="cuda"))


@gpu
def test_other_streams():
    params, grads, opt = _setup(seed=6)
    twin, _, ref = _setup(seed=6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s):
            opt.step(grads, max_norm=1.0)
        ref.step(grads, max_norm=1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(p, twin[n]) for n, p in params.items())


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_saved_and_loaded_states_and_moved_memory(states):
    params, grads, opt = _setup(states=states, seed=7, master=True)
    for _ in range(3):
        opt.step(grads, max_norm=1.0)
    saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
    copies = {n: p.clone() for n, p in params.items()}
    again = AdamW(copies, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, states=states, master=True)
    again.load_state_dict(saved)
    assert again.step_count == 3
    moved = {n: p.clone() for n, p in copies.items()}
    again.rebind(moved)
    for o in (opt, again):
        o.step(grads, max_norm=1.0)
    assert all(torch.equal(p, moved[n]) for n, p in params.items())
    with pytest.raises(ValueError, match="missing or of another"):
        again.load_state_dict({k: v for k, v in saved.items() if k != "exp_avg"})
    with pytest.raises(ValueError, match="names"):
        again.load_state_dict({**saved, "names": ["x"]})
    with pytest.raises(ValueError, match="names"):
        again.rebind({"x": moved["p0"]})
    with pytest.raises(ValueError, match="another shape"):
        again.rebind({n: p.float() for n, p in moved.items()})
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW({"p": p})
    p.data = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="rebind"):
        opt.step({"p": torch.ones(8, device="cuda")})


@gpu
def test_refusals_on_the_gpu():
    p = torch.ones(64, 64, device="cuda")
    for tensors, match in (({"a": p[:, :32]}, "holes"), ({"a": p.expand(2, 64, 64)}, "holes"), ({"a": p, "b": p}, "share memory"),
                           ({"a": p[:40], "b": p[30:]}, "share memory"), ({"a": p.long()}, "bfloat16"), ({"a": p, "b": p.cpu()}, "device"),
                           ({}, "no parameters")):
        with pytest.raises(ValueError, match=match):
            AdamW(tensors)
    with pytest.raises(ValueError, match="16-bit"):
        AdamW({"a": p}, master=True)
    opt = AdamW({"a": p, "b": torch.ones(3, dtype=torch.bfloat16, device="cuda")})
    g = torch.ones(64, 64, device="cuda")
    for grads, match in (({"a": g[:3]}, "shape"), ({"a": g.half()}, "type"), ({"c": g}, "not one of"), ({"a": g.cpu()}, "device"),
                         ({"a": g.t()}, "layout"), ({"b": g[0, :3].half()}, "type")):
        with pytest.raises(ValueError, match=match):
            opt.step(grads)
    with pytest.raises(TypeError):
        opt.step([g])
    with pytest.raises(TypeError):
        opt.step({"a": 3})
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            opt.step({"a": g}, max_norm=bad)
    with pytest.raises(ValueError, match="lr"):
        opt.step({"a": g}, lr=-1.0)
    with pytest.raises(ValueError, match="sparse"):
        opt.step({"a": g.to_sparse()})
    with pytest.raises(ValueError, match="sparse"):
        grad_norm([g.to_sparse()])
    with pytest.raises(ValueError, match="max_norm, too"):
        opt.step({"a": g}, group=object())
    with pytest.raises(ValueError, match="one value per element"):
        opt.slices(torch.zeros(3))
    for tensors, match in (([], "no tensors"), ([g.long()], "bfloat16"), ([g, g.cpu()], "device"), ([g[:, :3]], "holes")):
        with pytest.raises(ValueError, match=match):
            grad_norm(tensors)
    assert opt.step_count == 0 and bool((p == 1).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_norm(dtype, shift):
    ts = {f"g{i}": _rand(s, dtype, i, 0.5, shift) for i, s in enumerate(SIZES + [(16384,), (16385,), (300000,)])}
    want = math.sqrt(sum(float(t.double().square().sum()) for t in ts.values()))
    got = grad_norm(ts)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 64 * U * want
    assert torch.equal(got, grad_norm(list(ts.values()))) and torch.equal(got, grad_norm([None, *ts.values()]))
    assert float(grad_norm([torch.zeros(0, dtype=dtype, device="cuda")])) == 0.0
    assert float(grad_norm([torch.zeros(5, dtype=dtype, device="cuda")])) == 0.0
    many = [torch.full((1 + i % 3,), 2.0, dtype=dtype, device="cuda") for i in range(3000)]
    assert abs(float(grad_norm(many)) - math.sqrt(4 * sum(t.numel() for t in many))) < 1e-3
    for value in (math.inf, math.nan):
        ts["g4"][0] = value
        assert not math.isfinite(float(grad_norm(ts)))


def test_refusals_without_a_gpu():
    p = {"a": torch.ones(4)}
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(p)
    with pytest.raises(ValueError, match="CUDA"):
        grad_norm(p)
    for kw, match in ((dict(states="int8"), "states"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
                      (dict(eps=0.0), "eps"), (dict(eps=1e-40), "eps"), (dict(lr=math.inf), "lr"), (dict(weight_decay=-1.0), "eps"), (dict(lr=-1.0), "lr"), (dict(no_decay=["b"]), "no_decay")):
        with pytest.raises(ValueError, match=match):
            AdamW(p, **kw)


@gpu
def test_fsdp_parameters_by_their_local_tensors():
    """DTensors are refused; the views that convert_to_wb makes of them are the local tensors."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import DeviceMesh
    from torch.distributed.tensor import Shard, distribute_tensor
    from weightbridge_b200.parallel.fsdp import convert_to_wb
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = DeviceMesh("cuda", [0])
        p = distribute_tensor(torch.ones(64, 8, device="cuda"), mesh, [Shard(0)])
        g = distribute_tensor(torch.full((64, 8), 2.0, device="cuda"), mesh, [Shard(0)])
        with pytest.raises(ValueError, match="DTensor"):
            AdamW({"p": p})
        with pytest.raises(ValueError, match="DTensor"):
            grad_norm({"p": g})
        _, views = convert_to_wb({"p": p})
        opt = AdamW(views, lr=0.5, weight_decay=0.0)
        with pytest.raises(ValueError, match="DTensor"):
            opt.step({"p": g})
        norm = opt.step({"p": g.to_local()}, max_norm=1e9)
        assert abs(float(norm) - 2.0 * math.sqrt(512)) < 1e-4
        assert float((p.to_local() - 0.5).abs().max()) < 1e-6       # the first step is lr along the gradient's sign
    finally:
        dist.destroy_process_group()


def _rank(rank, port, out):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    params = {"p": torch.ones(1000, device="cuda")}
    opt = AdamW(params, lr=1e-2)
    grads = {"p": torch.full((1000,), 3.0 if rank == 0 else 4.0, device="cuda")}
    norms = [float(grad_norm(grads, group=dist.group.WORLD)), float(opt.step(grads, max_norm=1.0, group=dist.group.WORLD)),
             float(opt.step(grads if rank else {}, max_norm=1.0, group=dist.group.WORLD))]
    out.put((rank, norms, opt.step_count))
    dist.destroy_process_group()


@gpu
def test_norm_over_ranks():
    """Two ranks (gloo on the host; no kernel waits for another) share the norm and take the same step."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(out.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    for _, norms, steps in got:
        assert steps == 2
        for n, want in zip(norms, (math.sqrt(25000), math.sqrt(25000), math.sqrt(16000))):
            assert abs(n - want) < 1e-4 * want
