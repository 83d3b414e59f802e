"""Token log probabilities, entropy and alternatives against the definitions in 64 bits.

Tolerances (u = 2^-24, half a step of fp32) follow the kernel's arithmetic.  With z = (x - max) / T:
z carries 3 |z| u (difference, reciprocal temperature, product); the exponential's documented
error is (2 + 1.2 |z|) steps; a thread adds at most ``seq`` terms in a row before the tree.  So
ln S is off by at most u (seq + 64 + 6 E|z| + 4) with E over the row's own distribution, a log
probability by that and 4 |z_t| u, and A / S likewise with the second moment of z.  Outputs of
16 bits add half a step of their type.
"""
import math

import pytest
import torch

from weightbridge_b200 import token_logprobs

gpu = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _oracle(logits, tokens, vocab, temperature=1.0, ignore_index=-100):
    """(logprobs, entropy, logp, keep, z) of 2-D logits in 64 bits."""
    x = logits.detach()[:, :vocab].double()
    m = x.amax(1, keepdim=True)
    empty = m[:, 0] == -math.inf
    z = (x - torch.where(m == -math.inf, 0.0, m)) / temperature
    s = z.exp().sum(1, keepdim=True)
    logp = z - s.log()
    p = torch.where(empty[:, None], 0.0, logp.exp())
    h = -torch.where(p > 0, p * logp, torch.where(p == 0, 0.0, math.nan)).sum(1)
    keep = tokens != ignore_index
    lp = logp.gather(1, tokens.long().clamp(0, vocab - 1)[:, None])[:, 0]
    lp = torch.where(empty, -math.inf, lp)
    lp = torch.where((tokens < 0) | (tokens >= vocab), math.nan, lp)
    # fp32 outputs: a log probability below -3.4e38 (the lowest value's, at a temperature below 1) is -inf
    lp = torch.where(lp < -3.4028236e38, -math.inf, lp)
    logp = torch.where(logp < -3.4028236e38, -math.inf, logp)
    return torch.where(keep, lp, 0.0), torch.where(keep, h, 0.0), torch.where(empty[:, None], -math.inf, logp), keep, z, p


def _bounds(z, p, logprobs, vocab):
    seq = max(vocab / 256, 64)
    za = torch.where(p > 0, z.abs(), 0.0)
    e1, e2 = (p * za).sum(1).nan_to_num(), (p * za * za).sum(1).nan_to_num()     # NaN: a row that is not compared by size
    ln = U * (seq + 64 + 6 * e1 + 4)
    lp = ln + 8 * U * logprobs.abs().nan_to_num(posinf=0.0) + 8 * U * e1
    return lp, ln + U * ((seq + 64) * 2 * e1 + 8 * (e1 + e2))


def _close(got, want, tol, what):
    got, want = got.detach().double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    fin = want.isfinite()
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), what
    off = (got - want).abs()[fin] - (tol[fin] if isinstance(tol, torch.Tensor) else tol)
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want).abs()[fin].max()))


def _check(logits, tokens, vocab=None, temperature=1.0, top_k=0, grad=True):
    """One call on [rows, columns] logits against the oracle, with gradients."""
    vocab = vocab or logits.shape[1]
    leaf = logits.detach().requires_grad_(grad)
    out = token_logprobs(leaf, tokens, vocab=vocab, temperature=temperature, top_k=top_k)
    lp, h, logp, keep, z, p = _oracle(logits, tokens, vocab, temperature)
    tol_lp, tol_h = _bounds(z, p, lp, vocab)
    assert out.logprobs.dtype == out.entropy.dtype == torch.float32
    _close(out.logprobs, lp, tol_lp, "logprobs")
    _close(out.entropy, h, tol_h, "entropy")
    if top_k:
        x = logits.detach()[:, :vocab].double()
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
        want = logp.gather(1, ids)
        assert torch.equal(out.top_ids, torch.where(keep[:, None], ids, -1))
        tol = tol_lp[:, None] + 8 * U * want.abs().nan_to_num(posinf=0.0)
        _close(out.top_logprobs, torch.where(keep[:, None], want, -math.inf), tol, "top_logprobs")
        assert not out.top_logprobs.requires_grad
    if grad:
        g = torch.Generator(device="cuda").manual_seed(1)
        g1, g2 = (torch.randn(tokens.shape, device="cuda", generator=g) for _ in range(2))
        d, = torch.autograd.grad((out.logprobs, out.entropy), leaf, (g1, g2))
        _check_grad(d, g1, g2, lp, h, logp, p, keep, tokens, vocab, temperature, tol_lp, tol_h)
    return out


def _check_grad(d, g1, g2, lp, h, logp, p, keep, tokens, vocab, temperature, tol_lp, tol_h):
    live = keep & ~torch.isneginf(logp).all(1)
    a, b = (torch.where(live, g, 0.0).double()[:, None] for g in (g1, g2))
    one = torch.zeros_like(p).scatter_(1, tokens.long().clamp(0, vocab - 1)[:, None], 1.0)
    fl = torch.where(p > 0, logp, 0.0)
    want = (a * (one - p) - b * p * (fl + h[:, None])) / temperature
    size = p * (a.abs() + b.abs() * (fl.abs() + h[:, None])) + one * a.abs()
    tol = size * (U * (16 + 8 * fl.abs()) + tol_lp[:, None]) + p * b.abs() * (tol_lp + tol_h)[:, None]
    # p = 2^z 2^-f with |f| <= 1/2, and a 2^z below the normal numbers of fp32 (2^-126) may be taken as
    # 0: so may a probability below 2^-125.5
    tol = tol + 2.0 ** -125.5 * (a.abs() + b.abs() * (fl.abs() + h[:, None]))
    half = torch.finfo(d.dtype).eps / 2
    tol = tol / temperature * 1.01 + half * want.abs() * 1.01 + torch.finfo(d.dtype).tiny * torch.finfo(d.dtype).eps
    assert torch.equal(d[:, vocab:], torch.zeros_like(d[:, vocab:]))
    assert torch.equal(d[~live], torch.zeros_like(d[~live]))
    _close(d[:, :vocab][live], want[live], tol[live], "d_logits")


def _inputs(rows, cols, dtype, seed=0, std=3.0, vocab=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, device="cuda", generator=g) * std).to(dtype)
    t = torch.randint(0, vocab or cols, (rows,), device="cuda", generator=g)
    return x, t


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 33), (7, 255), (4, 1000), (3, 1001), (2, 2048), (2, 2049), (3, 4097), (2400, 1500), (2400, 9001),
                                        (33, 5003), (1, 128256), (2, 151937)])
def test_sizes_and_types(dtype, rows, vocab):
    x, t = _inputs(rows, vocab, dtype)
    _check(x, t, temperature=0.8, top_k=min(vocab, 5))


@gpu
@pytest.mark.parametrize("rows", [1, 2, 18, 19, 37, 74, 75, 148, 149, 300])
def test_row_counts_around_the_splits(rows):
    x, t = _inputs(rows, 32000, torch.bfloat16, seed=rows)
    _check(x, t, top_k=3)


@gpu
@pytest.mark.parametrize("pad", [1, 7, 64, 500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_columns_take_no_part(pad, dtype):
    x, t = _inputs(9, 1999 + pad, dtype, vocab=1999)
    x[:, 1999:] = math.nan
    _check(x, t, vocab=1999, top_k=20)
    x, t = _inputs(3, 20011 + pad, dtype, vocab=20011)
    x[:, 20011:] = math.inf
    _check(x, t, vocab=20011, top_k=20)


@gpu
@pytest.mark.parametrize("top_k", [1, 2, 20, 31, 32])
@pytest.mark.parametrize("vocab", [32, 700, 9000, 50257])
def test_alternatives_with_ties(top_k, vocab):
    x, t = _inputs(6, vocab, torch.bfloat16, std=0.5)          # coarse values: many ties
    x[1] = 0.25                                                 # a row of one value: the lowest ids
    x[2] = (torch.arange(vocab, device="cuda") % 3).to(x.dtype)
    x[3] = -0.0
    x[3, ::2] = 0.0                                             # both zeros are the same value
    x[4] = torch.arange(vocab, device="cuda").to(x.dtype)      # ascending: the last ones
    x[5] = -torch.arange(vocab, device="cuda").to(x.dtype)
    _check(x, t, top_k=top_k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 999, 3001, 70001])
def test_masked_columns_and_empty_rows(dtype, vocab):
    low = torch.finfo(dtype).min
    x, t = _inputs(10, vocab, dtype, seed=3)
    x[0, ::2] = -math.inf
    x[1] = -math.inf                                            # empty
    x[2] = -math.inf
    x[2, vocab // 2] = 1.5                                      # one column left
    t[2] = vocab // 2
    x[3, 1:] = low
    x[4] = low                                                  # the type's lowest value everywhere: uniform
    x[5] = -math.inf
    x[5, :3] = low
    x[6, vocab // 3:] = -math.inf
    t[6] = vocab - 1                                            # the token itself is masked
    x[7] = torch.finfo(dtype).max
    x[8, 0], t[8] = torch.finfo(dtype).max, 0
    t[9] = -100
    for temperature in (1.0, 0.25):
        _check(x, t, temperature=temperature, top_k=min(vocab, 20))


@gpu
@pytest.mark.parametrize("vocab", [50, 3000, 40000])
def test_nan_and_infinity_stay_in_their_row(vocab):
    x, t = _inputs(6, vocab, torch.bfloat16, seed=4)
    x[1, vocab - 1] = math.nan
    x[2, 5] = math.inf
    x[3] = -math.inf
    x[3, 7] = math.nan
    t[4] = vocab                                                # no such token
    leaf = x.detach().requires_grad_()
    out = token_logprobs(leaf, t, top_k=20)
    assert out.logprobs.isnan().tolist() == [False, True, True, True, True, False]
    assert out.entropy.isnan().tolist() == [False, True, True, True, False, False]
    assert bool(((out.top_ids >= 0) & (out.top_ids < vocab)).all())
    good = torch.tensor([0, 5], device="cuda")
    _check(x[good], t[good], top_k=20)
    d, = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), leaf)
    assert bool(d[good].isfinite().all()) and bool(d[4].isnan().all())
    t[4] = -1                                                   # nor this
    assert bool(token_logprobs(x, t).logprobs[4].isnan())


@gpu
def test_ignored_rows_are_not_read():
    x, t = _inputs(8, 5000, torch.float16)
    t[::3] = -100
    x[::3] = math.nan
    out = _check(x, t, top_k=4)
    assert out.top_ids[0].tolist() == [-1] * 4
    t[::3] = 7                                                  # another mark, a token's own number
    out = token_logprobs(x, t, ignore_index=7)
    assert bool((out.logprobs[::3] == 0).all()) and bool(out.logprobs.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [101, 3333, 20001])
def test_strided_batches_and_int32_tokens(dtype, vocab):
    """The usual shift: logits[:, :-1] against tokens[:, 1:]; neither is copied, rows at any alignment."""
    g = torch.Generator(device="cuda").manual_seed(5)
    full = torch.randn(3, 6, vocab + 4, device="cuda", generator=g).to(dtype)
    ids = torch.randint(0, vocab, (3, 6), device="cuda", generator=g)
    for view in (full[:, :-1, :vocab], full[:, :-1, 3:vocab + 3], full.transpose(0, 1)[:5, :, 1:vocab + 1].transpose(0, 1)):
        tok = ids[:, 1:]
        want = token_logprobs(view.reshape(15, vocab).clone(), tok.reshape(15), top_k=3)
        for tokens in (tok, tok.int(), tok.contiguous(), tok.t().contiguous().t()):
            out = token_logprobs(view, tokens, top_k=3)
            assert out.logprobs.shape == (3, 5) and out.top_ids.shape == (3, 5, 3)
            _, _, _, _, z, p = _oracle(view.reshape(15, vocab), tok.reshape(15), vocab)
            tol, tol_h = _bounds(z, p, want.logprobs.double(), vocab)       # another alignment adds in another order
            _close(out.logprobs.reshape(15), want.logprobs, 2 * tol, "logprobs")
            _close(out.entropy.reshape(15), want.entropy, 2 * tol_h, "entropy")
            assert torch.equal(out.top_ids.reshape(15, 3), want.top_ids)
    leaf = full.detach().requires_grad_()
    out = token_logprobs(leaf[:, :-1, :vocab], ids[:, 1:])
    d, = torch.autograd.grad(out.logprobs.sum(), leaf)                   # an expanded gradient
    p = torch.softmax(full[:, :-1, :vocab].double(), -1)
    want = torch.zeros_like(p).scatter_(-1, ids[:, 1:, None], 1.0) - p
    assert torch.equal(d[:, -1], torch.zeros_like(d[:, -1]))
    tol = want.abs() * torch.finfo(dtype).eps / 2 + p * U * (vocab / 256 + 200)
    _close(d[:, :-1, :vocab], want, tol + 1e-40, "grad")
    lead = torch.randn(2, 1, 3, 1, 50, device="cuda")                    # leading dimensions that merge
    assert token_logprobs(lead, torch.zeros(2, 1, 3, 1, dtype=torch.long, device="cuda")).logprobs.shape == (2, 1, 3, 1)
    assert token_logprobs(lead[0, 0, 0, 0], torch.tensor(3, device="cuda")).logprobs.shape == ()


@gpu
def test_gradient_against_differences():
    """Differences of the 64-bit value, step 1e-5: exact to 1e-9 of the second derivative, far below fp32."""
    x, t = _inputs(4, 37, torch.float32, seed=6, std=1.0)
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, t, temperature=0.7)
    d, = torch.autograd.grad((out.logprobs * 0.5 - 0.3 * out.entropy).sum(), leaf)

    def value(y):
        logp = torch.log_softmax(y / 0.7, 1)
        return (0.5 * logp.gather(1, t[:, None])[:, 0] + 0.3 * (logp.exp() * logp).sum(1))

    for j in range(37):
        e = torch.zeros_like(x, dtype=torch.float64)
        e[:, j] = 1e-5
        diff = (value(x.double() + e) - value(x.double() - e)) / 2e-5
        assert float((diff - d[:, j].double()).abs().max()) < 2e-6          # |d| < 2: a few dozen steps of fp32


@gpu
def test_partial_gradients_none_and_second_derivative():
    x, t = _inputs(5, 300, torch.float32)
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, t)
    only_h, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
    only_lp, = torch.autograd.grad(out.logprobs.sum(), leaf, retain_graph=True)
    both, = torch.autograd.grad(out.entropy.sum() + out.logprobs.sum(), leaf, retain_graph=True)
    assert torch.allclose(only_h + only_lp, both, rtol=1e-5, atol=1e-6)
    changed = x.clone().requires_grad_()
    view = changed * 1.0
    late = token_logprobs(view, t).logprobs.sum()
    view.detach().zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.logprobs.sum(), leaf, create_graph=True)
    shared = torch.randn(1, 300, device="cuda", requires_grad=True)          # broadcast input: gradients add up
    d, = torch.autograd.grad(token_logprobs(shared.expand(5, 300), t).logprobs.sum(), shared)
    want = sum(torch.autograd.grad(torch.log_softmax(shared, 1)[0, int(k)], shared)[0] for k in t)
    assert torch.allclose(d, want, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        assert not token_logprobs(leaf, t).logprobs.requires_grad


@gpu
@pytest.mark.parametrize("temperature", [1e-30, 1e-6, 1e-2, 50.0, 1e6, 1e30])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperatures(temperature, dtype):
    """From one-hot rows to uniform ones; z is finite or -inf in between, and exact ties stay ties."""
    x, t = _inputs(6, 3001, dtype, seed=11)
    t[0] = int(x[0].argmax())
    x[1, 5] = x[1, 7] = 30.0                                     # two largest
    t[1] = 7
    _check(x, t, temperature=temperature, top_k=5, grad=temperature >= 1e-2)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1500, 40000])
def test_rows_that_outgrow_their_beginning(dtype, vocab):
    """The largest logits come last, a little or far above the first ones (2^20 to 2^200 times as
    probable), in steps, and below them."""
    x, t = _inputs(8, vocab, dtype, seed=12, std=1.0)
    for row, up in enumerate((15.0, 40.0, 60.0, 80.0, 140.0)):
        x[row, -3:] += up
    x[5] += torch.linspace(-60, 60, vocab, device="cuda").to(dtype)
    x[6] += torch.linspace(60, -60, vocab, device="cuda").to(dtype)
    x[7, :vocab // 2] -= 200.0
    t[::2] = vocab - 2
    _check(x, t, top_k=10)
    x *= 1000.0                                                 # large logits, far apart
    _check(x, t, top_k=10, grad=False)


@gpu
@pytest.mark.parametrize("vocab", [616, 20000])
def test_jumps_of_every_size(vocab):
    """A late column J nats above the others, J = 1 .. 96: neither sum loses bits to the reference's distance."""
    x, t = _inputs(96, vocab, torch.float32, seed=13, std=1.0)
    x[:, -40] = x[:, :-40].amax(1) + torch.arange(1, 97, device="cuda")
    x[:, -7] = x[:, -40] - 1.5
    t[::2] = vocab - 40
    _check(x, t, top_k=3)
    _check(x * 0.31, t, temperature=0.31, grad=False)


@gpu
def test_no_rows():
    x = torch.randn(0, 64, device="cuda", requires_grad=True)
    out = token_logprobs(x, torch.zeros(0, dtype=torch.long, device="cuda"), top_k=3)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 3)
    d, = torch.autograd.grad(out.logprobs.sum(), x)
    assert d.shape == (0, 64)


@gpu
def test_rows_beyond_32_bit_offsets():
    """33000 rows of 70000 columns: element offsets past 2^31."""
    x = torch.zeros(33000, 70000, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(70000, device="cuda").to(x.dtype)
    t = torch.zeros(33000, dtype=torch.long, device="cuda")
    t[-1] = 69999
    out = token_logprobs(x, t, top_k=2)
    last = token_logprobs(x[-1:].clone(), t[-1:], top_k=2)
    assert torch.equal(out.top_ids[-1], last.top_ids[0])
    assert abs(float(out.logprobs[-1] - last.logprobs[0])) < 1e-4
    assert abs(float(out.logprobs[100]) + math.log(70000)) < 1e-4
    leaf = x.requires_grad_()
    d, = torch.autograd.grad(token_logprobs(leaf, t).logprobs, leaf, torch.ones(33000, device="cuda"))
    assert float(d[-1, 69999]) > 0.9 and float(d[100, 0]) > 0.9 and abs(float(d[-1].float().sum())) < 0.05


@gpu
def test_other_streams_and_repeatable_bits():
    x, t = _inputs(64, 50000, torch.bfloat16, seed=8)
    a = token_logprobs(x, t, top_k=8)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2, s1, s2):
        with torch.cuda.stream(s):
            outs.append(token_logprobs(x, t, top_k=8))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(a, o))


@gpu
def test_captured_and_replayed():
    x, t = _inputs(40, 9001, torch.bfloat16, seed=9)
    static = x.clone().requires_grad_()
    g1 = torch.randn(40, device="cuda")

    def call():
        out = token_logprobs(static, t, top_k=4)
        d, = torch.autograd.grad((out.logprobs, out.entropy), static, (g1, g1))
        return [t.detach() for t in (*out, d)]      # no graph of the leaf outlives the call

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    y, t2 = _inputs(40, 9001, torch.bfloat16, seed=10)
    with torch.no_grad():
        static.copy_(y)
    t.copy_(t2)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def test_refusals():
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)

    def refused(match, logits=x, tokens=t, **kw):
        with pytest.raises(ValueError, match=match):
            token_logprobs(logits, tokens, **kw)

    refused("CUDA tensors")
    refused("bfloat16, float16 or float32", x.double())
    refused("bfloat16, float16 or float32", x.long())
    refused("int64 or int32", tokens=t.float())
    refused("do not match", tokens=t[:3])
    refused("do not match", tokens=t[:, None])
    refused("vocabulary dimension", torch.tensor(1.0), torch.tensor(0))
    for v in (0, -1, 11):
        refused("vocab must be", vocab=v)
    for k in (-1, 11, 33):
        refused("top_k must be", top_k=k)
    refused("top_k must be between 0 and 32", torch.randn(4, 100), top_k=33)
    refused("top_k must be between 0 and 3", vocab=3, top_k=4)
    refused("at most 2097152 columns", torch.empty(1, 2 ** 21 + 1, dtype=torch.float16), torch.zeros(1, dtype=torch.long), top_k=1)
    refused("2\\^30 columns", torch.empty(1, dtype=torch.float16).expand(1, 2 ** 30 + 1), torch.zeros(1, dtype=torch.long))
    for v in (0.0, -1.0, math.nan, math.inf, 1e-60, 1e60):
        refused("temperature", temperature=v)
    refused("contiguous", torch.randn(10, 4).t())
    refused("vocab must be", torch.randn(4, 0))
    refused("sparse", x.to_sparse())
    with pytest.raises(TypeError):
        token_logprobs([[1.0]], t)
