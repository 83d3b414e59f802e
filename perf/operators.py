"""Cases of the framework's operators beside the weight sync: what is measured, and on which sizes.

Three operators: the log probabilities of given tokens with entropy and top alternatives
(forward alone, and with the gradient of the logits), the AdamW step over many tensors (states
in 32 or 8 bits), and the global gradient norm.  ``run`` computes each in plain torch
operations where ``own`` is false, and calls the framework where it is true.

The tensors of an optimizer case are views of flat buffers in which every tensor starts at a
multiple of 128 elements (zeros between them), so the plain form is a few operations over the
flat buffers while the framework gets the dict of tensors that a trainer holds.
"""
import math

import torch

own = False

BLOCK = 128          # elements that share a scale in the 8-bit states
E4M3_MAX = 448.0
IGNORED = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# -- cases ----------------------------------------------------------------------------------------
def _logprobs(name, rows, vocab, **kw):
    case = {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "pad": 0, "dtype": "bf16", "train": False,
            "top_k": 0, "temperature": 1.0, "ignored": 0.0}
    case.update(kw)
    return case


def _adamw(name, **kw):
    case = {"name": name, "op": "adamw", "dtype": "bf16", "grad": "bf16", "states": "fp32", "master": False,
            "max_norm": 1.0, "shift": 0}
    case.update(kw)
    return case


def listed():
    return [
        # one decoded token of an 8B model: the engine returns its log probability and five alternatives
        _logprobs("token", 1, 128256, top_k=5),
        # a decode batch over a large vocabulary, sampled at 0.7, with the twenty alternatives an API offers
        _logprobs("decode_batch", 64, 151936, top_k=20, temperature=0.7),
        # scoring sampled sequences with the reference policy: forward alone, ordinary size
        _logprobs("score", 4096, 128256),
        # a training micro-batch: vocabulary padded by the trainer, policy loss and entropy bonus
        _logprobs("train", 4096, 151936, pad=128, train=True),
        # fp32 logits, a padded batch (a third of its positions ignored), temperature as sampled
        _logprobs("train_padded_batch", 777, 32000, dtype="fp32", train=True, ignored=0.35, temperature=0.8),
        # a small test model: odd vocabulary, many short rows
        _logprobs("train_small_vocab", 2047, 1001, dtype="fp16", train=True, ignored=0.1),
        # a two-layer model of 256 channels: latency counts
        _adamw("adamw_tiny", shapes="dense", layers=2, hidden=256, kv=128, ffn=688),
        # two dense layers of an 8B model with fp32 master weights and fp32 gradients, as mixed-precision trainers keep them
        _adamw("adamw_dense_master", shapes="dense", layers=2, hidden=4096, kv=1024, ffn=14336, grad="fp32", master=True),
        # one layer of 128 experts: hundreds of tensors, states in 8 bits
        _adamw("adamw_experts_8bit", shapes="experts", experts=128, hidden=2048, ffn=768, states="fp8"),
        # shards cut anywhere: odd sizes at odd addresses, fp32 parameters, 8-bit states, no clipping
        _adamw("adamw_ragged_8bit", shapes="ragged", tensors=61, largest=1500001, dtype="fp32", grad="fp32", states="fp8", max_norm=0.0,
               shift=3),
        # the norm alone (logged every step): the experts' gradients, and a small adapter's
        {"name": "norm_experts", "op": "norm", "shapes": "experts", "experts": 128, "hidden": 2048, "ffn": 768, "grad": "bf16", "shift": 0},
        {"name": "norm_ragged", "op": "norm", "shapes": "ragged", "tensors": 97, "largest": 300007, "grad": "fp32", "shift": 1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "train", "adamw", "adamw", "norm"])
    if op in ("logprobs", "train"):
        vocab = _log_int(rng, 33, 160000)
        rows = max(1, min(_log_int(rng, 1, 8192), 400_000_000 // vocab))
        top_k = 0 if op == "train" or rows > 512 else rng.choice([0, 1, 5, 20])
        return {"op": "logprobs", "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 1, 7, 64, 128]), "dtype": rng.choice(list(DTYPES)),
                "train": op == "train", "top_k": min(top_k, vocab), "temperature": rng.choice([1.0, 0.6, 0.8, 1.3]),
                "ignored": rng.choice([0.0, 0.0, 0.25])}
    shapes = {"shapes": "ragged", "tensors": _log_int(rng, 1, 600), "largest": _log_int(rng, 100, 3_000_000),
              "shift": rng.choice([0, 0, 0, 1, 3, 8])}
    if rng.random() < 0.3:
        shapes = {"shapes": "dense", "layers": rng.randint(1, 3), "hidden": 64 * rng.randint(1, 32), "kv": 64 * rng.randint(1, 8),
                  "ffn": _log_int(rng, 100, 9000), "shift": 0}
    dtype = rng.choice(list(DTYPES))
    grad = "fp32" if dtype == "fp32" else rng.choice([dtype, "fp32"])
    if op == "norm":
        return {"op": "norm", "grad": grad, **shapes}
    return {"op": "adamw", "dtype": dtype, "grad": grad, "states": rng.choice(["fp32", "fp8"]),
            "master": dtype != "fp32" and rng.random() < 0.5, "max_norm": rng.choice([0.0, 1.0]), **shapes}


def _sizes(case):
    """Elements of each tensor of an optimizer case."""
    if case["shapes"] == "dense":
        h, kv, f = case["hidden"], case["kv"], case["ffn"]
        return [h, h * h, h * kv, h * kv, h * h, h, f * h, f * h, f * h] * case["layers"]
    if case["shapes"] == "experts":
        h, f, e = case["hidden"], case["ffn"], case["experts"]
        return [e * h] + [f * h] * (3 * e)
    n, big = case["tensors"], case["largest"]
    return [big] + [1 + int((big - 1) * ((i * 0.6180339887) % 1.0) ** 3) for i in range(1, n)]


def work(case):
    if case["op"] == "logprobs":
        live = case["rows"] - int(case["rows"] * case["ignored"])
        read, wrote = live * case["vocab"], case["rows"] * (case["vocab"] + case["pad"]) if case["train"] else 0
        return {"bytes": (read + wrote) * BYTES[case["dtype"]] + case["rows"] * (16 + 12 * case["top_k"]), "flops": (6 if not case["train"] else 14) * read}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": n * BYTES[case["grad"]], "flops": 2 * n}
    p = BYTES[case["dtype"]]
    states = 16 if case["states"] == "fp32" else 4 + 16 / BLOCK
    return {"bytes": n * (p + (8 if case["master"] else p) + BYTES[case["grad"]] + states), "flops": 16 * n}


# -- inputs ---------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        return _prepare_logprobs(case, g)
    return _prepare_tensors(case, g)


def _prepare_logprobs(case, g):
    rows, vocab, cols, dtype = case["rows"], case["vocab"], case["vocab"] + case["pad"], DTYPES[case["dtype"]]
    logits = torch.empty(rows, cols, dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=g)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    # sampled tokens are likely ones: most stand out of their row
    at = logits.gather(1, tokens[:, None])
    logits.scatter_(1, tokens[:, None], at + 16 * torch.rand(rows, 1, device="cuda", generator=g).to(dtype))
    order = torch.randperm(rows, device="cuda", generator=g)
    tokens[order[:int(rows * case["ignored"])]] = IGNORED
    state = {"case": case, "logits": logits, "tokens": tokens}
    if case["train"]:
        state["logits"].requires_grad_()
        state["g_logprobs"] = torch.randn(rows, device="cuda", generator=g) / rows      # advantages over the batch
        state["g_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")           # entropy bonus
    return state


def _flat(n, shift, dtype):
    """n zeros whose first element lies `shift` elements behind an aligned address."""
    return torch.zeros(n + shift, dtype=dtype, device="cuda")[shift:]


def _prepare_tensors(case, g):
    sizes, starts, n = _sizes(case), [], 0
    for s in sizes:
        starts.append(n)
        n += -(-s // BLOCK) * BLOCK
    spans = list(zip(starts, sizes))
    real = torch.zeros(n, dtype=torch.bool, device="cuda")
    for a, s in spans:
        real[a:a + s] = True

    def filled(dtype, std, shift=0):
        return _flat(n, shift, dtype).normal_(0.0, std, generator=g).mul_(real)

    def named(flat):
        return {"model.%d.weight" % i: flat[a:a + s] for i, (a, s) in enumerate(spans)}

    grad = filled(DTYPES[case["grad"]], 1e-3, case["shift"])
    state = {"case": case, "grad": grad, "grads": named(grad), "n": n, "tensors": len(sizes)}
    if case["op"] == "norm":
        return state
    param = filled(DTYPES[case["dtype"]], 0.02, case["shift"])
    step = 100
    exp_avg = filled(torch.float32, 4e-4)
    rms = filled(torch.float32, 8e-4).abs_().add_(1e-4 * real)
    if case["states"] == "fp32":
        saved = {"exp_avg": exp_avg, "exp_avg_sq": rms * rms}
    else:
        q, s = _quantise(exp_avg)
        r, t = _quantise(rms)
        saved = {"exp_avg": q, "exp_avg_scale": s, "rms": r, "rms_scale": t}
    if case["master"]:      # the parameters are the rounded master weights
        saved["master"] = param.float() * (1 + 2.0 ** -11 * torch.rand(n, device="cuda", generator=g))
    state.update(param=param, step=step, saved=saved, lr=1e-5, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    if own:                 # the optimizer that a trainer resumed, instead of its bare states
        from weightbridge_b200 import AdamW
        opt = AdamW(named(param), lr=state["lr"], betas=state["betas"], eps=state["eps"], weight_decay=state["weight_decay"],
                    states=case["states"], master=case["master"])
        opt.load_state_dict({**opt.state_dict(), "step": step, **saved})
        state["opt"] = opt
        del state["saved"]
    return state


# -- one pass -------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state["grad"]).float()
    return _own_adamw(state) if own else _plain_adamw(state)


def _own_logprobs(state):
    from weightbridge_b200 import token_logprobs
    case = state["case"]
    out = token_logprobs(state["logits"], state["tokens"], vocab=case["vocab"], temperature=case["temperature"], top_k=case["top_k"])
    got = {"logprobs": out.logprobs, "entropy": out.entropy}
    if case["top_k"]:
        got.update(top_logprobs=out.top_logprobs, top_ids=out.top_ids)
    if case["train"]:
        got["d_logits"], = torch.autograd.grad((out.logprobs, out.entropy), state["logits"], (state["g_logprobs"], state["g_entropy"]))
    return got


def _plain_logprobs(state):
    case, vocab = state["case"], state["case"]["vocab"]
    full = state["logits"].detach()
    x = full[:, :vocab].float()
    live = state["tokens"] != IGNORED
    token = state["tokens"].clamp(min=0)[:, None]
    z = (x - x.amax(1, keepdim=True)) / case["temperature"]
    logp = z - z.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    entropy = -(p * logp).sum(1)
    got = {"logprobs": torch.where(live, logp.gather(1, token)[:, 0], 0.0), "entropy": torch.where(live, entropy, 0.0)}
    if case["top_k"]:
        # distinct whole numbers in the order wanted: by the logit, then the lower id first
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits) * 2 ** 31 - torch.arange(vocab, device=x.device)
        ids = key.topk(case["top_k"], dim=1).indices
        got["top_logprobs"] = torch.where(live[:, None], logp.gather(1, ids), -math.inf)
        got["top_ids"] = torch.where(live[:, None], ids, -1)
    if case["train"]:
        g_lp, g_h = (torch.where(live, state[k], 0.0)[:, None] for k in ("g_logprobs", "g_entropy"))
        d = -p * (g_lp + g_h * (logp + entropy[:, None]))
        d.scatter_add_(1, token, g_lp)
        got["d_logits"] = torch.zeros_like(full)
        got["d_logits"][:, :vocab] = d / case["temperature"]
    return got


def _own_norm(state):
    from weightbridge_b200 import grad_norm
    return grad_norm(state["grads"])


def _plain_norm(grad):
    return grad.double().square().sum().sqrt()


def _own_adamw(state):
    case, opt = state["case"], state["opt"]
    norm = opt.step(state["grads"], max_norm=case["max_norm"] or None)
    got = {"params": state["param"], **opt.states()}
    if norm is not None:
        got["norm"] = norm
    return got


def _quantise(x):
    """Blocks of 128 values as e4m3 and the fp32 scales they are multiplied with."""
    b = x.view(-1, BLOCK)
    amax = b.abs().amax(1)
    scale = torch.where(amax > 0, (amax / torch.full_like(amax, E4M3_MAX)).clamp(min=2.0 ** -126), 1.0)
    q = (b * (1.0 / scale)[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn).view(-1), scale


def _values(q, scale):
    return (q.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _plain_adamw(state):
    case, saved = state["case"], state["saved"]
    (b1, b2), lr = state["betas"], state["lr"]
    state["step"] += 1
    c1, c2 = 1 - b1 ** state["step"], 1 - b2 ** state["step"]
    g = state["grad"].float()
    got = {"params": state["param"]}
    if case["max_norm"]:
        norm = _plain_norm(state["grad"])
        g = g * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        got["norm"] = norm.float()
    small = case["states"] == "fp8"
    m = _values(saved["exp_avg"], saved["exp_avg_scale"]) if small else saved["exp_avg"]
    v = _values(saved["rms"], saved["rms_scale"]).square() if small else saved["exp_avg_sq"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = saved["master"] if case["master"] else state["param"].float()
    p = p * (1 - lr * state["weight_decay"]) - (lr / c1) * m / ((v / c2).sqrt() + state["eps"])
    state["param"].copy_(p)
    if case["master"]:
        saved["master"] = p
    if small:
        saved["exp_avg"], saved["exp_avg_scale"] = _quantise(m)
        r = v.sqrt()
        q, saved["rms_scale"] = _quantise(r)
        # a positive value keeps the smallest code, so that no denominator becomes zero
        saved["rms"] = torch.where((r > 0) & (q.float() == 0), 2.0 ** -9, q.float()).to(torch.float8_e4m3fn)
    else:
        saved["exp_avg"], saved["exp_avg_sq"] = m, v
    return {**got, **saved}


# -- the same from the definitions, in 64 bits ----------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, state)
    if case["op"] == "norm":
        return torch.linalg.vector_norm(state["grad"].double())
    return _exact_adamw(case, state)


def _exact_logprobs(case, state):
    vocab, t, out = case["vocab"], case["temperature"], []
    for row in range(0, case["rows"], 256):
        part = slice(row, row + 256)
        full = state["logits"].detach()[part]
        x = full[:, :vocab].double().div(t)
        tok, n = state["tokens"][part], full.shape[0]
        keep = tok.ge(0).double()
        lse = torch.logsumexp(x, 1)
        prob = torch.softmax(x, 1)
        h = lse - (prob * x).sum(1)
        i = torch.arange(n, device=x.device)
        got = {"logprobs": keep * (x[i, tok.clamp(min=0)] - lse), "entropy": keep * h}
        if case["top_k"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
            lp = torch.gather(x, 1, order) - lse[:, None]
            got["top_logprobs"] = lp.masked_fill(keep[:, None] == 0, -math.inf)
            got["top_ids"] = order.masked_fill(keep[:, None] == 0, -1)
        if case["train"]:
            glp, gh = (keep * state[k][part].double() for k in ("g_logprobs", "g_entropy"))
            one = torch.zeros_like(prob)
            one[i, tok.clamp(min=0)] = 1.0
            d = glp[:, None] * (one - prob) - gh[:, None] * prob * (x - lse[:, None] + h[:, None])
            got["d_logits"] = torch.zeros(full.shape, dtype=torch.float64, device=x.device)
            got["d_logits"][:, :vocab] = d / t
            if case["rows"] * vocab > 100_000_000:      # 64 bits of all rows would take more memory than they tell
                got["d_logits"] = got["d_logits"].to(torch.float32)
        out.append(got)
    return {k: torch.cat([o[k] for o in out]).double() if k != "top_ids" else torch.cat([o[k] for o in out]) for k in out[0]}


def _exact_adamw(case, state):
    saved, t = state["saved"], state["step"] + 1
    (b1, b2), eps, lr = state["betas"], state["eps"], state["lr"]
    g = state["grad"].double()
    norm = torch.linalg.vector_norm(g)
    if case["max_norm"]:
        g *= min(1.0, case["max_norm"] / (norm.item() + 1e-6))

    def wide(name, scale):
        return saved[name].double() * saved[scale].double().repeat_interleave(BLOCK)

    if case["states"] == "fp8":
        m, v = wide("exp_avg", "exp_avg_scale"), wide("rms", "rms_scale") ** 2
    else:
        m, v = saved["exp_avg"].double(), saved["exp_avg_sq"].double()
    m = m.mul_(b1).add_(g, alpha=1 - b1)
    v = v.mul_(b2).add_(g.square_(), alpha=1 - b2)
    start = saved["master"] if case["master"] else state["param"]
    new = start.double() * (1 - lr * state["weight_decay"])
    new -= lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    got = {"params": new}
    if case["master"]:
        got["master"] = new
    if case["max_norm"]:
        got["norm"] = norm
    if case["states"] == "fp32":
        return {**got, "exp_avg": m, "exp_avg_sq": v}

    def narrow(x):
        blocks = x.reshape(-1, BLOCK)
        top = blocks.abs().max(dim=1).values
        s = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        return (blocks / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(-1), s

    q, got["exp_avg_scale"] = narrow(m)
    r, got["rms_scale"] = narrow(v.sqrt())
    got["exp_avg"] = q.to(torch.float8_e4m3fn).double()
    got["rms"] = torch.where(r > 0, r.clamp(min=2.0 ** -9), r).to(torch.float8_e4m3fn).double()
    return got
