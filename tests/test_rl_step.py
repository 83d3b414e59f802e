"""The operators together, as an RL step uses them: score the rollout's tokens, differentiate the
policy loss, clip and step the parameters, sync them, and check that the rollout serves them."""
import math

import pytest
import torch

from weightbridge_b200 import AdamW, PolicyGap, TransferConfig, WeightSender, grad_norm, policy_gap, token_logprobs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("states", ["fp32", "fp8"])
def test_step_sync_and_check(states):
    import threading
    from weightbridge_b200 import MegatronLayout, SGLangLayout, WeightReceiver, WeightReceiverController
    from weightbridge_b200.models.arch import get_arch
    torch.cuda.set_device(0)
    arch = get_arch("tiny-qwen3-moe")                    # 1000 tokens, padded by the layouts
    cfg = TransferConfig(mode="gpu_direct", connect_timeout_s=60, sync_timeout_s=60)
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(3, 17, arch.hidden, device="cuda", dtype=torch.bfloat16, generator=g)
    with WeightReceiverController(worker_num=1, timeout_s=30) as ctl:
        rl = SGLangLayout(arch, tp=1)
        rp = rl.allocate(device="cuda:0", dtype=torch.bfloat16)
        rm, rv = rl.to_wb(rp)
        sl = MegatronLayout(arch, tp=1)
        sp = sl.allocate(device="cuda:0", dtype=torch.bfloat16, seed=1)
        sm, sv = sl.to_wb(sp)
        head = next(n for n in sp if "output_layer" in n)
        opt = AdamW(sp, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, states=states, master=True,
                    no_decay=lambda n: "norm" in n)
        rollout_head = next(t for n, t in rp.items() if "lm_head" in n)
        with WeightReceiver(ctl.ipc_name, 0, rm, state_dict=rv, config=cfg) as recv, WeightSender("gpu_direct", [ctl.serve()], config=cfg) as s:
            s.connect(sm)

            def sync(step):
                th = threading.Thread(target=lambda: recv.request_update(timeout=30))
                th.start()
                s.send(sv, version=step)
                th.join(30)
                assert recv.weights_version == step

            def rollout():                               # one token a row, with the alternatives it returns
                out = token_logprobs(h @ rollout_head.t(), tokens, vocab=arch.vocab, top_k=5)
                kept = tokens != -100
                assert bool((out.top_ids < arch.vocab).all()) and bool((out.top_logprobs[..., 0] >= out.logprobs)[kept].all())
                return out.logprobs

            tokens = torch.randint(0, arch.vocab, (3, 17), device="cuda", generator=g)
            tokens[2, 9:] = -100                         # a padded batch
            sync(0)
            for step in range(1, 3):
                behaviour = rollout()
                leaf = sp[head].detach().requires_grad_()
                out = token_logprobs(h @ leaf.t(), tokens, vocab=arch.vocab)
                assert s.check_policy(h @ sp[head].t(), tokens, behaviour, version=step - 1, vocab=arch.vocab, tolerance=0.0).tokens == 43
                keep = tokens != -100
                ratio = (out.logprobs - behaviour).exp()
                (-(ratio * torch.where(keep, 1.0, 0.0)).sum() / 43 - 0.01 * out.entropy.sum() / 43).backward()
                grads = {n: leaf.grad if n == head else torch.full_like(p, 1e-4) for n, p in sp.items()}
                before = sp[head].clone()
                norm = opt.step(grads, max_norm=0.5)
                assert torch.equal(norm, grad_norm(grads)) and not torch.equal(before, sp[head])
                # what the rollout holds is now one step old
                assert s.check_policy(h @ sp[head].t(), tokens, rollout(), vocab=arch.vocab).mean_abs > 0
                sync(step)
                gap = s.check_policy(h @ sp[head].t(), tokens, rollout(), version=step, vocab=arch.vocab)
                assert gap == PolicyGap(43, 0.0, 0.0, 0.0, step)
            with pytest.raises(ValueError, match="version 1, the last sync carried 2"):
                s.check_policy(h @ sp[head].t(), tokens, rollout(), version=1)
            assert s.summary()["policy_gap"]["tokens"] == 43
            from weightbridge_b200.control.sender import TransferError
            with pytest.raises(TransferError, match="does not serve"):
                s.check_policy(h @ sp[head].t(), tokens, rollout() - 0.5, vocab=arch.vocab, tolerance=0.1)
            assert abs(s.last_gap.mean_abs - 0.5) < 1e-5


@gpu
def test_whole_step_captured_and_replayed():
    """Scoring, gradient, norm and update in one graph; replays equal eager steps bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(20, 64, device="cuda", generator=g)
    tokens = torch.randint(0, 500, (20,), device="cuda", generator=g)
    weight = torch.randn(500, 64, device="cuda", generator=g) * 0.1
    adv = torch.randn(20, device="cuda", generator=g)

    def make():
        w = {"w": weight.clone()}
        return w, AdamW(w, lr=1e-2, betas=(0.9, 0.95), states="fp8")

    def step(w, opt):
        logits = (h @ w["w"].t()).requires_grad_()
        out = token_logprobs(logits, tokens)
        d, = torch.autograd.grad((out.logprobs, out.entropy), logits, (-adv, -0.01 * torch.ones_like(adv)))
        return opt.step({"w": d.t() @ h}, max_norm=1.0)

    a, opt_a = make()
    b, opt_b = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, opt_a)
    torch.cuda.current_stream().wait_stream(side)
    step(b, opt_b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(a, opt_a)
    for _ in range(3):
        graph.replay()
        assert torch.equal(norm, step(b, opt_b))
    torch.cuda.synchronize()
    assert opt_a.step_count == opt_b.step_count == 4 and torch.equal(a["w"], b["w"])


@gpu
def test_policy_gap_values():
    x = torch.randn(6, 50, device="cuda")
    t = torch.tensor([0, 1, 2, 3, -100, 5], device="cuda")
    x[3, 3] = -math.inf
    mine = token_logprobs(x, t).logprobs
    theirs = mine.cpu()                                  # the rollout's come from its own process
    theirs[4] = 123.0                                    # padding is not compared
    gap = policy_gap(x, t, theirs)
    assert gap == PolicyGap(5, 0.0, 0.0, 0.0) and gap.within(0.0)
    theirs[0] += 0.25
    theirs[1] -= 0.5
    gap = policy_gap(x, t, theirs)
    want = sum(math.exp(d) - 1 - d for d in (-0.25, 0.5)) / 5
    assert gap.tokens == 5 and abs(gap.mean_abs - 0.15) < 1e-6 and abs(gap.max_abs - 0.5) < 1e-6 and abs(gap.kl - want) < 1e-6
    theirs[3] = -4.0                                     # the rollout sampled what the trainer cannot
    gap = policy_gap(x, t, theirs)
    assert gap.mean_abs == gap.max_abs == gap.kl == math.inf and not gap.within(1e9)
    theirs[3], theirs[0] = -math.inf, math.nan
    assert not policy_gap(x, t, theirs).within(1e9)
    assert policy_gap(x[:0], t[:0], mine[:0]) == PolicyGap(0, 0.0, 0.0, 0.0)
    assert policy_gap(x[4:5], t[4:5], mine[4:5]).tokens == 0


def test_refusals_without_a_gpu():
    x, t = torch.randn(4, 10), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match="rollout log probabilities"):
        policy_gap(x, t, torch.zeros(3))
    with pytest.raises(ValueError, match="CUDA"):
        policy_gap(x, t, torch.zeros(4))
    s = WeightSender("cpu_direct", [])
    with pytest.raises(ValueError, match="version 3, the last sync carried None"):
        s.check_policy(x, t, torch.zeros(4), version=3)
    assert "policy_gap" not in s.summary()
