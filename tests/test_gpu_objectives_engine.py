"""Fine-tuning passes of the engine on the GPU: log-probabilities, policy and preference passes, dropout and updates together, against the same
run of the CPU oracle in fp32."""
import pytest
import torch

from util import assert_close

pytestmark = pytest.mark.gpu


def _engine(device, family, recompute="none", dropout=0.1):
    from context_parallelism_b200.config import Config
    from context_parallelism_b200.engine import TrainEngine
    cfg = Config.from_env(family, 1, env={}).replace(
        n_embd=256, n_layer=2, n_head=4, n_kv_head=2 if family == "llama" else 4, head_dim=64, ffn_hidden=512 if family == "llama" else 1024, vocab_size=1000,
        T=200, B=4, max_steps=20, warmup_steps=1, checkpointing=False, recompute=recompute, dtype="bf16" if device == "cuda" else "fp32",
        weight_tying=family == "gpt2", dropout=dropout)
    return TrainEngine(cfg, torch.device(device, 0) if device == "cuda" else torch.device("cpu"))


@pytest.mark.parametrize("family,recompute", [("llama", "none"), ("llama", "selective"), ("gpt2", "none"), ("gpt2", "full")])
def test_passes_together(family, recompute):
    a, b = _engine("cuda", family, recompute), _engine("cpu", family)
    g = torch.Generator().manual_seed(3)
    for step in range(4):
        t = torch.randint(0, 1000, (4, 201), generator=g)
        x, y = t[:, :-1].contiguous().pin_memory(), t[:, 1:].contiguous().pin_memory()
        for i in range(4):
            y[i, : 20 + 10 * i], y[i, 200 - 9 * i:] = -100, -100
        old_a, old_b = a.token_logprobs(x, y), b.token_logprobs(x, y)
        # two layers in bf16: logits of a model that has not learnt are off by some 2^-8 of their deviation of about one
        assert float((old_a.cpu() - old_b).abs().max()) < 0.1
        noise, adv = 0.1 * torch.randn(4, 200, generator=g), torch.randn(4, generator=g)
        outs = []
        for e, old in ((a, old_a), (b, old_b)):
            old = old + noise.to(old.device)
            if step % 2:
                out = e.preference_forward_backward(x, y, old, beta=0.5)
                outs.append((out.loss, out.ratios))
            else:
                # the CPU's seeds, positions and masks are those of the GPU; advantages on either device
                out = e.policy_forward_backward(x, y, old, adv if step else adv.to(old.device), ref_logp=old, kl_coef=0.05, clip=(0.4, 0.4))
                outs.append((out.loss, out.terms))
        assert abs(float(outs[0][0]) - float(outs[1][0])) < 0.02 * (1 + abs(float(outs[1][0])))
        assert_close(a.flat.grad.cpu(), b.flat.grad, cos=0.99, name="gradient")
        for e in (a, b):
            e.finish_step()
            e.optimizer_step()
        b.flat.master.copy_(a.flat.master.cpu()), b.flat.sync_compute_copy()
    a.check_kernels()


def test_tokens_that_do_not_count_change_nothing():
    a = _engine("cuda", "llama", dropout=0.0)
    t = torch.randint(0, 1000, (4, 201), device="cuda")
    x, y = t[:, :-1].contiguous(), t[:, 1:].contiguous()
    y[:, 150:] = -100
    old, adv = a.token_logprobs(x, y), torch.ones(4, 200, device="cuda")
    a.policy_forward_backward(x, y, old, adv)
    one = a.flat.grad.clone()
    a.opt.zero_grad()
    # causal attention: what stands behind the answers reaches no counted token
    x2, bad = x.clone(), old.clone()
    x2[:, 160:] = 7
    bad[:, 150:] = float("nan")
    adv[:, 150:] = float("inf")
    a.policy_forward_backward(x2, y, bad, adv)
    # embedding, norm and dQ sums in arrival order
    assert_close(a.flat.grad, one, cos=0.999999, rel=1e-3)


def test_page_locked_buffers_may_be_written_again():
    """What a call reads of page-locked buffers it has taken over when it returns."""
    a, b = _engine("cuda", "llama", dropout=0.0), _engine("cuda", "llama", dropout=0.0)
    g = torch.Generator().manual_seed(5)
    t = torch.randint(0, 1000, (4, 201), generator=g)
    x, y = t[:, :-1].contiguous().pin_memory(), t[:, 1:].contiguous().pin_memory()
    vals = [(torch.randn(4, 200, generator=g) - s).pin_memory() for s in (7, 0, 7)] + [(torch.rand(4, 200, generator=g) / 800).pin_memory()]
    pair = torch.rand(2, generator=g).pin_memory()
    keep = [v.clone() for v in (x, y, *vals, pair)]
    big = torch.randn(8192, 8192, device="cuda")
    outs = []
    for e, (x, y, old, adv, ref, wt, pw), spoil in ((a, keep, False), (b, (x, y, *vals, pair), True)):
        for _ in range(20):
            big = big @ big * 1e-4                                   # the device is behind
        p = e.policy_forward_backward(x, y, old, adv, wt, ref, kl_coef=0.1, accum=2, last=False)
        q = e.preference_forward_backward(x, y, ref, pw, accum=2)
        lp = e.token_logprobs(x, y)
        if spoil:
            x.fill_(1), y.fill_(-100)
            for v in (old, adv, ref, wt, pw):
                v.fill_(float("nan"))
        outs.append((p.loss, p.terms, q.loss, q.ratios, lp))
    for u, v in zip(*outs):
        assert torch.allclose(u, v, rtol=1e-4, atol=1e-5)
    assert_close(a.flat.grad, b.flat.grad, cos=0.99999, rel=1e-2)
