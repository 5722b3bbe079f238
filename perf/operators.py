"""The fine-tuning operators of this framework as cases that can be timed on one GPU, and their plain forms.

Four operators, each through its public entry point, forward and backward:

* ``logprobs``    log-probabilities of given tokens under the language-model head, with any gradient per token;
* ``policy``      clipped policy loss with a KL term, from hidden states and the head's weights;
* ``preference``  paired log-ratio loss over whole sequences, from hidden states and the head's weights;
* ``dropout``     counter-based dropout: in front of a norm, on the residual branch, or alone (embedding).

In ``logprobs``, ``policy`` and ``preference`` a case's ``spans`` says which tokens count: ``"all"``, or ``"response"``, one span per
sequence behind a prompt and in front of padding, as fine-tuning data has them.
"""
from __future__ import annotations

import math

import torch

own = False


def _objective(kind, B, T, d, n_valid, spans="response", **more):
    return dict(kind=kind, B=B, T=T, d=d, n_valid=n_valid, spans=spans, **more)


def _policy(B, T, d, n_valid, spans="response", kl=0.05, low=0.2, high=0.2):
    return _objective("policy", B, T, d, n_valid, spans, kl=kl, low=low, high=high)


def _preference(pairs, T, d, n_valid, spans="response", beta=0.1, smoothing=0.0):
    return _objective("preference", 2 * pairs, T, d, n_valid, spans, beta=beta, smoothing=smoothing)


def _dropout(form, B, T, d, p=0.1):
    return dict(kind="dropout", form=form, B=B, T=T, d=d, p=p)


def listed():
    return [
        # one short rollout of GPT-2 124M scored by a user's own objective: latency and one sweep over the weights
        dict(_objective("logprobs", 1, 136, 768, 50257, "all"), name="logprobs_124m_136"),
        # the Llama-style 48M micro-batch, prompts masked
        dict(_objective("logprobs", 2, 4096, 384, 50304), name="logprobs_48m_2x4096"),
        # a few ragged rollouts of GPT-2 124M, KL against a reference policy
        dict(_policy(3, 1111, 768, 50257), name="policy_124m_3x1111"),
        # a group of eight rollouts of the 1B shape for one prompt, asymmetric clipping
        dict(_policy(8, 1024, 2048, 128256, high=0.28), name="policy_1b_8x1024"),
        # one long rollout of the 8B shape, every token counted, no reference policy
        dict(_policy(1, 8192, 4096, 128256, "all", kl=0.0), name="policy_8b_8192"),
        # one short pair through GPT-2 124M
        dict(_preference(1, 301, 768, 50257), name="preference_124m_1x301"),
        # two pairs through the GPT-2 44M shape, noisy labels
        dict(_preference(2, 1024, 384, 50304, beta=0.03, smoothing=0.1), name="preference_44m_2x1024"),
        # pairs of long answers, 1B shape
        dict(_preference(2, 4096, 2048, 128256, beta=0.01), name="preference_1b_2x4096"),
        # a block's norm behind dropout, one short window of GPT-2 124M: latency
        dict(_dropout("layernorm", 1, 136, 768), name="dropout_layernorm_136x768"),
        # the same in the Llama-style 48M micro-batch
        dict(_dropout("rmsnorm", 2, 4096, 384), name="dropout_rmsnorm_8192x384"),
        # dropout behind the embedding of GPT-2 124M, an odd length
        dict(_dropout("alone", 4, 1021, 768), name="dropout_alone_4084x768"),
        # the benchmark's sequence of the 1B shape
        dict(_dropout("rmsnorm", 1, 131072, 2048, p=0.05), name="dropout_rmsnorm_131072x2048"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "policy", "policy", "preference", "preference", "dropout", "dropout"])
    if kind == "dropout":
        d = rng.choice([64, 384, 520, 768, 1032, 2048, 4096])
        rows = _log_int(rng, 1, (131072 << 11) // d if d > 1024 else 65536)
        B = rng.choice([1, 1, 2, 5])
        return _dropout(rng.choice(["layernorm", "rmsnorm", "alone"]), B, max(1, rows // B), d, rng.choice([0.05, 0.1, 0.25, 0.5]))
    d = rng.choice([128, 384, 520, 768, 1032, 2048, 4096])
    n_valid = rng.choice([1000, 8192, 50257, 50304, 128256])
    most = min(16384, (8192 * 4096 * 128256) // (d * max(n_valid, 50257)))     # no dearer than the largest listed case
    B = 2 * rng.choice([1, 1, 2, 3]) if kind == "preference" else rng.choice([1, 1, 2, 3, 8])
    T = max(1, _log_int(rng, 8, most) // B)
    spans = rng.choice(["all", "response", "response"])
    if kind == "logprobs":
        return _objective(kind, B, T, d, n_valid, spans)
    if kind == "policy":
        return _policy(B, T, d, n_valid, spans, rng.choice([0.0, 0.02, 0.1]), 0.2, rng.choice([0.2, 0.28]))
    # log-ratios grow with the length, and the factor in front of them is chosen to go with it
    return _preference(B // 2, T, d, n_valid, spans, rng.choice([5.0, 10.0, 20.0]) / max(T, 50), rng.choice([0.0, 0.0, 0.1]))


# ---------------------------------------------------------------------------------------------------------- preparation
def _span(case, b):
    """First counted position of sequence ``b`` and the number of them."""
    T = case["T"]
    if case["spans"] == "all":
        return 0, T
    n = max(1, int(T * (0.3 + 0.6 * ((0.618034 * (b + 1)) % 1.0))))
    return int((T - n) * ((0.414214 * (b + 1)) % 1.0)), n


def _live(case):
    return sum(_span(case, b)[1] for b in range(case["B"]))


def _vocab_rows(case):
    return (case["n_valid"] + 63) // 64 * 64            # the head's weights have zero rows behind the vocabulary


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, T, d = case["B"], case["T"], case["d"]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, device=dev, generator=gen) * std + mean
    if case["kind"] == "dropout":
        key = torch.randint(-2 ** 62, 2 ** 62, (1,), device=dev, generator=gen)
        state = dict(case=case, seed=key, site=seed % 100, x=normal(B, T, d).bfloat16().requires_grad_(), dy=normal(B, T, d).bfloat16())
        if case["form"] != "alone":
            state.update(res=normal(B, T, d, std=0.5).bfloat16().requires_grad_(), dnew=normal(B, T, d).bfloat16(),
                         w=normal(d, std=0.1, mean=1.0).requires_grad_())
        if case["form"] == "layernorm":
            state["b"] = normal(d, std=0.1).requires_grad_()
        return state
    V = _vocab_rows(case)
    x = normal(B, T, d).bfloat16()                      # behind the final norm
    w = normal(V, d, std=4.0 / math.sqrt(d))            # logits with a deviation of four: some tokens are likely
    w[case["n_valid"]:] = 0
    w = w.bfloat16()
    logits = (x.view(-1, d).float() @ w.float().T)[:, : case["n_valid"]]
    # the tokens were sampled from the policy
    targets = (logits - torch.empty_like(logits).exponential_(generator=gen).log_()).argmax(1, keepdim=True)
    logp = (logits.gather(1, targets)[:, 0] - torch.logsumexp(logits, 1)).view(B, T)
    del logits
    targets = targets.view(B, T)
    for b in range(B):
        s, n = _span(case, b)
        targets[b, :s] = -100
        targets[b, s + n:] = -100
    state = dict(case=case, x=x.requires_grad_(), w=w.requires_grad_(), targets=targets)
    if case["kind"] == "logprobs":
        state["grad"] = normal(B, T)
    elif case["kind"] == "policy":
        # the policy has moved a little since the rollout; no ratio within half a percent of where it is clipped
        moved = normal(B, T, std=0.15)
        for border in (math.log(1 - case["low"]), math.log(1 + case["high"])):
            moved = torch.where((moved - border).abs() < 0.005, border + 0.01, moved)
        state["old"] = logp - moved
        state["ref"] = logp + normal(B, T, std=0.3) if case["kl"] else None
        state["advantages"] = normal(B, T, mean=0.5)
        state["weights"] = torch.full((B, T), 1.0 / _live(case), device=dev)
    else:
        # training has made the chosen answers likelier than they were and the rejected ones less likely
        drift = torch.full((B, 1), 0.05, device=dev)
        drift[B // 2:] = -0.05
        state["ref"] = logp - drift + normal(B, T, std=0.3)
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return _RUN[state["case"]["kind"]](state)


def _token_terms(x, w, targets, n_valid):
    """fp32 probabilities, log-probabilities of the targets and the counted tokens."""
    logits = (x.reshape(-1, x.shape[-1]).float() @ w.float().T)[:, :n_valid]
    t = targets.reshape(-1)
    live = t >= 0
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    s = e.sum(1, keepdim=True)
    logp = (logits.gather(1, t.clamp(min=0)[:, None]) - top - torch.log(s))[:, 0]
    return e / s, torch.where(live, logp, torch.zeros_like(logp)), t, live


def _head_gradients(x, w, p, t, live, u):
    """Gradients of ``sum(u * logp)``."""
    u = torch.where(live, u, torch.zeros_like(u))
    dz = p * -u[:, None]
    dz.scatter_add_(1, t.clamp(min=0)[:, None], u[:, None])
    dx = dz @ w.float()[: p.shape[1]]
    dw = torch.zeros(w.shape, device=w.device)
    dw[: p.shape[1]] = dz.T @ x.reshape(-1, x.shape[-1]).float()
    return dx.view(x.shape).to(x.dtype), dw.to(w.dtype)


def _run_logprobs(state):
    case, x, w, targets, grad = (state[k] for k in ("case", "x", "w", "targets", "grad"))
    if own:
        from context_parallelism_b200.ops import objectives
        logp = objectives.token_logprobs(x, w, targets, case["n_valid"])
        dx, dw = torch.autograd.grad(logp, [x, w], grad)
        return dict(logp=logp.detach(), dx=dx, dw=dw)
    with torch.no_grad():
        p, logp, t, live = _token_terms(x, w, targets, case["n_valid"])
        dx, dw = _head_gradients(x, w, p, t, live, grad.reshape(-1))
        return dict(logp=logp.view(targets.shape), dx=dx, dw=dw)


def _run_policy(state):
    case, x, w, targets = (state[k] for k in ("case", "x", "w", "targets"))
    old, ref, adv, weights = (state[k] for k in ("old", "ref", "advantages", "weights"))
    if own:
        from context_parallelism_b200.ops import objectives
        out = objectives.linear_policy_loss(x, w, targets, old, adv, weights=weights, ref_logp=ref, clip=(case["low"], case["high"]),
                                            kl_coef=case["kl"], n_valid=case["n_valid"])
        dx, dw = torch.autograd.grad(out.loss, [x, w])
        return dict(loss=out.loss.detach(), logp=out.logp, terms=out.terms, dx=dx, dw=dw)
    with torch.no_grad():
        p, logp, t, live = _token_terms(x, w, targets, case["n_valid"])
        loss, terms, u = _policy_terms(case, logp.double(), live, old, ref, adv, weights)
        dx, dw = _head_gradients(x, w, p, t, live, u.float())
        return dict(loss=loss.float(), logp=logp.view(targets.shape), terms=terms.float(), dx=dx, dw=dw)


def _policy_terms(case, logp, live, old, ref, adv, weights):
    """Loss, its four sums and the gradient with respect to ``logp``, in 64 bits."""
    old, adv, wt = (v.reshape(-1).double() for v in (old, adv, weights))
    wt = torch.where(live, wt, torch.zeros_like(wt))
    ratio = torch.exp(logp - old)
    plain, clipped = ratio * adv, ratio.clamp(1 - case["low"], 1 + case["high"]) * adv
    cut = ((adv > 0) & (ratio > 1 + case["high"])) | ((adv < 0) & (ratio < 1 - case["low"]))
    surrogate = -torch.minimum(plain, clipped)
    u = torch.where(cut, torch.zeros_like(plain), -plain)
    kl = torch.zeros_like(plain)
    if ref is not None:
        delta = ref.reshape(-1).double() - logp
        kl = torch.expm1(delta) - delta
        u = u - case["kl"] * torch.expm1(delta)
    terms = torch.stack([torch.where(live, wt * v, torch.zeros_like(v)).sum() for v in (surrogate, kl, cut.double(), torch.ones_like(kl))])
    return terms[0] + case["kl"] * terms[1], terms, torch.where(live, wt * u, torch.zeros_like(u))


def _run_preference(state):
    case, x, w, targets, ref = (state[k] for k in ("case", "x", "w", "targets", "ref"))
    if own:
        from context_parallelism_b200.ops import objectives
        out = objectives.linear_preference_loss(x, w, targets, ref, beta=case["beta"], smoothing=case["smoothing"], n_valid=case["n_valid"])
        dx, dw = torch.autograd.grad(out.loss, [x, w])
        return dict(loss=out.loss.detach(), logp=out.logp, ratios=out.ratios, dx=dx, dw=dw)
    with torch.no_grad():
        p, logp, t, live = _token_terms(x, w, targets, case["n_valid"])
        loss, ratios, u = _preference_terms(case, logp.double(), live, ref)
        dx, dw = _head_gradients(x, w, p, t, live, u.float())
        return dict(loss=loss.float(), logp=logp.view(targets.shape), ratios=ratios.float(), dx=dx, dw=dw)


def _preference_terms(case, logp, live, ref):
    """Loss, log-ratio of every sequence and the gradient with respect to ``logp``, in 64 bits."""
    diff = logp - ref.reshape(-1).double()
    ratios = torch.where(live, diff, torch.zeros_like(diff)).view(case["B"], -1).sum(1)
    chosen, rejected = ratios.chunk(2)
    z, s = case["beta"] * (chosen - rejected), case["smoothing"]
    loss = ((1 - s) * _softplus(-z) + s * _softplus(z)).sum()
    dh = case["beta"] * (s * torch.sigmoid(z) - (1 - s) * torch.sigmoid(-z))
    return loss, ratios, torch.cat([dh, -dh])[:, None].expand(-1, case["T"]).reshape(-1)


def _softplus(z):
    return z.clamp(min=0) + torch.log1p(torch.exp(-z.abs()))


def _philox(row, groups, site, seed):
    """Philox4x32 with seven rounds (Salmon et al., 2011): counter (column group, row, row >> 32, site), key ``seed``; ``[rows, 4 groups]``."""
    low = 0xffffffff
    c0 = torch.arange(groups, device=row.device).expand(row.numel(), -1)
    c1, c2 = (row & low)[:, None].expand_as(c0), (row >> 32 & low)[:, None].expand_as(c0)
    c3 = torch.full_like(c0, site)
    k0, k1 = seed & low, seed >> 32 & low
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    c0, c1, c2, c3, k0, k1 = _philox_round(c0, c1, c2, c3, k0, k1)
    return torch.stack([c0, c1, c2, c3], dim=2).view(row.numel(), 4 * groups)


def _philox_round(c0, c1, c2, c3, k0, k1):
    low = 0xffffffff
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57             # 64-bit products; the sign is masked away
    return (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low, (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low


def _keep(state):
    case = state["case"]
    rows = torch.arange(case["B"] * case["T"], device=state["x"].device)
    return (_philox(rows, case["d"] // 4, state["site"], state["seed"]) >= int(case["p"] * 2 ** 32)).view(state["x"].shape)


def _run_dropout(state):
    case, x = state["case"], state["x"]
    alone = case["form"] == "alone"
    if own:
        from context_parallelism_b200.ops import elementwise as E
        drop = E.Dropout(case["p"], state["seed"], state["site"])
        if alone:
            y = E.dropout(x, drop)
            return dict(y=y.detach(), dx=torch.autograd.grad(y, [x], state["dy"])[0])
        if case["form"] == "layernorm":
            y, new = E.layernorm(x, state["w"], state["b"], 1e-5, state["res"], drop)
            grads = torch.autograd.grad([y, new], [x, state["res"], state["w"], state["b"]], [state["dy"], state["dnew"]])
        else:
            y, new = E.rmsnorm(x, state["w"], 1e-5, state["res"], drop)
            grads = torch.autograd.grad([y, new], [x, state["res"], state["w"]], [state["dy"], state["dnew"]])
        return dict(y=y.detach(), new=new.detach(), grads=list(grads))
    with torch.no_grad():
        return _dropout_form(state)


def _dropout_form(state):
    case, keep = state["case"], _keep(state)
    scale = 1.0 / (1.0 - case["p"])
    x, dy = state["x"].float(), state["dy"].float()
    if case["form"] == "alone":
        return dict(y=torch.where(keep, x * scale, 0.0).bfloat16(), dx=torch.where(keep, dy * scale, 0.0).bfloat16())
    # the residual stream is bf16, and the norm is of what it holds
    new = (x + torch.where(keep, state["res"].float() * scale, 0.0)).bfloat16()
    v = new.float()
    centred = v - v.mean(-1, keepdim=True) if case["form"] == "layernorm" else v
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    hat = centred * rstd
    g = dy * state["w"]
    dx = g - hat * (g * hat).mean(-1, keepdim=True)
    y, dw = hat * state["w"], [(dy * hat).sum((0, 1))]
    if case["form"] == "layernorm":
        dx = dx - g.mean(-1, keepdim=True)
        y = y + state["b"]
        dw.append(dy.sum((0, 1)))
    dx = dx * rstd + state["dnew"].float()
    return dict(y=y.bfloat16(), new=new, grads=[dx.bfloat16(), torch.where(keep, dx * scale, 0.0).bfloat16(), *dw])


_RUN = dict(logprobs=_run_logprobs, policy=_run_policy, preference=_run_preference, dropout=_run_dropout)


# ------------------------------------------------------------------------------------------------------- work, 64 bits
def work(case):
    B, T, d = case["B"], case["T"], case["d"]
    n = B * T * d
    if case["kind"] == "dropout":
        if case["form"] == "alone":
            return {"bytes": 8 * n, "flops": 4.0 * n}
        # x, the branch and two gradients in, two results and two gradients out
        return {"bytes": 16 * n, "flops": 30.0 * n}
    live, V = _live(case), case["n_valid"]
    # hidden states of counted tokens and weights in, both gradients out; targets, and up to four numbers per token
    return {"bytes": 2 * (live * d + n) + 4 * _vocab_rows(case) * d + 28 * B * T, "flops": 6.0 * live * V * d}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "dropout":
        return _exact_dropout(case, state)
    x, w, targets = state["x"].detach(), state["w"].detach().double()[: case["n_valid"]], state["targets"].reshape(-1)
    flat = x.reshape(-1, case["d"])
    logp = torch.zeros(flat.shape[0], dtype=torch.float64, device=x.device)
    for r in range(0, flat.shape[0], 1024):
        z = torch.log_softmax(flat[r:r + 1024].double() @ w.T, 1)
        logp[r:r + 1024] = z.gather(1, targets[r:r + 1024].clamp(min=0)[:, None])[:, 0]
    logp[targets < 0] = 0
    out, u = _exact_loss(case, state, logp, targets >= 0)
    dx = torch.zeros(flat.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros((_vocab_rows(case), case["d"]), dtype=torch.float64, device=x.device)
    for r in range(0, flat.shape[0], 1024):
        xc, t, uc = flat[r:r + 1024].double(), targets[r:r + 1024].clamp(min=0), u[r:r + 1024]
        dz = torch.softmax(xc @ w.T, 1) * -uc[:, None]
        dz[torch.arange(t.numel(), device=t.device), t] += uc
        dx[r:r + 1024] = dz @ w
        dw[: case["n_valid"]] += dz.T @ xc
    return dict(out, logp=logp.view(state["targets"].shape), dx=dx.view(x.shape), dw=dw)


def _exact_loss(case, state, logp, live):
    """What comes beside the gradients, and the loss's gradient with respect to the log-probabilities, by autograd."""
    if case["kind"] == "logprobs":
        return {}, torch.where(live, state["grad"].reshape(-1).double(), 0.0)
    leaf = logp.clone().requires_grad_()
    if case["kind"] == "preference":
        ratios = torch.stack([(leaf - state["ref"].reshape(-1).double())[b * case["T"]:][: case["T"]][live[b * case["T"]:][: case["T"]]].sum()
                              for b in range(case["B"])])
        z = case["beta"] * (ratios[: case["B"] // 2] - ratios[case["B"] // 2:])
        loss = -(torch.nn.functional.logsigmoid(z) * (1 - case["smoothing"]) + torch.nn.functional.logsigmoid(-z) * case["smoothing"]).sum()
        out = dict(loss=loss.detach(), ratios=ratios.detach())
    else:
        at = live.nonzero()[:, 0]
        adv, wt = (state[k].reshape(-1)[at].double() for k in ("advantages", "weights"))
        r = (leaf[at] - state["old"].reshape(-1)[at].double()).exp()
        surrogate = torch.maximum(-adv * r, -adv * r.clip(1 - case["low"], 1 + case["high"]))
        kl = torch.zeros_like(r)
        if state["ref"] is not None:
            kl = torch.special.expm1(state["ref"].reshape(-1)[at].double() - leaf[at]) - state["ref"].reshape(-1)[at].double() + leaf[at]
        loss = (wt * (surrogate + case["kl"] * kl)).sum()
        cut = torch.where(adv > 0, r > 1 + case["high"], (r < 1 - case["low"]) & (adv < 0))
        terms = torch.stack([(wt * v).sum() for v in (surrogate, kl, cut.double(), torch.ones_like(wt))])
        out = dict(loss=loss.detach(), terms=terms.detach())
    return out, torch.autograd.grad(loss, leaf)[0]


def _exact_dropout(case, state):
    factor = _keep(state).double() / (1.0 - case["p"])
    x, dy = state["x"].detach().double(), state["dy"].double()
    if case["form"] == "alone":
        return dict(y=x * factor, dx=dy * factor)
    new = x + state["res"].detach().double() * factor
    # the residual stream is bf16, and the norm is of what it holds: the sum in 32 bits, rounded
    kept = torch.where(factor != 0, state["res"].detach().float() * (1.0 / (1.0 - case["p"])), 0.0)
    v = (state["x"].detach().float() + kept).bfloat16().double().requires_grad_()
    w = state["w"].detach().double().requires_grad_()
    if case["form"] == "layernorm":
        leaves = [v, w, state["b"].detach().double().requires_grad_()]
        y = torch.nn.functional.layer_norm(v, v.shape[-1:], w, leaves[2], 1e-5)
    else:
        leaves = [v, w]
        y = torch.nn.functional.rms_norm(v, v.shape[-1:], w, 1e-5)
    dv, *dw = torch.autograd.grad(y, leaves, dy)
    dv = dv + state["dnew"].double()
    return dict(y=y.detach(), new=new, grads=[dv, dv * factor, *dw])
