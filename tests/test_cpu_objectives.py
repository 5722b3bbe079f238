"""Fine-tuning objectives without a GPU: the plain form against formulas and differences, and what is refused before a launcher gets an address."""
import math

import pytest
import torch

from context_parallelism_b200 import _native as nv
from context_parallelism_b200.ops import objectives as O


def _case(B=4, T=5, d=8, V=24, n_valid=21, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, d, generator=g, dtype=dtype).requires_grad_()
    w = (torch.randn(V, d, generator=g, dtype=dtype) / 2).requires_grad_()
    t = torch.randint(0, n_valid, (B, T), generator=g)
    t[0, :2], t[1, 3:] = -100, -1
    return x, w, t, g


def test_logprobs():
    x, w, t, g = _case()
    logp = O.token_logprobs(x, w, t, 21)
    want = torch.log_softmax((x @ w.T)[..., :21], -1).gather(-1, t.clamp(min=0)[..., None])[..., 0]
    assert torch.allclose(logp, torch.where(t >= 0, want, 0.0), rtol=1e-12)
    assert torch.autograd.gradcheck(lambda x, w: O.token_logprobs(x, w, t, 21), (x, w))


def _policy_by_hand(logp, t, old, adv, wt, ref, clip, kl):
    """Token by token with Python's floats."""
    sums = [0.0] * 4
    for i in range(t.numel()):
        lp, o, a, k = (float(v.reshape(-1)[i]) for v in (logp, old, adv, wt))
        if int(t.reshape(-1)[i]) < 0 or k == 0:
            continue
        r = math.exp(lp - o)
        c = min(max(r, 1 - clip[0]), 1 + clip[1])
        sums[0] += -k * min(r * a, c * a)
        sums[2] += k * ((a > 0 and r > 1 + clip[1]) or (a < 0 and r < 1 - clip[0]))
        sums[3] += k
        if ref is not None:
            d = float(ref.reshape(-1)[i]) - lp
            sums[1] += k * (math.expm1(d) - d)
    return sums[0] + kl * sums[1], sums


@pytest.mark.parametrize("kl", [None, 0.0, 0.3])
@pytest.mark.parametrize("clip", [(0.2, 0.2), (0.1, 0.5), (1.0, 0.0)])
def test_policy(clip, kl):
    x, w, t, g = _case(seed=3)
    logp = O.token_logprobs(x, w, t, 21).detach()
    # fp32 inputs, as they are taken; a third of the ratios beyond either border, none at one
    old = (logp - torch.tensor([-1.5, -0.05, 0.03, 1.5, 0.02]).expand(4, 5)).float()
    adv = torch.randn(4, 5, generator=g)
    adv[2, 2] = 0
    wt = torch.rand(4, 5, generator=g)
    wt[3, 1] = 0
    ref = None if kl is None else (logp + 0.3 * torch.randn(4, 5, generator=g)).float()
    args = dict(weights=wt, ref_logp=ref, clip=clip, kl_coef=kl or 0.0, n_valid=21)
    out = O.linear_policy_loss(x, w, t, old, adv, **args)
    loss, sums = _policy_by_hand(logp, t, old, adv, wt, ref, clip, kl or 0.0)
    assert float(out.loss) == pytest.approx(loss, rel=1e-12) and out.terms.tolist() == pytest.approx(sums, rel=1e-12)
    keep = (t >= 0) & (wt != 0)
    assert torch.equal(out.logp, torch.where(keep, logp, 0.0)) and not out.logp.requires_grad and not out.terms.requires_grad
    assert torch.autograd.gradcheck(lambda x, w: O.linear_policy_loss(x, w, t, old, adv, **args).loss, (x, w))


@pytest.mark.parametrize("smoothing", [0.0, 0.2, 1.0])
@pytest.mark.parametrize("beta", [0.1, 3.0])
def test_preference(beta, smoothing):
    x, w, t, g = _case(seed=5)
    t[3] = -100                                                      # an answer without tokens
    logp = O.token_logprobs(x, w, t, 21).detach()
    ref, wt = torch.randn(4, 5, generator=g) - 3, torch.tensor([0.7, 1.5])
    args = dict(weights=wt, beta=beta, smoothing=smoothing, n_valid=21)
    out = O.linear_preference_loss(x, w, t, ref, **args)
    ratios = [sum(float(logp[b, i]) - float(ref[b, i]) for i in range(5) if t[b, i] >= 0) for b in range(4)]
    want = 0.0
    for i in range(2):
        z = beta * (ratios[i] - ratios[2 + i])
        want += float(wt[i]) * ((1 - smoothing) * math.log1p(math.exp(-z)) + smoothing * math.log1p(math.exp(z)))
    assert out.ratios.tolist() == pytest.approx(ratios, rel=1e-12) and float(out.loss) == pytest.approx(want, rel=1e-12)
    assert torch.autograd.gradcheck(lambda x, w: O.linear_preference_loss(x, w, t, ref, **args).loss, (x, w))


def test_values_in_masked_places():
    x, w, t, g = _case(dtype=torch.float32)
    old, adv, ref = (torch.randn(4, 5, generator=g) - 3 for _ in range(3))
    off = t < 0
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min])

    def spoil(v):
        v = v.clone().detach()
        v[off] = bad[torch.arange(int(off.sum())) % 4].view(-1, *[1] * (v.dim() - 2)).expand_as(v[off])
        return v
    clean = (lambda x, o, a, r: O.linear_policy_loss(x, w, t, o, a, ref_logp=r, kl_coef=0.1, n_valid=21), lambda x, o, a, r: O.linear_preference_loss(x, w, t, r, n_valid=21))
    for f in clean:
        a = x.detach().clone().requires_grad_()
        b = spoil(x).requires_grad_()
        la, lb = f(a, old, adv, ref).loss, f(b, spoil(old), spoil(adv), spoil(ref)).loss
        ga, gb = torch.autograd.grad(la, [a, w]), torch.autograd.grad(lb, [b, w])
        assert torch.equal(la, lb) and all(torch.equal(p, q) for p, q in zip(ga, gb)) and not bool(ga[0][off].any())


def test_nothing_counts():
    x, w, t, g = _case(dtype=torch.float32)
    z = torch.zeros(4, 5)
    for out in (O.linear_policy_loss(x, w, torch.full_like(t, -100), z, z, n_valid=21), O.linear_policy_loss(x, w, t, z, z, weights=z, n_valid=21)):
        assert float(out.loss) == 0 and out.terms.tolist() == [0, 0, 0, 0]
    out = O.linear_preference_loss(x, w, torch.full_like(t, -100), z, n_valid=21)
    assert float(out.loss) == pytest.approx(2 * math.log(2)) and out.ratios.tolist() == [0] * 4
    assert not bool(torch.autograd.grad(out.loss, w)[0].any())


class _OnGpu(torch.Tensor):
    """Host memory that takes the GPU's branches."""
    is_cuda = property(lambda self: True)


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


class _Status:
    @staticmethod
    def ptr():
        return 0


@pytest.fixture
def calls(monkeypatch):
    import contextlib
    made = []
    monkeypatch.setattr(nv, "call", lambda name, *a: made.append(name))
    monkeypatch.setattr(nv, "status_for", lambda dev: _Status)
    monkeypatch.setattr(nv, "stream_ptr", lambda dev=None: 0)
    monkeypatch.setattr(nv, "on", lambda dev: contextlib.nullcontext())
    return made


def _entries(x, w, t, **kw):
    z = torch.zeros(t.shape)
    return [lambda: O.token_logprobs(x, w, t, **kw), lambda: O.linear_policy_loss(x, w, t, z, z, **kw), lambda: O.linear_preference_loss(x, w, t, z, **kw)]


@pytest.mark.parametrize("x,w,t,kw", [
    ((2, 6, 64, torch.float32), (16, 64, torch.bfloat16), (2, 6), {}), ((2, 6, 64, torch.bfloat16), (16, 64, torch.float32), (2, 6), {}),
    ((2, 6, 64, torch.float16), (16, 64, torch.float16), (2, 6), {}), ((2, 6, 64, torch.bfloat16), (16, 56, torch.bfloat16), (2, 6), {}),
    ((2, 6, 60, torch.bfloat16), (16, 60, torch.bfloat16), (2, 6), {}), ((2, 6, 64, torch.bfloat16), (20, 64, torch.bfloat16), (2, 6), {}),
    ((2, 6, 64, torch.bfloat16), (16, 64, torch.bfloat16), (2, 5), {}), ((2, 6, 64, torch.bfloat16), (16, 64, torch.bfloat16), (12,), {}),
    ((2, 6, 64, torch.bfloat16), (16, 64, torch.bfloat16), (2, 6), dict(n_valid=17)), ((2, 6, 64, torch.bfloat16), (16, 64, torch.bfloat16), (2, 6), dict(n_valid=-1))])
def test_refused_before_a_launch(calls, x, w, t, kw):
    for entry in _entries(_t(*x[:3], dtype=x[3]), _t(*w[:2], dtype=w[2]), torch.zeros(t, dtype=torch.int64), **kw):
        with pytest.raises(AssertionError):
            entry()
    assert not calls


def test_accepted(calls):
    x, w = _t(2, 6, 64), _t(16, 64)
    for dtype in (torch.int32, torch.int64):
        for entry in _entries(x, w, torch.zeros(2, 6, dtype=dtype)):
            entry()
    assert calls == ["objective_fwd", "objective_fwd", "objective_fwd", "preference"] * 2


@pytest.mark.parametrize("gpu", [False, True])
def test_constants_refused(calls, gpu):
    x, w, t = (_t(2, 6, 64), _t(16, 64), torch.zeros(2, 6, dtype=torch.int64)) if gpu else (torch.zeros(2, 6, 64), torch.zeros(16, 64), torch.zeros(2, 6, dtype=torch.int64))
    z = torch.zeros(2, 6)
    grad = z.clone().requires_grad_()
    for bad in (dict(old_logp=grad), dict(advantages=grad), dict(weights=grad), dict(ref_logp=grad), dict(old_logp=z.long()), dict(advantages=torch.zeros(6)),
                dict(advantages=torch.zeros(3, 6)), dict(weights=torch.zeros(2, 6, device="meta")), dict(old_logp=None), dict(clip=(-0.1, 0.2)), dict(clip=(1.1, 0.2)),
                dict(clip=(0.2, -0.1)), dict(clip=(0.2, float("inf"))), dict(clip=(float("nan"), 0.2)), dict(kl_coef=0.1), dict(kl_coef=-0.1, ref_logp=z),
                dict(kl_coef=float("nan"), ref_logp=z)):
        with pytest.raises((AssertionError, RuntimeError)):
            O.linear_policy_loss(x, w, t, **{**dict(old_logp=z, advantages=z), **bad})
    for bad in (dict(ref_logp=grad), dict(ref_logp=None), dict(beta=0.0), dict(beta=-1.0), dict(beta=float("inf")), dict(smoothing=-0.1), dict(smoothing=1.1),
                dict(weights=torch.zeros(2)), dict(weights=torch.zeros(1, 1)), dict(weights=torch.zeros(1).requires_grad_())):
        with pytest.raises((AssertionError, RuntimeError)):
            O.linear_preference_loss(x, w, t, **{**dict(ref_logp=z), **bad})
    for odd in (slice(0, 1), slice(0, 0)):
        with pytest.raises(AssertionError):
            O.linear_preference_loss(x[odd], w, t[odd], z[odd])
    assert not calls


def test_plans():
    """The buffers hold what the layouts put there, and dlogits are taken in chunks."""
    for N, d, V in ((1, 8, 8), (136, 768, 50304), (8192, 2048, 128256), (131072, 64, 50304)):
        chunk = O._chunk(V)
        assert chunk % 256 == 0 and 256 <= chunk <= 65280
        for keep in range(3 if N <= O.FEW_ROWS else 2):
            rows = min(N, chunk) if keep < 2 else 2 * (-(-N // 64) * 64)
            kept, bwd = O._plan(N, d, V, chunk, keep, 2, True)
            assert kept >= N * (4 + 4 + 8 + 8 + 4 + 2 * V * (keep > 0)) + max(N, rows * (keep > 1)) * 2 * d + (V + 255) // 256 * min(N, chunk) * 8
            assert kept % 256 == 0 and bwd >= rows * V * 2 + rows * d * 4 * 2
        assert O._plan(N, d, V, chunk, 0, 0, False)[1] < bwd
    with pytest.raises(nv.NativeError):
        O._plan(O.FEW_ROWS + 1, 64, 64, 256, 2, 2, True)
    for bad in ((0, 8, 8, 256), (1, 0, 8, 256), (1, 8, 0, 256), (1, 8, 8, 0), (1, 8, 8, 100)):
        with pytest.raises(nv.NativeError):
            O._plan(*bad, 0, 2, True)


def _engine(**kw):
    from context_parallelism_b200.config import Config
    from context_parallelism_b200.engine import TrainEngine
    cfg = Config.from_env("llama", 1, env={}).replace(**{**dict(n_embd=32, n_layer=1, n_head=2, n_kv_head=2, head_dim=16, ffn_hidden=64, vocab_size=50, T=8,
                                                                B=4, dtype="fp32", checkpointing=False), **kw})
    return TrainEngine(cfg, torch.device("cpu"))


def _tokens(seed=0):
    t = torch.randint(0, 50, (4, 9), generator=torch.Generator().manual_seed(seed))
    x, y = t[:, :-1].contiguous(), t[:, 1:].contiguous()
    y[0, :3], y[2, 6:] = -100, -1
    return x, y


def test_engine_means():
    """Without weights a pass is the mean over counted tokens or pairs, and micro-batches add up to their mean."""
    eng = _engine()
    x, y = _tokens()
    old = eng.token_logprobs(x, y)
    n = int((y >= 0).sum())
    adv = torch.tensor([1.0, -0.5, 0.25, 2.0])
    out = eng.policy_forward_backward(x, y, old, adv, ref_logp=old - 0.2, kl_coef=0.5)
    per = adv[:, None].expand(4, 8)[y >= 0]
    assert float(out.loss) == pytest.approx(float(-per.mean() + 0.5 * (math.exp(-0.2) + 0.2 - 1)), rel=1e-5)
    assert float(out.terms[3]) == pytest.approx(1.0, rel=1e-6)
    one = eng.flat.grad.clone()
    eng.opt.zero_grad()
    for i in range(2):
        eng.policy_forward_backward(x, y, old, adv, ref_logp=old - 0.2, kl_coef=0.5, accum=2, last=i == 1)
    assert torch.allclose(eng.flat.grad, one, rtol=1e-5, atol=1e-8)
    eng.opt.zero_grad()
    wt = torch.full((4, 8), 1.0 / n)
    eng.policy_forward_backward(x, y, old.double(), adv[:, None].expand(4, 8), weights=wt, ref_logp=old - 0.2, kl_coef=0.5)
    assert torch.allclose(eng.flat.grad, one, rtol=1e-5, atol=1e-8)
    eng.opt.zero_grad()
    pref = eng.preference_forward_backward(x, y, old)
    assert float(pref.loss) == pytest.approx(math.log(2), rel=1e-5) and pref.ratios.abs().max() < 1e-4
    both = eng.flat.grad.clone()
    eng.opt.zero_grad()
    eng.preference_forward_backward(x, y, old, weights=torch.tensor([0.5, 0.5]))
    assert torch.allclose(eng.flat.grad, both, rtol=1e-5, atol=1e-8)


def test_engine_refuses():
    eng = _engine()
    x, y = _tokens()
    z = torch.zeros(4, 8)
    for bad in (torch.zeros(4, 7), torch.zeros(3, 8), torch.zeros(3), torch.zeros(4, 8, 1)):
        for kw in (dict(old_logp=bad), dict(advantages=bad), dict(weights=bad), dict(ref_logp=bad)):
            with pytest.raises(ValueError):
                eng.policy_forward_backward(x, y, **{**dict(old_logp=z, advantages=z), **kw})
        with pytest.raises(ValueError):
            eng.preference_forward_backward(x, y, bad)
    with pytest.raises(AssertionError):
        eng.preference_forward_backward(x[:3], y[:3], z[:3])


def test_what_counts_nothing_may_be_infinite():
    """A reference that gives a token no chance: without a KL coefficient it has no part in the loss, and a pair that it decides is decided."""
    x, w, t, g = _case(dtype=torch.float32)
    z, ref = torch.zeros(4, 5), torch.full((4, 5), -3.0)
    ref[0, 4] = -float("inf")
    a, b = O.linear_policy_loss(x, w, t, z - 3, z + 1, ref_logp=ref, n_valid=21), O.linear_policy_loss(x, w, t, z - 3, z + 1, n_valid=21)
    assert torch.equal(a.loss, b.loss) and float(a.terms[1]) == float("inf")
    for p, q in zip(torch.autograd.grad(a.loss, [x, w]), torch.autograd.grad(b.loss, [x, w])):
        assert torch.equal(p, q)
    out = O.linear_preference_loss(x, w, t, ref, n_valid=21)
    rest = torch.nn.functional.softplus(-0.1 * (out.ratios[1] - out.ratios[3]))
    assert float(out.loss) == pytest.approx(float(rest), rel=1e-6)


def test_main_grad_has_to_be_dense(calls):
    x, w = _t(2, 6, 64), _t(16, 64).requires_grad_()
    for bad in (torch.zeros(16, 64, dtype=torch.bfloat16), torch.zeros(64, 16).T, torch.zeros(16, 32)):
        head = O._Head(x, w, torch.zeros(2, 6, dtype=torch.int64), 16, True)
        head.w.main_grad = bad
        with pytest.raises(AssertionError):
            O._backward(head, torch.zeros(1), w, 0, 0, 0, None, False, True)
    assert not calls
