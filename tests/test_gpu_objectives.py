"""Fine-tuning objectives on the GPU against 64-bit results of the same bf16 operands, with bounds from the arithmetic."""
import math

import pytest
import torch

from context_parallelism_b200 import _native as nv
from context_parallelism_b200.ops import objectives as O

pytestmark = pytest.mark.gpu
BF16, FP32 = 2.0 ** -8, 2.0 ** -24                           # half a step


def _case(B, T, d, V, n_valid, spans="response", spread=3.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + B * T + d)
    x = torch.randn(B, T, d, device="cuda", generator=g).bfloat16()
    w = torch.zeros(V, d, device="cuda")
    w[:n_valid] = torch.randn(n_valid, d, device="cuda", generator=g) * spread / d ** 0.5
    w = w.bfloat16()
    t = torch.randint(0, n_valid, (B, T), device="cuda", generator=g)
    t[0, 0], t[-1, -1] = n_valid - 1, 0
    if spans == "response":
        for b in range(B):
            t[b, : T // 3 + b % 3] = -100
            t[b, T - T // 5 * (b % 2):] = -100
    elif spans == "scattered":
        t[torch.rand(B, T, device="cuda", generator=g) < 0.5] = -1
    elif spans == "none":
        t.fill_(-100)
    elif spans != "all":
        t.view(-1)[int(spans):] = -100                               # so many
    return x, w, t, g


class _Exact:
    """64 bits, with what the kernels' roundings may add up to."""

    def __init__(self, x, w, t, n_valid):
        self.x, self.w, self.t = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double()[:n_valid], t.reshape(-1)
        self.on = self.t >= 0
        z = self.x @ self.w.T
        # sums of d products and of n_valid exponentials in fp32, as the cross entropy's tests have it
        self.tol = 1e-5 * (1 + float(z.abs().max()))
        lp = torch.log_softmax(z, 1)
        self.p = lp.exp()
        few = self.on.numel() <= O.FEW_ROWS
        # From a width on, the distance of a logit to its tile's maximum is kept in f16, half a step 2^-11 of the distance, which is no more than
        # that to the row's maximum: the probability changes by a factor of e to that at most, (1 + 2 x) for x below a half.
        self.kept = (2 * 2.0 ** -11 * (z.amax(1, keepdim=True) - z)).clamp(max=1) if (x.shape[-1] > O.KEEP_ABOVE or few) and O.KEEP_BYTES else 0.0 * z
        # few rows: what the rounding of dlogits leaves, 2^-8 of them at most, is rounded in its turn
        self.dz = BF16 * BF16 if few and O.KEEP_BYTES else BF16
        self.logp = torch.where(self.on, lp.gather(1, self.t.clamp(min=0)[:, None])[:, 0], 0.0)
        self.V, self.shape = w.shape[0], x.shape

    def gradients(self, h, size):
        """Gradients for dloss / dlogp = h, and their bounds: dlogits and results are rounded to bf16, a logit is off by tol at most, and
        h, of which ``size`` bounds the parts, follows it."""
        h, size = torch.where(self.on, h, 0.0), torch.where(self.on, size, 0.0)
        dz = -h[:, None] * self.p
        dz.scatter_add_(1, self.t.clamp(min=0)[:, None], h[:, None])
        kept = self.kept * h.abs()[:, None] * self.p
        kept.scatter_(1, self.t.clamp(min=0)[:, None], 0.0)          # the target's probability is kept in fp32
        off = self.dz * dz.abs() + 3 * self.tol * size[:, None] * self.p + kept * (1 + self.dz)
        off.scatter_add_(1, self.t.clamp(min=0)[:, None], 3 * self.tol * size[:, None])
        dx, dw = dz @ self.w, torch.zeros(self.V, self.x.shape[1], dtype=torch.float64, device="cuda")
        ex, ew = off @ self.w.abs(), torch.zeros_like(dw)
        dw[: dz.shape[1]], ew[: dz.shape[1]] = dz.T @ self.x, off.T @ self.x.abs()
        # fp32 accumulation of the products: far below 1e-5 of the sum of their sizes
        sx, sw = 1e-5 * (dz.abs() @ self.w.abs()), torch.zeros_like(dw)
        sw[: dz.shape[1]] = 1e-5 * (dz.abs().T @ self.x.abs())
        return (dx.view(self.shape), (BF16 * dx.abs() + ex * (1 + BF16) + sx).view(self.shape)), (dw, BF16 * dw.abs() + ew * (1 + BF16) + sw)


def _within(got, want, bound, name):
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (name, float((err - bound).max()), float(err.max()))


# one row, less and more than a warp's, a CTA's and a pair's rows; columns in one tile, one more than a tile's, a last tile of padding only;
# both sides of the width from which logits are stored
SHAPES = [(1, 1, 64, 8, 8, "all"), (1, 5, 8, 16, 16, "all"), (1, 300, 16, 24, 20, "scattered"), (1, 31, 64, 64, 57, "all"), (3, 11, 72, 264, 257, "response"), (2, 65, 128, 512, 250, "scattered"),
          (4, 96, 384, 1024, 1000, "response"), (2, 150, 1024, 8192, 8192, "scattered"), (2, 150, 1032, 4096, 4090, "response"),
          (1, 700, 1032, 512, 512, "scattered"), (8, 200, 384, 50304, 50257, "response"), (1, 520, 2048, 1000, 990, "all"),
          (2, 40, 64, 512, 500, "none"), *[(1, 600, 64, 264, 260, str(n)) for n in (1, 63, 64, 65, 255, 256, 257, 320, 512)],
          *[(1, 600, 1032, 264, 260, str(n)) for n in (1, 64, 65, 256, 257)]]


@pytest.fixture(params=["one chunk", "chunks", "chunks, logits again"])
def chunks(request, monkeypatch):
    if request.param != "one chunk":
        monkeypatch.setattr(O, "_chunk", lambda V: 256)
    if request.param == "chunks, logits again":
        monkeypatch.setattr(O, "KEEP_BYTES", 0)


@pytest.mark.parametrize("B,T,d,V,n_valid,spans", SHAPES)
def test_logprobs(B, T, d, V, n_valid, spans, chunks):
    x, w, t, g = _case(B, T, d, V, n_valid, spans)
    x.requires_grad_(), w.requires_grad_()
    u = torch.randn(B, T, device="cuda", generator=g)
    logp = O.token_logprobs(x, w, t, n_valid)
    dx, dw = torch.autograd.grad(logp, [x, w], u)
    e = _Exact(x, w, t, n_valid)
    _within(logp.reshape(-1), e.logp, e.tol, "logp")
    (wx, bx), (ww, bw) = e.gradients(u.reshape(-1).double(), u.reshape(-1).double().abs())
    _within(dx, wx, bx, "dx")
    _within(dw, ww, bw, "dw")
    assert not bool(dx[t < 0].any()) and not bool(dw[n_valid:].any())
    with torch.no_grad():
        assert torch.equal(O.token_logprobs(x, w, t, n_valid), logp)
    nv.status_for(x.device).check()


def _policy_inputs(e, g, t, clip, kl):
    """Ratios in and beyond the clipped range, none within twice the error of a border."""
    n = t.numel()
    moved = 0.3 * torch.randn(n, device="cuda", generator=g).double()
    for border in (math.log1p(-clip[0]) if clip[0] < 1 else -1e9, math.log1p(clip[1])):
        moved = torch.where((moved - border).abs() < 2 * e.tol + 1e-5, border + 4 * e.tol + 1e-4, moved)
    old = (e.logp - moved).float().view(t.shape)
    adv = (torch.randn(n, device="cuda", generator=g) + 0.3).view(t.shape)
    adv.view(-1)[::7] = 0
    wt = torch.rand(t.shape, device="cuda", generator=g) / n
    wt.view(-1)[::5] = 0
    ref = (e.logp + 0.3 * torch.randn(n, device="cuda", generator=g)).float().view(t.shape) if kl is not None else None
    return old, adv, wt, ref


@pytest.mark.parametrize("kl,clip", [(None, (0.2, 0.2)), (0.0, (0.2, 0.28)), (0.3, (1.0, 0.0))])
@pytest.mark.parametrize("B,T,d,V,n_valid,spans", SHAPES)
def test_policy(B, T, d, V, n_valid, spans, kl, clip, chunks):
    x, w, t, g = _case(B, T, d, V, n_valid, spans)
    e = _Exact(x, w, t, n_valid)
    old, adv, wt, ref = _policy_inputs(e, g, t, clip, kl)
    x.requires_grad_(), w.requires_grad_()
    out = O.linear_policy_loss(x, w, t, old, adv, wt, ref, clip, kl or 0.0, n_valid)
    up = torch.tensor(1.7, device="cuda")
    dx, dw = torch.autograd.grad(out.loss, [x, w], up)
    e.on = e.on & (wt.reshape(-1) != 0)
    e.logp = torch.where(e.on, e.logp, 0.0)
    lp, o, a, k = (v.reshape(-1).double() for v in (e.logp, old, adv, wt))
    r = (lp - o).exp()
    cut = ((a > 0) & (r > 1 + clip[1])) | ((a < 0) & (r < 1 - clip[0]))
    surrogate, h = -torch.minimum(r * a, r.clamp(1 - clip[0], 1 + clip[1]) * a), torch.where(cut, 0.0, -a * r)
    size, klv = a.abs() * r, torch.zeros_like(r)
    if ref is not None:
        d_ = ref.reshape(-1).double() - lp
        klv, h, size = torch.expm1(d_) - d_, h - (kl or 0.0) * torch.expm1(d_), size + (kl or 0.0) * (d_.exp() + 1)
    k = torch.where(e.on, k, 0.0)
    terms = torch.stack([(k * v).sum() for v in (surrogate, klv, cut.double(), torch.ones_like(k))])
    loss = terms[0] + (kl or 0.0) * terms[1]
    _within(out.logp.reshape(-1), e.logp, e.tol, "logp")
    # a term moves with logp by its derivative
    move = torch.stack([(k * a.abs() * r).sum(), 0 * loss if ref is None else (k * ((ref.reshape(-1).double() - lp).exp() - 1).abs()).sum() + e.tol * k.sum(), 0 * loss, 0 * loss]) * e.tol * 1.1
    _within(out.terms, terms, move + 4 * FP32 * terms.abs(), "terms")
    _within(out.loss, loss, move[0] + (kl or 0.0) * move[1] + 4 * FP32 * loss.abs(), "loss")
    (wx, bx), (ww, bw) = e.gradients(1.7 * k * h, 1.7 * k * size)
    _within(dx, wx, bx, "dx")
    _within(dw, ww, bw, "dw")
    nv.status_for(x.device).check()


@pytest.mark.parametrize("smoothing,beta", [(0.0, 0.1), (0.1, 0.02), (1.0, 2.0)])
@pytest.mark.parametrize("B,T,d,V,n_valid,spans", [(2, 1, 64, 8, 8, "all"), (2, 33, 72, 264, 257, "response"), (6, 50, 384, 1024, 1000, "scattered"),
                                                   (4, 300, 1032, 512, 500, "response"), (2, 5000, 64, 512, 500, "response"), (2, 40, 64, 512, 500, "none"),
                                                   (4, 64, 128, 264, 264, "64")])
def test_preference(B, T, d, V, n_valid, spans, smoothing, beta, chunks):
    x, w, t, g = _case(B, T, d, V, n_valid, spans)
    e = _Exact(x, w, t, n_valid)
    ref = (e.logp + 0.1 * torch.randn(B * T, device="cuda", generator=g)).float().view(B, T)
    wt = torch.rand(B // 2, device="cuda", generator=g) + 0.5
    x.requires_grad_(), w.requires_grad_()
    out = O.linear_preference_loss(x, w, t, ref, wt, beta, smoothing, n_valid)
    diff = torch.where(e.on, e.logp - ref.reshape(-1).double(), 0.0).view(B, T)
    R, off = diff.sum(1), e.tol * e.on.view(B, T).sum(1)
    z, far = beta * (R[: B // 2] - R[B // 2:]), beta * (off[: B // 2] + off[B // 2:])
    soft = torch.nn.functional.softplus
    loss = (wt.double() * ((1 - smoothing) * soft(-z) + smoothing * soft(z))).sum()
    dh = wt.double() * beta * (smoothing * torch.sigmoid(z) - (1 - smoothing) * torch.sigmoid(-z))
    _within(out.logp.reshape(-1), e.logp, e.tol, "logp")
    _within(out.ratios, R, off + FP32 * R.abs(), "ratios")
    _within(out.loss, loss, (wt.double() * far).sum() + 2 * FP32 * loss, "loss")
    h = torch.cat([dh, -dh])[:, None].expand(B, T).reshape(-1)
    # the derivative of h with respect to z is at most weight x beta / 4
    size = h.abs() + torch.cat([wt, wt]).double()[:, None].expand(B, T).reshape(-1) * beta / 4 * torch.cat([far, far])[:, None].expand(B, T).reshape(-1) / (3 * e.tol)
    # the gradient is taken at a power of two, which has to go out of it again whatever comes in
    for up in (0.6, -3.0, 2.0 ** 40, 1e-20, 0.0):
        dx, dw = torch.autograd.grad(out.loss, [x, w], torch.tensor(up, device="cuda"), retain_graph=True)
        (wx, bx), (ww, bw) = e.gradients(up * h, abs(up) * size)
        _within(dx, wx, bx, f"dx at {up}")
        _within(dw, ww, bw, f"dw at {up}")


def _calls(x, w, t, old, adv, ref, n_valid):
    def policy():
        out = O.linear_policy_loss(x, w, t, old, adv, ref_logp=ref, kl_coef=0.1, n_valid=n_valid)
        return [out.loss, out.logp, out.terms]

    def preference():
        out = O.linear_preference_loss(x, w, t, ref, n_valid=n_valid)
        return [out.loss, out.logp, out.ratios]
    return dict(policy=policy, preference=preference, logprobs=lambda: [(v := O.token_logprobs(x, w, t, n_valid)).sum(), v])


def _setup(d=1032, B=4, T=150, grad=True):
    x, w, t, g = _case(B, T, d, 512, 500, "response")
    old, adv, ref = (torch.randn(B, T, device="cuda", generator=g) - s for s in (7, 0, 7))
    if grad:
        x.requires_grad_(), w.requires_grad_()
    return x, w, t, old, adv, ref


@pytest.mark.parametrize("d", [64, 1032])
@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_values_in_masked_places(kind, d):
    x, w, t, old, adv, ref = _setup(d, grad=False)
    off = t < 0
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min], device="cuda")[torch.arange(int(off.sum()), device="cuda") % 4]
    results = []
    for spoil in (False, True):
        a = [v.clone() for v in (x, old, adv, ref)]
        if spoil:
            for v in a:
                v[off] = (bad if v.dim() == 2 else bad[:, None].expand(-1, d)).to(v.dtype)
        a[0].requires_grad_(), w.requires_grad_()
        outs = _calls(a[0], w, t, *a[1:], 500)[kind]()
        results.append([*outs, *torch.autograd.grad(outs[0], [a[0], w])])
    for p, q in zip(*results):
        assert torch.equal(p, q)
    assert bool(results[0][-2].isfinite().all())


@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_a_value_that_is_no_number_stays_in_its_row(kind):
    x, w, t, old, adv, ref = _setup(64, grad=False)
    x[1, 60, 3] = float("nan")
    assert int(t[1, 60]) >= 0
    x.requires_grad_(), w.requires_grad_()
    outs = _calls(x, w, t, old, adv, ref, 500)[kind]()
    assert bool(outs[0].isnan()) and int(outs[1].isnan().sum()) == 1
    dx, dw = torch.autograd.grad(outs[0], [x, w])
    rows = dx.isnan().any(-1)
    # a pair's gradient has both sequences' log-ratios in it
    want = torch.zeros_like(rows)
    if kind == "preference":
        want[[1, 3]] = t[[1, 3]] >= 0
    else:
        want[1, 60] = True
    assert torch.equal(rows, want) and bool(dw.isnan().any())


@pytest.mark.parametrize("d", [64, 1032])
@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_frozen_operands_accumulation_and_repeats(kind, d):
    x, w, t, old, adv, ref = _setup(d)
    call = _calls(x, w, t, old, adv, ref, 500)[kind]
    outs = call()
    dx, dw = torch.autograd.grad(outs[0], [x, w], retain_graph=True)
    again = torch.autograd.grad(outs[0], [x, w])
    other = call()
    for a, b in zip((*outs, dx, dw, dx, dw), (*other, *torch.autograd.grad(other[0], [x, w]), *again)):
        assert torch.equal(a, b)                                     # bit for bit
    x.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(call()[0], [w])[0], dw)
    x.requires_grad_(), w.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(call()[0], [x])[0], dx)
    w.requires_grad_()
    w.main_grad = torch.full(w.shape, 0.5, device="cuda")
    told = []
    w._grad_ready = told.append
    call()                                                           # no gradient asked for: none is added
    assert not told and bool((w.main_grad == 0.5).all())
    call()[0].backward()
    assert torch.equal(x.grad, dx) and told == [w] and w.grad is None
    added = w.main_grad.double() - 0.5
    assert bool(((added - dw.double()).abs() <= 2 ** -8 * dw.double().abs() + 4 * FP32).all())


@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_strides_types_and_streams(kind):
    x, w, t, old, adv, ref = _setup(72)
    want = _calls(x, w, t, old, adv, ref, 500)[kind]()
    wg = torch.autograd.grad(want[0], [x, w])
    B, T, d = x.shape
    wide = torch.zeros(B, T + 1, d + 8, device="cuda", dtype=torch.bfloat16)
    odd = torch.zeros(B, T, d + 1, device="cuda", dtype=torch.bfloat16)
    late = torch.zeros(T, B, d, device="cuda", dtype=torch.bfloat16)
    views = [wide[:, :-1, :d], odd[..., 1:], late.transpose(0, 1), torch.zeros(B * T * d + 4, device="cuda", dtype=torch.bfloat16)[4:].view(B, T, d),
             torch.zeros(B, d, T, device="cuda", dtype=torch.bfloat16).transpose(1, 2)]
    W = torch.zeros(512, d + 16, device="cuda", dtype=torch.bfloat16)[:, 8:-8]
    WT = torch.zeros(d, 512, device="cuda", dtype=torch.bfloat16).T
    side = torch.cuda.Stream()
    for i, v in enumerate(views):
        v.copy_(x.detach())
        wv = (W, WT)[i % 2].copy_(w.detach())
        v, wv = v.detach().requires_grad_(), wv.detach().requires_grad_()
        args = (t.int(), old.double(), adv.half().float(), ref) if i % 2 else (t.t().contiguous().t(), old, adv.half().float(), ref.t().contiguous().t())
        exp = _calls(x, w, t, old, adv.half().float(), ref, 500)[kind]()
        eg = torch.autograd.grad(exp[0], [x, w])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            outs = _calls(v, wv, *args, 500)[kind]()
            grads = torch.autograd.grad(outs[0], [v, wv])
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip((*outs, *grads), (*exp, *eg)):
            assert torch.equal(a, b)
    assert all(g.isfinite().all() for g in wg)


def test_broadcast_advantages_and_shapes():
    x, w, t, old, adv, ref = _setup(64)
    per = adv[:, :1]
    a = O.linear_policy_loss(x, w, t, old, per, n_valid=500)
    b = O.linear_policy_loss(x, w, t, old, per.expand(-1, t.shape[1]).contiguous(), torch.ones_like(old), n_valid=500)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.terms, b.terms)
    flat = O.token_logprobs(x.reshape(-1, 64), w, t.reshape(-1), 500)
    deep = O.token_logprobs(x.view(2, 2, -1, 64), w, t.view(2, 2, -1), 500)
    assert flat.shape == (t.numel(),) and torch.equal(flat, deep.reshape(-1)) and torch.equal(deep.view(t.shape), O.token_logprobs(x, w, t, 500))
    none = x[:, :0]
    assert O.token_logprobs(none, w, t[:, :0]).shape == (4, 0)
    for out in (O.linear_policy_loss(none, w, t[:, :0], old[:, :0], adv[:, :0]), O.linear_preference_loss(none, w, t[:, :0], ref[:, :0])):
        dx, dw = torch.autograd.grad(out.loss, [x, w])
        assert not bool(dx.any()) and not bool(dw.any())
    assert float(out.loss) == pytest.approx(2 * math.log(2))


def test_zero_weight_pairs():
    x, w, t, old, adv, ref = _setup(64)
    spoiled = ref.clone()
    spoiled[[1, 3]] = float("nan")
    wt = torch.tensor([1.5, 0.0], device="cuda")
    a, b = (O.linear_preference_loss(x, w, t, r, wt, n_valid=500) for r in (ref, spoiled))
    assert torch.equal(a.loss, b.loss) and bool(a.loss.isfinite())
    for p, q in zip(torch.autograd.grad(a.loss, [x, w]), torch.autograd.grad(b.loss, [x, w])):
        assert torch.equal(p, q)
    assert bool(b.ratios[[1, 3]].isnan().all())


def test_far_ratios():
    """A ratio beyond fp32 under an advantage that clips it, or of nothing, leaves loss and gradient finite."""
    x, w, t, old, adv, ref = _setup(64)
    logp = O.token_logprobs(x, w, t, 500).detach()
    for a in (1.0, 0.0):
        out = O.linear_policy_loss(x, w, t, logp - 200, torch.full_like(adv, a), n_valid=500)
        n = int((t >= 0).sum())
        assert float(out.loss) == pytest.approx(-1.2 * a * n, rel=1e-6) and float(out.terms[2]) == n * a
        assert not any(bool(v.any()) for v in torch.autograd.grad(out.loss, [x, w]))


def test_a_target_outside_the_vocabulary_is_reported():
    x, w, t, old, adv, ref = _setup(64)
    bad = t.clone()
    bad[0, 100] = 500
    got = O.token_logprobs(x, w, bad, 500)
    with pytest.raises(nv.NativeError, match="index out of range"):
        nv.status_for(x.device).check()
    want = O.token_logprobs(x, w, t, 500).clone()
    want[0, 100] = 0
    assert torch.equal(got, want)
    nv.status_for(x.device).check()


@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_two_captured_graphs(kind):
    """Captured calls take new inputs at each replay, and two graphs have no workspace in common."""
    sets = [_setup(1032), _setup(64, T=200)]
    graphs, outs = [], []
    for s in sets:
        call = _calls(*s, 500)[kind]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call()[0], s[:2])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
            outs.append([*(v.detach() for v in o), *torch.autograd.grad(o[0], s[:2])])
        graphs.append(graph)
    for turn in range(3):
        for s in sets:
            with torch.no_grad():
                s[0].copy_(s[0] * 0.75)
                s[2][0, 60 + 10 * turn:] = -100                      # fewer tokens than when it was captured, then more
                s[2][1, : 20 * turn] = 3
        streams = [torch.cuda.Stream() for _ in graphs]
        for graph, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for s, got in zip(sets, outs):
            o = _calls(*s, 500)[kind]()
            for a, b in zip(got, [*o, *torch.autograd.grad(o[0], s[:2])]):
                assert torch.equal(a, b)


def test_what_counts_nothing_may_be_infinite():
    x, w, t, old, adv, ref = _setup(64)
    ref = ref.clone()
    ref[0, 100] = -float("inf")
    assert int(t[0, 100]) >= 0
    a, b = (O.linear_policy_loss(x, w, t, old, adv, ref_logp=r, n_valid=500) for r in (ref, None))
    assert torch.equal(a.loss, b.loss) and float(a.terms[1]) == float("inf")
    for p, q in zip(torch.autograd.grad(a.loss, [x, w]), torch.autograd.grad(b.loss, [x, w])):
        assert torch.equal(p, q)
    out = O.linear_preference_loss(x, w, t, ref, n_valid=500)
    rest = torch.nn.functional.softplus(-0.1 * (out.ratios[1] - out.ratios[3]).double())
    assert float(out.loss) == pytest.approx(float(rest), rel=1e-5)
    assert all(bool(v.isfinite().all()) for v in torch.autograd.grad(out.loss, [x, w]))


@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_threads_modes_and_recomputation(kind):
    """Calls of two threads on streams of their own, without autograd, and recomputed by a checkpoint."""
    import threading

    from torch.utils.checkpoint import checkpoint
    sets = [_setup(1032), _setup(64, T=200)]
    want = []
    for s in sets:
        o = _calls(*s, 500)[kind]()
        want.append([*(v.detach() for v in o), *torch.autograd.grad(o[0], s[:2])])
    got, errors = [None, None], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    o = _calls(*sets[i], 500)[kind]()
                    got[i] = [*(v.detach() for v in o), *torch.autograd.grad(o[0], sets[i][:2])]
            st.synchronize()
        except Exception as e:                                       # shown by the assertion below
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for s, w in zip(sets, want):
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                assert all(torch.equal(p, q) for p, q in zip(_calls(*s, 500)[kind](), w))
        x, rest = s[0], s[1:]
        loss = checkpoint(lambda x: _calls(x, *rest, 500)[kind]()[0], x, use_reentrant=False)
        for p, q in zip(torch.autograd.grad(loss, s[:2]), w[-2:]):
            assert torch.equal(p, q)


def test_more_than_two_to_the_31_logits():
    """Offsets of kept logits and dlogits pass 32 bits; the same rows in two calls give the same."""
    B, T, d, V = 2, 8600, 520, 128256
    x, w, t, g = _case(B, T, d, V, V, "all")
    assert B * T * V > 1 << 31
    x.requires_grad_(), w.requires_grad_()
    u = torch.randn(B, T, device="cuda", generator=g)
    logp = O.token_logprobs(x, w, t)
    dx, dw = torch.autograd.grad(logp, [x, w], u)
    parts = [O.token_logprobs(x[b], w, t[b]) for b in range(2)]
    grads = [torch.autograd.grad(p, [x, w], u[b]) for b, p in enumerate(parts)]
    assert torch.equal(logp, torch.stack(parts))
    # dx: the same dlogits, their products added in other ranges of K and rounded once more to bf16; dw: halves that were rounded each
    whole = sum(g[0] for g in grads).double()
    assert float((dx.double() - whole).norm() / whole.norm()) < BF16
    whole = sum(g[1].double() for g in grads)
    assert float((dw.double() - whole).norm() / whole.norm()) < 2 * BF16


def test_no_room_for_logits(monkeypatch):
    x, w, t, old, adv, ref = _setup(1032)
    want = [torch.autograd.grad(_calls(x, w, t, old, adv, ref, 500)[k]()[0], [x, w]) for k in ("policy", "preference", "logprobs")]
    real, refused = torch.empty, []

    def empty(*shape, **kw):
        if kw.get("dtype") == torch.uint8 and shape[0] >= 2 * x.shape[0] * x.shape[1] * 512 + x.numel() * 2:
            refused.append(shape[0])
            raise torch.OutOfMemoryError("no room")
        return real(*shape, **kw)
    monkeypatch.setattr(torch, "empty", empty)
    got = []
    for k in ("policy", "preference", "logprobs"):
        outs = _calls(x, w, t, old, adv, ref, 500)[k]()
        monkeypatch.setattr(torch, "empty", real)
        got.append(torch.autograd.grad(outs[0], [x, w]))
        monkeypatch.setattr(torch, "empty", empty)
    assert len(refused) == 3
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            # each is rounded twice to bf16, of which the second time alone is at one place
            assert float((p.double() - q.double()).norm() / q.double().norm()) < 4 * BF16


# more rows than one launch takes: 65280
@pytest.mark.parametrize("B,T,d,V,n_valid,spans", [(1, 70001, 64, 264, 260, "scattered"), (3, 40000, 520, 128, 128, "response"), (1, 66000, 128, 64, 60, "65281"),
                                                   (1, 66000, 128, 64, 60, "3"), (70000, 2, 8, 16, 16, "none")])
def test_more_rows_than_a_launch_takes(B, T, d, V, n_valid, spans):
    assert B * T > O._chunk(V)
    test_logprobs(B, T, d, V, n_valid, spans, None)
    if spans != "none":
        test_policy(B, T, d, V, n_valid, spans, 0.3, (0.2, 0.28), None)


@pytest.mark.parametrize("B,T,d", [(65534, 1, 64), (3000, 7, 520), (2, 70000, 64)])
def test_many_pairs_and_long_ones(B, T, d):
    test_preference(B, T, d, 64, 60, "scattered", 0.1, 0.3, None)
