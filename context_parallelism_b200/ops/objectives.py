"""Fine-tuning objectives over the language-model head (``csrc/kernels/objectives.cu``): log-probabilities of tokens with a gradient, the
clipped policy loss with a KL term, the paired log-ratio (preference) loss.

All take final hidden states ``x`` ``[..., T, d]``, the head's weights ``w`` ``[V, d]`` and ``targets`` of ``x``'s leading shape, as
``xent.linear_cross_entropy`` does, and never hold ``[tokens, V]`` probabilities.  A token counts where its target is not negative (and its
weight not 0); the others cost nothing and whatever stands in their places, NaN included, is not read into a result.  They differ from the
cross entropy in two ways: tokens that count are gathered before the products, and gradients are made in ``backward``, so that any
gradient may come in and a loss that is never differentiated costs no more than its forward pass.

Each takes what the head's GEMM takes: bf16 ``x`` and ``w`` on one GPU, ``d`` and ``V`` multiples of 8.  ``n_valid``: rows of ``w`` from there on
are padding, with finite numbers in them.  Gradients of ``w`` are added to ``w.main_grad`` when it has one.  Nothing waits for the GPU, and all calls can be captured.
CPU tensors take the plain form."""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional, Tuple

import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

from .. import _native as nv
from .gemm import EPI_BF16, EPI_F32_ACC, acc_splits

# Of bf16 dlogits, the rows that go through the gradient's products at a time: each further chunk adds its dw to an fp32 buffer, 4 bytes read and
# written per weight (two chunks of 8192 rows, 128256 columns of 2048: 14.3 ms, one of 16384 13.9).
CHUNK_BYTES = 4 << 30
# Of logits in 16 bits, kept from the forward to the backward pass, a tenth of the GPU's memory; beyond, and where there is no room, they are
# computed again.
KEEP_BYTES = 16 << 30
# Width of the hidden states above which that is faster than to compute them again.  token_logprobs and its gradient, us, kept and computed
# again: 4608 x 50304, width 384 757 and 728 (without a pause), 512 871 and 876, 520 914 and 952, 640 918 and 967, 768 932 and 1029, 1024 1148 and
# 1278; 4608 x 128256, 2048 5513 and 6843.
KEEP_ABOVE = 512
# Rows up to which dlogits are the sum of two bf16 numbers, and logits always kept.  136 rows, width 768, 50304 columns: 14 us more of the GPU's 110,
# which a call of this size does not notice; beyond, the products would take up to twice as long.
FEW_ROWS = 256
PART = 4096                      # tokens of a sequence that one block adds up
COUNT_ROWS = 4096                # up to which rows are counted and gathered in one launch


class PolicyLoss(NamedTuple):
    """``loss``: the weighted sum; ``logp``: log-probabilities of the counted tokens, 0 elsewhere, and ``terms``: weighted sums of the clipped
    surrogate, of the KL estimate, of the tokens whose ratio was clipped, and of 1.  Only ``loss`` has a gradient."""
    loss: torch.Tensor
    logp: torch.Tensor
    terms: torch.Tensor


class PreferenceLoss(NamedTuple):
    """``loss``: the weighted sum over pairs; ``logp``: log-probabilities of the counted tokens, 0 elsewhere, and ``ratios``: ``sum(logp - ref_logp)``
    of every sequence.  Only ``loss`` has a gradient."""
    loss: torch.Tensor
    logp: torch.Tensor
    ratios: torch.Tensor


# ----------------------------------------------------------------------------- arguments
def _checked(x, w, targets, n_valid):
    assert x.dim() >= 2 and w.dim() == 2 and x.shape[-1] == w.shape[1], f"hidden states of {tuple(x.shape)}, weights of {tuple(w.shape)}"
    assert targets.shape == x.shape[:-1], f"targets of {tuple(targets.shape)} for hidden states of {tuple(x.shape)}"
    assert not targets.is_floating_point() and targets.dtype != torch.bool, f"targets of type {targets.dtype}"
    assert w.device == x.device and targets.device == x.device, f"operands on {x.device}, {w.device} and {targets.device}"
    assert 0 <= n_valid <= w.shape[0], f"n_valid={n_valid} of {w.shape[0]} rows"
    if x.is_cuda:
        assert x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16, f"the head computes in bf16 (got {x.dtype} and {w.dtype})"
        assert x.shape[-1] % 8 == 0 and w.shape[0] % 8 == 0, f"the head takes widths and rows in multiples of 8 (got {tuple(w.shape)})"
        assert targets.numel() < 1 << 31, f"{targets.numel()} tokens in one call"
    return targets.long().contiguous(), n_valid or w.shape[0]


def _per_token(name, t, like, optional=False):
    """fp32 values of the shape of ``like``, to which ``t`` may be broadcast (one value per sequence as ``[B, 1]``)."""
    if t is None and optional:
        return None
    assert isinstance(t, torch.Tensor) and t.is_floating_point() and t.device == like.device, f"{name} must be floating-point values on {like.device}"
    assert not t.requires_grad, f"{name} is a constant of the objective and has no gradient: detach it"
    if t.shape == like.shape:
        return t.float().contiguous()
    assert t.dim() == like.dim(), f"{name} of {tuple(t.shape)} for tokens of {tuple(like.shape)}"
    return t.float().expand(like.shape).contiguous()


# ----------------------------------------------------------------------------- launches
@functools.lru_cache(maxsize=4096)
def _plan(N: int, d: int, V: int, chunk: int, keep: int, dw: int, want_dx: bool) -> Tuple[int, int]:
    out = (ctypes.c_int64 * 2)()
    nv.check(nv.lib().cpb_objective_plan(N, d, V, chunk, keep, dw, want_dx, ctypes.addressof(out)), "objective_plan")
    return tuple(out)


@functools.lru_cache(maxsize=4096)
def _backward_launches(N: int, d: int, V: int, chunk: int, keep: int, dw: int, want_dx: bool) -> int:
    n = (keep == 0) + (dw == 2 and N > chunk)
    for r0 in range(0, N, chunk):
        rows = min(chunk, N - r0) if keep < 2 else 2 * (-(-N // 64) * 64)
        n += 1 + 2 * want_dx
        if dw:
            epi = EPI_BF16 if dw == 2 and N <= chunk else EPI_F32_ACC
            n += 1 + (acc_splits(V, d, rows, epi) > 1 and not (dw == 2 and N > chunk and r0 == 0))
    return n


def _chunk(V: int) -> int:
    return min(65280, max(256, CHUNK_BYTES // (2 * V) // 256 * 256))


class _Head:
    """What the backward pass needs of the forward pass beside the hidden states' and weights' own gradients."""

    def __init__(self, x, w, targets, n_valid, grad):
        self.shape, self.w, self.n_valid, self.grad = x.shape, w, n_valid, grad
        self.N, self.d, self.V = targets.numel(), x.shape[-1], w.shape[0]
        self.chunk = _chunk(self.V)
        # 0 nothing, 1 the logits, 2 those of few rows
        self.keep = 0 if not grad or 2 * self.N * self.V > KEEP_BYTES else 2 if self.N <= FEW_ROWS else int(self.d > KEEP_ABOVE)


def _rows16(t):
    """Whether rows of ``t`` can be read 16 bytes at a time where they are."""
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])


def _forward(x, w, targets, n_valid, grad, policy=None, more=0):
    """Log-probabilities, what is kept for the backward pass (and ``more`` bytes behind it), and for a policy loss the loss and its terms."""
    head = _Head(x, w, targets, n_valid, grad)
    logp = torch.empty(targets.shape, dtype=torch.float32, device=x.device)
    loss = terms = None
    if policy is not None:
        loss, terms = torch.empty((), dtype=torch.float32, device=x.device), torch.empty(4, dtype=torch.float32, device=x.device)
    if head.N == 0:
        return head, torch.empty(more, dtype=torch.uint8, device=x.device), logp, loss if loss is None else loss.zero_(), terms if terms is None else terms.zero_()
    xr = x if x.dim() <= 3 and _rows16(x) else _dense16(x)
    if xr.dim() == 3:
        T, sb, st = xr.shape[1], xr.stride(0), xr.stride(1)
    else:
        T, sb, st = head.N, 0, xr.stride(-2)
    wr = _weights(w)
    try:
        kept = torch.empty(_plan(head.N, head.d, head.V, head.chunk, head.keep, 0, False)[0] + more, dtype=torch.uint8, device=x.device)
    except torch.OutOfMemoryError:
        if not head.keep:
            raise
        head.keep = 0                                                # no room for logits: they are computed again
        kept = torch.empty(_plan(head.N, head.d, head.V, head.chunk, 0, 0, False)[0] + more, dtype=torch.uint8, device=x.device)
    old, adv, weights, ref, low, high, kl = policy or (None, None, None, None, 0.0, 0.0, 0.0)
    chunks = -(-head.N // head.chunk)
    nv.LAUNCHES[0] += (head.N > COUNT_ROWS) + 2 * chunks
    nv.call("objective_fwd", xr.data_ptr(), sb, st, head.N, T, head.d, wr.data_ptr(), wr.stride(0), head.V, n_valid, targets.data_ptr(), nv.ptr(old),
            nv.ptr(adv), nv.ptr(weights), nv.ptr(ref), low, high, kl, logp.data_ptr(), nv.ptr(loss), nv.ptr(terms), kept.data_ptr(), head.keep, head.chunk, nv.status_for(x.device).ptr(), nv.stream_ptr(x.device))
    return head, kept, logp, loss, terms


def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _weights(w):
    return w if w.stride(0) >= w.shape[1] and _rows16(w) else _dense16(w)


def _backward(head, kept, w, h, each, most, g, want_dx, want_dw):
    """``dx`` and ``dw`` (None where it went to ``main_grad``) from ``dloss / dlogp``, whose address is ``h``, and of which ``most`` is that of the largest
    size, or 0."""
    dx = torch.empty(head.shape, dtype=torch.bfloat16, device=w.device) if want_dx else None
    mg = getattr(head.w, "main_grad", None) if want_dw else None
    assert mg is None or (mg.dtype == torch.float32 and mg.is_contiguous() and mg.numel() == w.numel() and mg.device == w.device), "main_grad is fp32 and dense"
    own = torch.empty(w.shape, dtype=torch.bfloat16, device=w.device) if want_dw and mg is None else None
    kind = 0 if not want_dw else 1 if mg is not None else 2
    if head.N == 0:
        if own is not None:
            own.zero_()
    elif want_dx or want_dw:
        wr = _weights(w)
        scratch = torch.empty(_plan(head.N, head.d, head.V, head.chunk, head.keep, kind, want_dx)[1], dtype=torch.uint8, device=w.device)
        nv.LAUNCHES[0] += _backward_launches(head.N, head.d, head.V, head.chunk, head.keep, kind, want_dx) - 1
        nv.call("objective_bwd", head.N, head.d, wr.data_ptr(), wr.stride(0), head.V, head.n_valid, h, each, most, nv.ptr(g), nv.ptr(dx),
                (mg if mg is not None else own).data_ptr() if want_dw else 0, kind, kept.data_ptr(), head.keep, scratch.data_ptr(), head.chunk,
                nv.status_for(w.device).ptr(), nv.stream_ptr(w.device))
    if mg is not None:
        hook = getattr(head.w, "_grad_ready", None)
        if hook is not None:
            hook(head.w)
    return dx, own


def _sum_over(t, group):
    for g in () if group is None else group if isinstance(group, (list, tuple)) else (group,):
        dist.all_reduce(t, group=g)
    return t


# ----------------------------------------------------------------------------- autograd
class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, n_valid):
        ctx.head, kept, logp, *_ = _forward(x, w, targets, n_valid, any(ctx.needs_input_grad))
        ctx.save_for_backward(w, kept)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        w, kept = ctx.saved_tensors
        g = g.float().contiguous()
        dx, dw = _backward(ctx.head, kept, w, g.data_ptr(), 1, 0, None, *ctx.needs_input_grad[:2])
        return dx, dw, None, None


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, n_valid, policy):
        ctx.head, kept, logp, loss, terms = _forward(x, w, targets, n_valid, any(ctx.needs_input_grad), policy)
        ctx.save_for_backward(w, kept)
        ctx.mark_non_differentiable(logp, terms)
        ctx.set_materialize_grads(False)
        return loss, logp, terms

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return None, None, None, None, None
        w, kept = ctx.saved_tensors
        dx, dw = _backward(ctx.head, kept, w, 0, 0, 0, g.float().contiguous(), *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, n_valid, ref, weights, beta, smoothing, group):
        seqs, T = targets.shape
        parts = max(1, -(-T // PART))
        more = 8 * seqs * parts + 4 * (seqs + 1)                     # the sums, and dloss / dlogp of every sequence with the largest
        ctx.head, kept, logp, *_ = _forward(x, w, targets, n_valid, any(ctx.needs_input_grad), None, more)
        loss = torch.empty((), dtype=torch.float32, device=x.device)
        ratios = torch.empty(seqs, dtype=torch.float32, device=x.device)
        stream = nv.stream_ptr(x.device)
        sums = kept.data_ptr() + kept.numel() - more
        ctx.h = 8 * seqs * parts - more
        mine = (logp.data_ptr(), ref.data_ptr(), targets.data_ptr())
        if T == 0 or group is not None:
            t = kept[kept.numel() - more: kept.numel() + ctx.h].view(torch.float64)
            if T == 0:
                t.zero_()
            else:
                nv.call("sequence_sums", *mine, sums, seqs, T, parts, n_valid, stream)
            _sum_over(t, group)
            mine = (0, 0, 0)
        else:
            nv.LAUNCHES[0] += 1
        nv.call("preference", *mine, T, n_valid, sums, parts, seqs // 2, nv.ptr(weights), beta, smoothing, loss.data_ptr(), ratios.data_ptr(),
                sums + 8 * seqs * parts, stream)
        ctx.save_for_backward(w, kept)
        ctx.mark_non_differentiable(logp, ratios)
        ctx.set_materialize_grads(False)
        return loss, logp, ratios

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 9
        w, kept = ctx.saved_tensors
        end = kept.data_ptr() + kept.numel()
        dx, dw = _backward(ctx.head, kept, w, end + ctx.h, max(1, ctx.head.shape[1]), end - 4, g.float().contiguous(), *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None, None, None, None, None


# ----------------------------------------------------------------------------- public
def token_logprobs(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, n_valid: int = 0) -> torch.Tensor:
    """``log softmax(x w^T)[target]`` (fp32, ``targets``' shape; 0 where the target is negative), with the gradient of whatever is made of it."""
    targets, n_valid = _checked(x, w, targets, n_valid)
    if x.is_cuda:
        with nv.on(x.device):
            return _LogprobsFn.apply(x, w, targets, n_valid)
    return _plain_logprobs(x, w, targets, n_valid)


def linear_policy_loss(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                       weights: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip: Tuple[float, float] = (0.2, 0.2),
                       kl_coef: float = 0.0, n_valid: int = 0) -> PolicyLoss:
    """Sum over the counted tokens of ``weight (-min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (e^d - d - 1))`` with the ratio
    ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp`` (the KL term of a sampled token, never negative, against a reference policy).

    ``old_logp``: log-probabilities under the policy that drew the tokens, ``advantages`` ``A``, ``weights`` (None: 1) and ``ref_logp`` are
    constants of ``targets``' shape, or of one that broadcasts to it (``[B, 1]``: one advantage per answer).  The weights carry the mask and the
    mean: ``1 / counted tokens`` for a mean over tokens, ``1 / (B * tokens of the answer)`` for a mean over answers."""
    targets, n_valid = _checked(x, w, targets, n_valid)
    old, adv = _per_token("old_logp", old_logp, targets), _per_token("advantages", advantages, targets)
    wt, ref = _per_token("weights", weights, targets, True), _per_token("ref_logp", ref_logp, targets, True)
    low, high, kl = float(clip[0]), float(clip[1]), float(kl_coef)
    assert 0.0 <= low <= 1.0 and 0.0 <= high < float("inf"), f"clip={clip}"
    assert 0.0 <= kl < float("inf") and (ref is not None or kl == 0.0), f"kl_coef={kl_coef} with{'out' if ref is None else ''} reference log-probabilities"
    if x.is_cuda:
        with nv.on(x.device):
            return PolicyLoss(*_PolicyFn.apply(x, w, targets, n_valid, (old, adv, wt, ref, 1.0 - low, 1.0 + high, kl)))
    return _plain_policy(x, w, targets, n_valid, old, adv, wt, ref, 1.0 - low, 1.0 + high, kl)


def linear_preference_loss(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ref_logp: torch.Tensor, weights: Optional[torch.Tensor] = None,
                           beta: float = 0.1, smoothing: float = 0.0, n_valid: int = 0, group=None) -> PreferenceLoss:
    """Paired log-ratio loss.  ``x`` is ``[2 P, T, d]``: sequences ``0 .. P-1`` are the chosen answers, ``P + i`` the rejected one of pair ``i``.
    With ``R = sum over counted tokens of (logp - ref_logp)`` and ``z = beta (R_chosen - R_rejected)`` the sum over pairs of
    ``weight ((1 - smoothing) softplus(-z) + smoothing softplus(z))``.

    ``ref_logp`` ``[2 P, T]``: log-probabilities of the same tokens under the reference policy, token by token, so that differences are summed
    and not the difference of two long sums taken.  ``weights`` (``[P]``, None: 1); a pair of weight 0 has no part in loss and gradient.
    ``group``: the process group (or groups, one mesh axis each) that holds shards of these sequences; ``R`` is summed over it, every rank
    returns the loss of the whole pairs and the gradient of its own tokens."""
    assert x.dim() == 3 and x.shape[0] % 2 == 0 and x.shape[0] > 0, f"hidden states of {tuple(x.shape)}: chosen answers, then as many rejected ones"
    targets, n_valid = _checked(x, w, targets, n_valid)
    ref = _per_token("ref_logp", ref_logp, targets)
    if weights is not None:
        weights = _per_token("weights", weights, targets[: x.shape[0] // 2, 0] if targets.shape[1] else targets.new_empty(x.shape[0] // 2))
    beta, smoothing = float(beta), float(smoothing)
    assert 0.0 < beta < float("inf") and 0.0 <= smoothing <= 1.0, f"beta={beta}, smoothing={smoothing}"
    if x.is_cuda:
        assert x.shape[0] <= 65535, f"{x.shape[0]} sequences in one call"
        with nv.on(x.device):
            return PreferenceLoss(*_PreferenceFn.apply(x, w, targets, n_valid, ref, weights, beta, smoothing, group))
    return _plain_preference(x, w, targets, n_valid, ref, weights, beta, smoothing, group)


# ----------------------------------------------------------------------------- plain form
def _plain_logprobs(x, w, targets, n_valid):
    """On the CPU, and what the kernels are tested against; tokens that do not count are left out as they are there."""
    at = (targets.reshape(-1) >= 0).nonzero()[:, 0]
    t = targets.reshape(-1)[at]
    assert not t.numel() or int(t.max()) < n_valid, f"a target of {int(t.max())} of {n_valid}"
    logits = (x.reshape(-1, x.shape[-1])[at].float() if x.dtype != torch.float64 else x.reshape(-1, x.shape[-1])[at]) @ w.to(torch.promote_types(w.dtype, torch.float32))[:n_valid].T
    logp = torch.log_softmax(logits, 1).gather(1, t[:, None])[:, 0]
    return logp.new_zeros(targets.numel()).index_copy(0, at, logp).view(targets.shape)


def _plain_policy(x, w, targets, n_valid, old, adv, wt, ref, low, high, kl_coef):
    on = targets >= 0 if wt is None else (targets >= 0) & (wt != 0)
    logp = _plain_logprobs(x, w, torch.where(on, targets, -1), n_valid)
    lp, old, adv = logp[on].double(), old[on].double(), adv[on].double()
    wt = torch.ones_like(lp) if wt is None else wt[on].double()
    r = torch.where(adv == 0, 0.0, lp - old).exp()
    cut = ((adv > 0) & (r > high)) | ((adv < 0) & (r < low))
    surrogate = -torch.where(cut, r.detach().clamp(low, high), torch.where(cut, 0.0, r)) * adv
    kl = torch.zeros_like(lp) if ref is None else torch.expm1(ref[on].double() - lp) - (ref[on].double() - lp)
    terms = torch.stack([(wt * v).sum() for v in (surrogate, kl, cut.double(), torch.ones_like(lp))])
    return PolicyLoss((terms[0] + kl_coef * terms[1] if kl_coef else terms[0]).to(logp.dtype), logp.detach(), terms.detach().to(logp.dtype))


class _SumOver(torch.autograd.Function):
    """Sum over the ranks of a group; every rank's gradient is that of its own part."""
    @staticmethod
    def forward(ctx, t, group):
        return _sum_over(t.clone(), group)

    @staticmethod
    def backward(ctx, g):
        return g, None


def _plain_preference(x, w, targets, n_valid, ref, weights, beta, smoothing, group):
    on = targets >= 0
    logp = _plain_logprobs(x, w, targets, n_valid)
    ratios = torch.where(on, logp.double() - torch.where(on, ref, 0.0).double(), 0.0).sum(1)
    if group is not None:
        ratios = _SumOver.apply(ratios, group)
    chosen, rejected = ratios.chunk(2)
    if weights is not None:
        keep = weights != 0
        chosen, rejected, weights = chosen[keep], rejected[keep], weights[keep].double()
    z = beta * (chosen - rejected)
    sides = ((1 - smoothing, -z), (smoothing, z))                    # what counts nothing is left out, infinite or not
    each = sum(k * torch.nn.functional.softplus(v) for k, v in sides if k)
    return PreferenceLoss((each if weights is None else each * weights).sum().to(logp.dtype), logp.detach(), ratios.detach().to(logp.dtype))
