"""Counter-based dropout kernels against 64-bit results of the same mask (``reference.philox``)."""
import pytest
import torch

from context_parallelism_b200.ops import elementwise as E
from context_parallelism_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8                                             # half a step


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen).bfloat16()


def _case(shape, p, seed=3, site=5, pos=None, seq_len=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + shape[-1])
    drop = E.Dropout(p, torch.tensor([seed * 0x123456789abcdef], device="cuda"), site, pos, seq_len)
    T = shape[-2]
    t = torch.arange(T, device="cuda") if pos is None else pos
    n = shape[0] if len(shape) == 3 else 1
    row = (torch.arange(n, device="cuda")[:, None] * (seq_len or T) + t).reshape(-1)
    keep = (ref.philox(row, shape[-1], site, drop.seed) >= int(p * 2 ** 32)).view(shape)
    return gen, drop, keep


def _pos(kind, T):
    if kind == "whole":
        return None, 0
    if kind == "far":                                        # sequences longer than 2^32 rows
        return torch.arange(T, device="cuda") * 7 + 2 ** 33 + 1, 2 ** 36
    half = torch.arange(T // 2, device="cuda")               # a HeadTail shard
    return torch.cat([half, half + 3 * T, torch.arange(T % 2, device="cuda") + 4 * T]), 4 * T + 1


# every width class of the norms' kernels, single rows, odd numbers of rows
SHAPES = [(3, 1001, 64), (1, 2500, 520), (1, 1, 8), (1, 3, 64), (2, 33, 264), (3, 17, 384), (1, 136, 768), (4, 5, 1032), (2, 129, 2048), (1, 9, 2056), (1, 40, 4096), (131, 512)]


@pytest.mark.parametrize("kind", ["whole", "shard", "far"])
@pytest.mark.parametrize("shape", SHAPES)
def test_alone(shape, kind):
    pos, seq_len = _pos(kind, shape[-2])
    gen, drop, keep = _case(shape, 0.3, pos=pos, seq_len=seq_len)
    x, dy = _randn(gen, *shape).requires_grad_(), _randn(gen, *shape)
    y = E.dropout(x, drop)
    dx, = torch.autograd.grad(y, x, dy)
    scale = torch.tensor(1 / (1 - 0.3), dtype=torch.float32, device="cuda")
    assert torch.equal(y, torch.where(keep, x.float() * scale, 0.0).bfloat16())
    assert torch.equal(dx, torch.where(keep, dy.float() * scale, 0.0).bfloat16())


@pytest.mark.parametrize("kind", ["whole", "shard"])
@pytest.mark.parametrize("norm", ["layernorm", "rmsnorm"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("p", [0.1, 0.75])
def test_norms(shape, norm, p, kind):
    pos, seq_len = _pos(kind, shape[-2])
    gen, drop, keep = _case(shape, p, pos=pos, seq_len=seq_len)
    d = shape[-1]
    x, r = _randn(gen, *shape).requires_grad_(), _randn(gen, *shape).requires_grad_()
    dy, dnew = _randn(gen, *shape), _randn(gen, *shape)
    w = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).requires_grad_()
    b = (0.1 * torch.randn(d, device="cuda", generator=gen)).requires_grad_()
    layer = norm == "layernorm"
    y, new = E.layernorm(x, w, b, 1e-5, r, drop) if layer else E.rmsnorm(x, w, 1e-5, r, drop)
    leaves = [x, r, w] + ([b] if layer else [])
    dx, dr, *dw = torch.autograd.grad([y, new], leaves, [dy, dnew])
    scale = 1 / (1 - p)
    again = E.layernorm(x, w, b, 1e-5, r, drop) if layer else E.rmsnorm(x, w, 1e-5, r, drop)
    for p1, p2 in zip((y, new, dx, dr, *dw), (*again, *torch.autograd.grad(again, leaves, [dy, dnew]))):
        assert torch.equal(p1, p2)                                   # bit for bit
    assert torch.equal(new, (x.float() + torch.where(keep, r.float() * scale, 0.0)).bfloat16())
    v = new.detach().double().requires_grad_()
    W, B = w.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    Y = torch.nn.functional.layer_norm(v, (d,), W, B, 1e-5) if layer else torch.nn.functional.rms_norm(v, (d,), W, 1e-5)
    dv, *DW = torch.autograd.grad(Y, [v, W] + ([B] if layer else []), dy.double())
    # 32-bit arithmetic on rows of d: sums of d terms of order one and a reciprocal root, 2^-24 each; generously 64 of them.  A row of
    # few columns may have next to no variance: its rstd multiplies that.
    rstd = ((v - v.mean(-1, keepdim=True) if layer else v).pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
    slack = 64 * 2.0 ** -24 * (1 + rstd) * (1 + v.abs().amax(-1, keepdim=True)) * (1 + rstd * v.abs().amax(-1, keepdim=True)) * (1 + dy.double().abs().amax(-1, keepdim=True))
    want = dv + dnew.double()
    for name, got, exact in (("y", y, Y), ("dx", dx, want), ("dr", dr, torch.where(keep, want * scale, 0.0))):
        err = (got.double() - exact).abs()
        assert bool((err <= BF16 * exact.abs() + slack * scale).all()), (name, float((err - BF16 * exact.abs()).max()))
    assert not bool(dr[~keep].any())
    hat = (Y - (B if layer else 0)) / W
    rows = v.numel() // d
    for got, exact, terms in zip(dw, DW, ((dy.double() * hat).abs(), dy.double().abs())):
        bound = (terms.reshape(-1, d).sum(0) * (rows + 8) * 2.0 ** -24 + (slack * (1 + dy.double().abs())).reshape(rows, -1).sum(0))
        assert bool(((got.double() - exact).abs() <= bound).all())


def test_strided_and_other_stream():
    gen, drop, keep = _case((2, 10, 64), 0.5)
    wide = _randn(gen, 2, 10, 136)
    x = wide[..., 4:68]                                       # rows that start at 8 bytes
    y = E.dropout(x, drop)
    assert torch.equal(y, torch.where(keep, x.float() * 2, 0.0).bfloat16())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = E.dropout(x.transpose(0, 1).contiguous().transpose(0, 1), drop)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(z, y)


def test_a_captured_call_takes_the_seed_it_finds():
    gen, drop, _ = _case((2, 50, 256), 0.2)
    x = _randn(gen, 2, 50, 256).requires_grad_()
    r = _randn(gen, 2, 50, 256).requires_grad_()
    w = torch.ones(256, device="cuda", requires_grad=True)

    def step():
        y, new = E.rmsnorm(E.dropout(x, drop), w, 1e-5, r, drop)
        return [new.detach(), *torch.autograd.grad(y.float().sum(), [x, r])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, -5, 2 ** 60):
        drop.seed.fill_(seed)
        graph.replay()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_no_rows():
    _, drop, _ = _case((1, 4, 64), 0.5)
    assert E.dropout(torch.zeros(0, 4, 64, device="cuda", dtype=torch.bfloat16), drop).shape == (0, 4, 64)


def test_refused():
    from context_parallelism_b200._native import NativeError
    _, drop, _ = _case((1, 4, 64), 0.5)
    with pytest.raises(AssertionError):
        E.dropout(torch.zeros(1, 4, 64, device="cuda"), drop)
    with pytest.raises(AssertionError):
        E.dropout(torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16), drop._replace(seed=drop.seed.cpu()))
    x, w = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16), torch.ones(68, device="cuda")
    for bad in (w[:64].bfloat16(), w[:56], w[1:65], w[:64].cpu(), torch.ones(64, 2, device="cuda")[:, 0]):
        with pytest.raises(AssertionError):
            E.rmsnorm(x, bad, 1e-5, x, drop)
        with pytest.raises(AssertionError):
            E.layernorm(x, w[:64], bad, 1e-5, x, drop)
    with pytest.raises(NativeError):
        E.dropout(torch.zeros(1, 4, 60, device="cuda", dtype=torch.bfloat16), drop)


def _engine(family, recompute="none", **kw):
    from context_parallelism_b200.config import Config
    from context_parallelism_b200.engine import TrainEngine
    cfg = Config.from_env(family, 1, env={"CP_DROPOUT": "0.1"}).replace(**{**dict(
        n_embd=256, n_layer=2, n_head=4, n_kv_head=2 if family == "llama" else 4, head_dim=64, ffn_hidden=512 if family == "llama" else 1024,
        vocab_size=1000, T=200, B=2, max_steps=20, warmup_steps=1, checkpointing=False, recompute=recompute, dtype="bf16",
        weight_tying=family == "gpt2"), **kw})
    return TrainEngine(cfg, torch.device("cuda", 0))


def _batch(eng, seed):
    t = torch.randint(0, eng.cfg.vocab_size, (eng.cfg.B, eng.cfg.T + 1), generator=torch.Generator().manual_seed(seed))
    return t[:, :-1].contiguous().pin_memory(), t[:, 1:].contiguous().pin_memory()


@pytest.mark.parametrize("family,recompute", [("llama", "none"), ("llama", "selective"), ("llama", "full"), ("gpt2", "none"), ("gpt2", "selective")])
def test_recorded_micro_batches(family, recompute):
    """Every replay drops what its own seed says, as an eager call does."""
    from util import assert_close
    a, b = _engine(family, recompute), _engine(family)
    b._recordable = lambda *args: False
    for i in range(5):
        la, lb = (float(e.forward_backward(*_batch(e, 0), accum=5, last=i == 4)) for e in (a, b))
        assert abs(la - lb) <= 1e-4 * abs(lb)
    # dQ, norm, bias and embedding gradients are fp32 sums in arrival order; two eager passes differ as much
    assert_close(a.flat.grad, b.flat.grad, cos=0.99999, rel=1e-2, name="grad")
    assert len([r for r in a.model.graphs._records.values() if r is not None]) == 1
    a.check_kernels()


def test_recorded_evaluation_drops_nothing():
    a, b = _engine("llama"), _engine("llama", dropout=0.0)
    b.flat.master.copy_(a.flat.master), b.flat.sync_compute_copy()
    for i in range(4):
        x, y, pos = a.shard_batch(*_batch(a, i))
        a.forward_backward(*_batch(a, i))
        assert torch.equal(a.model.per_token_nll(x, y, pos), b.model.per_token_nll(x, y, pos))


def test_parameters_add_to_what_is_there():
    gen, drop, _ = _case((2, 50, 256), 0.2)
    x, r, dy = (_randn(gen, 2, 50, 256) for _ in range(3))
    x.requires_grad_()
    grads = []
    for main in ((), (0, 1), (0,), (1,)):
        w, b = both = [torch.ones(256, device="cuda", requires_grad=True) for _ in range(2)]
        told = []
        for i in main:
            both[i].main_grad = torch.full((256,), 2.0, device="cuda")
            both[i]._grad_ready = told.append
        y, _ = E.layernorm(x, w, b, 1e-5, r, drop)
        y.backward(dy)
        grads.append([both[i].main_grad - 2.0 if i in main else both[i].grad for i in range(2)])
        assert len(told) == len(main)
    for p, q in ((p, q) for other in grads[1:] for p, q in zip(grads[0], other)):
        assert float((p - q).abs().max()) <= 2.0 ** -24 * (4 + 2 * float(p.abs().max()))        # added to two and taken from it again
    y, _ = E.rmsnorm(x, None, 1e-5, r, drop)                          # no parameters at all
    y.backward(dy)


def test_no_rows_through_a_norm():
    drop = E.Dropout(0.1, torch.tensor([1], device="cuda"))
    x, r = (torch.zeros(2, 0, 64, device="cuda", dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    w, b = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))
    y, new = E.layernorm(x, w, b, 1e-5, r, drop)
    assert y.shape == new.shape == x.shape
    (y.sum() + new.sum()).backward()
    assert x.grad.shape == r.grad.shape == x.shape and not bool(w.grad.any()) and not bool(b.grad.any())


def test_second_derivatives_are_refused():
    gen, drop, _ = _case((2, 5, 64), 0.2)
    x, r, dy = (_randn(gen, 2, 5, 64).requires_grad_() for _ in range(3))
    for y in (E.dropout(x, drop), E.rmsnorm(x, None, 1e-5, r, drop)[0]):
        dx, = torch.autograd.grad(y, x, dy, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.float().sum().backward()
