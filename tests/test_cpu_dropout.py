"""Counter-based dropout without a GPU: the generator, the place of an element, what is refused."""
import pytest
import torch

from context_parallelism_b200.ops import elementwise as E
from context_parallelism_b200.ops import reference as ref


def _seed(v=7):
    return torch.tensor([v], dtype=torch.int64)


def _philox_plain(c, k):
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def test_generator():
    zero = torch.zeros(1, dtype=torch.int64)
    # the published value of Philox4x32-7 for a counter and a key of nothing but zeros
    assert ref.philox(zero, 4, 0, zero)[0].tolist() == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    for row, site, seed in ((3, 0, 1), (2 ** 40 + 5, 2 ** 32 - 1, -1), (2 ** 32 - 1, 9, -2 ** 63), (2 ** 32, 9, 2 ** 63 - 1)):
        got = ref.philox(torch.tensor([row]), 10, site, torch.tensor([seed]))[0].tolist()
        key = [seed & 0xffffffff, seed >> 32 & 0xffffffff]
        want = sum((_philox_plain([g, row & 0xffffffff, row >> 32, site], key) for g in range(3)), [])
        assert got == want[:10]


@pytest.mark.parametrize("p", [0.01, 0.1, 0.5, 0.9])
def test_share_and_scale(p):
    x = torch.ones(4, 256, 64)
    y = E.dropout(x, E.Dropout(p, _seed()))
    kept = y != 0
    n = x.numel()
    # a binomial share: six standard deviations
    assert abs(float((~kept).sum()) / n - p) < 6 * (p * (1 - p) / n) ** 0.5
    assert torch.equal(y[kept], torch.full_like(y[kept], 1 / (1 - p)))
    for other in (E.Dropout(p, _seed(8)), E.Dropout(p, _seed(), site=1)):
        same = float(((E.dropout(x, other) != 0) == kept).float().mean())
        assert abs(same - (p * p + (1 - p) ** 2)) < 6 * 0.5 / n ** 0.5


def test_shards_draw_what_the_whole_draws():
    x, seed = torch.randn(2, 24, 16), _seed(5)
    whole = E.dropout(x, E.Dropout(0.3, seed, 4))
    for pos in (torch.arange(6, 12), torch.tensor([0, 1, 2, 21, 22, 23]), torch.arange(24).flip(0)):
        got = E.dropout(x[:, pos], E.Dropout(0.3, seed, 4, pos, 24))
        assert torch.equal(got, whole[:, pos])
    # rows of a matrix are one sequence
    assert torch.equal(E.dropout(x[0], E.Dropout(0.3, seed, 4)), whole[0])


@pytest.mark.parametrize("norm", ["layernorm", "rmsnorm"])
def test_norms_and_gradients(norm):
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(2, 5, 16, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w, b = (torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    drop = E.Dropout(0.4, _seed(11), 2)

    def run(x, r):
        args = (w, b, 1e-5) if norm == "layernorm" else (w, 1e-5)
        y, new = getattr(E, norm)(x, *args, r, drop)
        return new
    assert torch.autograd.gradcheck(run, (x, r))
    new = run(x, r)
    assert torch.equal(new, x + E.dropout(r, drop))


def test_dropped_values_do_not_matter():
    drop = E.Dropout(0.5, _seed(3))
    x = torch.randn(8, 32)
    gone = E.dropout(torch.ones(8, 32), drop) == 0
    y = E.dropout(torch.where(gone, torch.full_like(x, float("nan")), x), drop)
    assert bool(y.isfinite().all()) and not bool(y[gone].any())


def test_nothing_to_drop():
    x = torch.randn(3, 4, 8)
    assert E.dropout(x, E.Dropout(0.0, _seed())) is x
    y, new = E.rmsnorm(x, None, 1e-5, x, E.Dropout(0.0, _seed()))
    assert torch.equal(new, x + x)
    assert E.dropout(torch.zeros(0, 4, 8), E.Dropout(0.5, _seed())).shape == (0, 4, 8)


@pytest.mark.parametrize("drop", [
    E.Dropout(1.0, _seed()), E.Dropout(-0.1, _seed()), E.Dropout(float("nan"), _seed()), E.Dropout(0.1, torch.tensor([1], dtype=torch.int32)),
    E.Dropout(0.1, torch.zeros(2, dtype=torch.int64)), E.Dropout(0.1, torch.zeros(1, dtype=torch.int64, device="meta")),
    E.Dropout(0.1, _seed(), -1), E.Dropout(0.1, _seed(), 1 << 32), E.Dropout(0.1, _seed(), 0, torch.arange(4)),
    E.Dropout(0.1, _seed(), 0, torch.arange(5), 24), E.Dropout(0.1, _seed(), 0, torch.arange(4, dtype=torch.int32), 24),
    E.Dropout(0.1, _seed(), 0, torch.arange(4), 3), E.Dropout(0.1, _seed(), 0, None, 24)])
def test_refused(drop):
    x = torch.randn(2, 4, 8)
    with pytest.raises(AssertionError):
        E.dropout(x, drop)
    with pytest.raises(AssertionError):
        E.layernorm(x, torch.ones(8), None, 1e-5, x, drop)


def test_a_norm_without_a_branch_has_nothing_to_drop():
    x = torch.randn(2, 4, 8)
    with pytest.raises(AssertionError):
        E.rmsnorm(x, None, 1e-5, None, E.Dropout(0.1, _seed()))
    with pytest.raises(AssertionError):
        E.rmsnorm(x, None, 1e-5, x[:, :1], E.Dropout(0.1, _seed()))


def _engine(family="llama", recompute="none", dropout=0.2, **kw):
    from context_parallelism_b200.config import Config
    from context_parallelism_b200.engine import TrainEngine
    cfg = Config.from_env(family, 1, env={"CP_DROPOUT": str(dropout)}).replace(**{**dict(
        n_embd=64, n_layer=2, n_head=2, n_kv_head=2, head_dim=32, ffn_hidden=128, vocab_size=100, T=16, B=2, dtype="fp32", recompute=recompute,
        checkpointing=False), **kw})
    return TrainEngine(cfg, torch.device("cpu"))


def _batch(eng, seed=0):
    t = torch.randint(0, eng.cfg.vocab_size, (eng.cfg.B, eng.cfg.T + 1), generator=torch.Generator().manual_seed(seed))
    return t[:, :-1].contiguous(), t[:, 1:].contiguous()


@pytest.mark.parametrize("family", ["llama", "gpt2"])
def test_models(family):
    engines = [_engine(family, r) for r in ("none", "selective", "full")]
    for step in range(2):
        losses = [[float(e.forward_backward(*_batch(e, i), accum=2, last=i == 1)) for i in range(2)] for e in engines]
        assert losses[0] == losses[1] == losses[2]
        for e in engines[1:]:
            assert torch.equal(e.flat.grad, engines[0].flat.grad)
        for e in engines:
            e.optimizer_step()
    # the same tokens, another micro-batch, other elements; without gradients nothing is dropped
    a, b = engines[0], _engine(family, dropout=0.0)
    assert float(a.forward_backward(*_batch(a))) != float(a.forward_backward(*_batch(a)))
    b.flat.master.copy_(a.flat.master)
    assert float(a.eval_loss(*_batch(a))) == float(b.eval_loss(*_batch(b)))
    assert float(a.forward_backward(*_batch(a))) != float(b.forward_backward(*_batch(b)))
    idx, tgt, pos = a.shard_batch(*_batch(a))
    a.model.eval()
    assert torch.equal(a.model.hidden(idx, pos), b.model.hidden(idx, pos))


def test_every_site_drops_on_its_own():
    from context_parallelism_b200.ops import elementwise
    eng, seen = _engine(), []
    kept = elementwise.ref.dropout
    try:
        elementwise.ref.dropout = lambda x, drop: seen.append((drop.site, int(drop.seed), drop.seq_len, drop.pos.tolist())) or kept(x, drop)
        eng.forward_backward(*_batch(eng))
        eng.forward_backward(*_batch(eng))
    finally:
        elementwise.ref.dropout = kept
    pos = list(range(eng.cfg.T))
    seeds = [seen[0][1], seen[5][1]]
    assert seeds[0] != seeds[1] and seen == [(s, seed, eng.cfg.T, pos) for seed in seeds for s in (0, 1, 2, 3, 4)]


def test_seeds():
    from context_parallelism_b200.engine import dropout_seed
    seeds = {dropout_seed(1234, r, s, m) for r in range(4) for s in range(16) for m in range(8)}
    assert len(seeds) == 4 * 16 * 8 and all(-2 ** 63 <= s < 2 ** 63 for s in seeds)


def test_configuration():
    from context_parallelism_b200.config import Config
    assert Config.from_env("gpt2", 1, env={}).dropout == 0.0
    for bad in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError):
            Config.from_env("llama", 1, env={}).replace(dropout=bad).validate()
