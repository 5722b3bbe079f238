"""Multi-process parity worker of the fine-tuning objectives (launched by torch.distributed.run from the tests): losses, log-probabilities and
gradients of the policy and preference passes, with dropout, under context (and data) parallelism against the unsharded engine."""
import argparse
import json
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--family", default="llama")
    ap.add_argument("--mode", default="ring")
    ap.add_argument("--rotator", default="p2p")
    ap.add_argument("--cp", type=int, default=0)
    ap.add_argument("--ulysses", type=int, default=1)
    ap.add_argument("--recompute", default="none")
    a = ap.parse_args()
    from context_parallelism_b200.config import Config
    from context_parallelism_b200.engine import TrainEngine
    from context_parallelism_b200.parallel.mesh import init_distributed
    rank, world, _ = init_distributed("gloo", timeout_s=120)
    dev, cp, B, T = torch.device("cpu"), a.cp or world, 4, 64
    cfg = Config.from_env(a.family, world, env={}).replace(
        cp_size=cp, attn_mode=a.mode, rotator=a.rotator, ulysses_size=a.ulysses, recompute=a.recompute, n_embd=64, n_layer=2, n_head=4,
        n_kv_head=2 if a.family == "llama" else 4, head_dim=16, ffn_hidden=128 if a.family == "llama" else 256, vocab_size=211, T=T, B=B, max_steps=50,
        warmup_steps=1, checkpointing=False, dtype="fp32", weight_tying=a.family == "gpt2", dropout=0.1)
    eng = TrainEngine(cfg, dev)
    ref = TrainEngine(cfg.replace(world_size=1, cp_size=1, ulysses_size=1, attn_mode="ring"), dev, standalone=True)
    dp, g = world // cp, torch.Generator().manual_seed(11)
    tok = torch.randint(0, cfg.vocab_size, (B * dp, T + 1), generator=g)
    x, y = tok[:, :-1].contiguous(), tok[:, 1:].contiguous()
    for b in range(B * dp):
        y[b, : 5 + 7 * b] = -100
        y[b, T - b:] = -100
    adv, noise = torch.randn(B * dp, generator=g), 0.3 * torch.randn(B * dp, T, generator=g)
    pos = eng.local_pos(T)
    worst = {}

    def note(name, got, want):
        worst[name] = max(worst.get(name, 0.0), float((got - want).norm() / want.norm()))
    mine = slice(eng.cp.dp_rank * B, (eng.cp.dp_rank + 1) * B)
    for step in range(3):
        kind = ("policy", "preference", "policy")[step]
        whole = torch.cat([ref.token_logprobs(x[d * B:(d + 1) * B], y[d * B:(d + 1) * B]) for d in range(dp)])
        local = eng.token_logprobs(x[mine], y[mine])
        note("logp", local, whole[mine][:, pos])
        old = whole + noise

        def passes(e, sl, accum, last, sharded):
            ref_logp = (old + 0.1)[sl]
            if sharded and step == 2:                                # constants as the local shards that token_logprobs gives
                ref_logp = ref_logp[:, pos]
            if kind == "policy":
                return e.policy_forward_backward(x[sl], y[sl], old[sl], adv[sl], ref_logp=ref_logp, kl_coef=0.1, accum=accum, last=last)
            return e.preference_forward_backward(x[sl], y[sl], ref_logp, smoothing=0.1, accum=accum, last=last)
        out = passes(eng, mine, 1, True, True)
        loss = eng.global_loss(out.loss)
        want = 0.0
        for d in range(dp):
            ref.cp.dp_rank, ref._micro = d, 0                        # the slice drops what the rank that has it drops
            w = passes(ref, slice(d * B, (d + 1) * B), dp, d == dp - 1, False)
            want = want + w.loss / dp
            if d == eng.cp.dp_rank:
                note("logp of the pass", out.logp, w.logp[:, pos])
                if kind == "preference":
                    note("ratios", out.ratios, w.ratios)
        note("loss", loss, want)
        note("gradient", eng.flat.grad, ref.flat.grad)
        eng.optimizer_step(), ref.optimizer_step()
        ref.flat.master.copy_(eng.flat.master), ref.flat.sync_compute_copy()
    # fp32 in another order of sums: 2^-24 each, some thousand terms
    ok = all(v < 2e-5 for v in worst.values())
    res = torch.tensor([1.0 if ok else 0.0])
    dist.all_reduce(res, op=dist.ReduceOp.MIN)
    if rank == 0:
        print(json.dumps({"ok": bool(res.item() > 0.5), "worst": worst}))
    eng.close()
    dist.barrier()
    dist.destroy_process_group()
    sys.exit(0 if res.item() > 0.5 else 1)


if __name__ == "__main__":
    main()
