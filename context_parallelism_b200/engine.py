"""Training engine: the public API a user (and ``bench.py``) drives.

``TrainEngine(cfg)`` builds the device mesh, the context-parallel context, the model, the flat
parameter store, the fused AdamW and the bucketed gradient reducer.  ``train_step(tokens, targets)``
takes FULL sequences ``[B, T]`` (pinned host or device int64), copies them to the device, gathers the
local shard with the same permutation for inputs and targets, and runs forward, backward, gradient
all-reduce (AVERAGE over all dp·cp ranks) and the optimiser step.  It returns the mean loss of the
local shard as a device scalar; ``global_loss`` averages it over ranks.  This is the step of the
reference trainers (Scripts/Blutrain/bluscriptCP.cpp:1653-1785, gpt2_cp_test.cpp:1497-1763).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.distributed as dist

from . import graphs
from .config import Config
from .ops import objectives, permute
from .ops.optim import AdamW, FlatParams
from .parallel.cp_attention import CPContext
from .parallel.ddp import GradReducer
from .parallel.mesh import DeviceMesh
from .utils.lr import cosine_lr, rewarmup_lr


class TrainEngine:
    def __init__(self, cfg: Config, device: Optional[torch.device] = None, mesh: Optional[DeviceMesh] = None,
                 standalone: bool = False):
        """``standalone=True`` builds a single-process engine (world size 1) even inside a distributed job; the
        parity tests use it for the unsharded reference run."""
        cfg.validate()
        self.cfg = cfg
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")
        self.device = device
        self.rank = dist.get_rank() if (dist.is_initialized() and not standalone) else 0
        self.world = dist.get_world_size() if (dist.is_initialized() and not standalone) else 1
        if cfg.world_size != self.world:
            raise ValueError(f"config world_size={cfg.world_size} but the job has {self.world} ranks")
        self.mesh = mesh or DeviceMesh.for_config(cfg, self.rank, self.world, create_groups=not standalone)
        self.cp = CPContext.from_mesh(cfg, self.mesh)
        if device.type == "cuda" and self.cp.cp_size > 1 and cfg.rotator == "fused":
            from .parallel.fused import FusedComm
            self.cp.fused = FusedComm.create(cfg, self.cp, device)
        self.native_pg = None
        import os
        if (device.type == "cuda" and self.cp.ring_size > 1 and cfg.rotator == "p2p" and self.cp.ring_group is not None
                and os.environ.get("CP_NATIVE_PG", "1") != "0"):
            # the NCCL baseline ring hops through the native process group: a communicator and a stream of its own
            from .parallel import rotators
            from .parallel.process_group import NativeProcessGroup
            self.native_pg = NativeProcessGroup.create(self.cp.ring_group, cfg.watchdog_s, True, device)
            rotators.NATIVE_GROUPS[id(self.cp.ring_group)] = self.native_pg
        if cfg.family == "gpt2":
            from .models.gpt2 import GPT2
            self.model = GPT2(cfg, self.cp, device)
        else:
            from .models.llama import Llama
            self.model = Llama(cfg, self.cp, device)
        if device.type == "cuda":
            from .ops import attention as _A
            _A.FP32_ACCURATE = bool(cfg.attn_fp32)
            if cfg.attn_fp32 and self.cp.cp_size > 1 and not (cfg.attn_mode == "ulysses" and cfg.rotator != "fused"):
                raise ValueError("ATTN_FP32=1 (fp32-accurate attention for parity runs) is supported on one GPU and for Ulysses "
                                 "with an NCCL rotator (CP_ROTATOR=alltoall); the other paths are built on the tensor-core kernels")
        bf16 = cfg.dtype == "bf16" and device.type == "cuda"
        if device.type == "cuda" and not bf16:
            raise ValueError("the CUDA kernels compute in bf16; CP_DTYPE=fp32 is the CPU oracle path")
        if self.world > 1:
            # every replica starts from rank 0's values (DDP ``init_sync``, bluscriptCP.cpp:1011)
            with torch.no_grad():
                for p in self.model.parameters():
                    dist.broadcast(p.data, 0)
        fused_world = self.cp.fused if (self.cp.fused is not None and self.cp.fused.covers_world()) else None
        shard = fused_world if (cfg.shard_optim and not cfg.no_grad_allreduce) else None
        self.flat = FlatParams(self.model.named_parameters(), bf16, cfg.grad_bucket_mb, shard)
        self.opt = AdamW(self.flat, cfg.max_lr, (cfg.beta1, cfg.beta2), cfg.adam_eps, cfg.weight_decay)
        fused_ar = fused_world.grad_allreduce_for(self.flat) if fused_world is not None else None
        self.reducer = GradReducer(self.flat, None, self.world, cfg.grad_bucket_mb, fused_ar,
                                   overlap=not (cfg.debug.no_overlap or cfg.debug.no_overlap_bwd))
        if cfg.no_grad_allreduce:
            self.reducer.enabled = False
        self.step_idx = 0
        self._micro = 0                     # micro-batches since the last update
        self.resume_anchor = -1
        self._pos_dev = {}
        self.last_grad_norm: Optional[torch.Tensor] = None

    # ------------------------------------------------------------------ helpers
    def lr_at(self, step: int) -> float:
        c = self.cfg
        anchor = c.rewarmup_anchor if c.rewarmup_anchor >= 0 else self.resume_anchor
        if c.rewarmup_steps > 0 and anchor >= 0:
            return rewarmup_lr(step, c.max_lr, c.min_lr, c.warmup_steps, c.max_steps, anchor, c.rewarmup_steps, c.rewarmup_peak)
        return cosine_lr(step, c.max_lr, c.min_lr, c.warmup_steps, c.max_steps)

    def local_pos(self, T: int) -> torch.Tensor:
        p = self._pos_dev.get(T)
        if p is None:
            p = self._pos_dev[T] = self.cp.local_positions(T).to(self.device)
        return p

    def shard_batch(self, tokens: torch.Tensor, targets: Optional[torch.Tensor]):
        """Full ``[B, T]`` (host or device) → local ``[B, T/cp]`` on the device, plus positions."""
        tokens = tokens.to(self.device, non_blocking=True)
        if targets is not None:
            targets = targets.to(self.device, non_blocking=True)
        pos = self.local_pos(tokens.shape[1])
        if self.cp.cp_size == 1:
            return tokens, targets, pos
        return (permute.gather_tokens(tokens, pos),
                permute.gather_tokens(targets, pos) if targets is not None else None, pos)

    # ------------------------------------------------------------------ one optimiser step
    def _taken(self, t):
        """``t``, or what it holds now when it is page-locked: the copy to the device is issued behind the GPU's work of earlier
        micro-batches, and the caller (a loader that hands out two buffers in turn) may write to ``t`` again as soon as the call returns.
        torch keeps the page-locked copy made here until the device has read it.  4 x 1024 tokens cost the host about 20 us."""
        if self.device.type != "cuda" or not isinstance(t, torch.Tensor) or t.is_cuda or not t.is_pinned():
            return t
        if torch.cuda.is_current_stream_capturing():                 # a graph of the caller's reads the caller's buffer at every replay
            return t
        return torch.empty(t.shape, dtype=t.dtype, pin_memory=True).copy_(t)

    def forward_backward(self, tokens, targets, accum: int = 1, last: bool = True) -> torch.Tensor:
        tokens, targets = self._taken(tokens), self._taken(targets)
        self._next_dropout()
        if self._recordable(targets):
            return self._recorded_micro_batch(tokens, targets, accum)
        idx, tgt, pos = self.shard_batch(tokens, targets)
        n_local = idx.numel()
        scale = 1.0 / (n_local * accum)
        self.reducer.begin_backward()
        ctx = self.reducer.no_sync() if not last else _null()
        with ctx:
            loss_sum = self.model.loss_sum(idx, tgt, pos, scale)
            # filled on the device: a host scalar copied there would wait for everything issued so far
            loss_sum.backward(torch.full_like(loss_sum, scale))
        if last:
            self.reducer.finish()
        return loss_sum.detach() / n_local

    def _next_dropout(self) -> None:
        """A seed of its own for every micro-batch, from what a resumed run knows as well: the configuration's seed, the step, the
        micro-batch and the data-parallel rank.  The ranks of a context-parallel group drop the same elements."""
        if self.cfg.dropout > 0:
            seed = dropout_seed(self.cfg.seed, self.cp.dp_rank, self.step_idx, self._micro)
            self.model.dropout_seed = torch.full((1,), seed, dtype=torch.int64, device=self.device)
            self._micro += 1

    def _recordable(self, targets) -> bool:
        """One GPU and nothing but this package's own forward and backward pass in the micro-batch."""
        return (self.device.type == "cuda" and not self.reducer.enabled and torch.is_grad_enabled() and isinstance(targets, torch.Tensor)
                and not torch.is_inference_mode_enabled() and self.model.recordable())

    def _recorded_micro_batch(self, tokens, targets, accum: int) -> torch.Tensor:
        scale = 1.0 / (tokens.numel() * accum)

        def micro_batch(idx, tgt, pos, *extra):
            loss_sum = self.model.loss_with(idx, tgt, pos, *extra, scale)
            loss_sum.backward(torch.full_like(loss_sum, scale))
            return (loss_sum.detach() / idx.numel(),)
        return self.model.graphs.run(f"micro-batch/{accum}", self.model, micro_batch,
                                     (tokens, targets, self.local_pos(tokens.shape[1]), *self.model.recorded_inputs()), self.device,
                                     graphs.model_flops(self.cfg, *tokens.shape, True), train=True)[0]

    # ------------------------------------------------------------------ fine-tuning objectives
    def _local_values(self, name: str, v, shape) -> Optional[torch.Tensor]:
        """fp32 constants of an objective for the local tokens, of ``shape``: whole sequences are sharded as tokens are, local shards (as
        ``token_logprobs`` returns them) and one value per sequence are taken as they are."""
        if v is None:
            return None
        v = self._taken(v).to(self.device, torch.float32, non_blocking=True)
        if v.dim() == 1:
            v = v[:, None]
        B, T = shape
        if v.dim() != 2 or v.shape[0] not in (1, B) or v.shape[1] not in (1, T, T * self.cp.cp_size):
            raise ValueError(f"{name} of shape {tuple(v.shape)} for {B} sequences of {T * self.cp.cp_size} tokens ({T} here)")
        if self.cp.cp_size > 1 and v.shape[1] == T * self.cp.cp_size:
            v = permute.gather_seq(v.contiguous(), self.local_pos(T * self.cp.cp_size), 1)
        return v

    @torch.no_grad()
    def token_logprobs(self, tokens, targets) -> torch.Tensor:
        """Log-probabilities of the local tokens' targets (fp32 ``[B, T/cp]``, 0 where the target is negative), without gradients: what the
        policy or a reference gives to the objectives below."""
        idx, tgt, pos = self.shard_batch(self._taken(tokens), self._taken(targets))
        return objectives.token_logprobs(self.model.hidden(idx, pos), self.model.head_weight(), tgt, self.cfg.vocab_size)

    def _objective(self, tokens, targets, last: bool, scale: float, loss_of):
        """Forward and backward pass of ``loss_of(hidden, head, local targets, targets)``, whose gradients count ``scale`` times."""
        tokens, targets = self._taken(tokens), self._taken(targets)
        self._next_dropout()
        idx, tgt, pos = self.shard_batch(tokens, targets)
        self.reducer.begin_backward()
        with self.reducer.no_sync() if not last else _null():
            out = loss_of(self.model.hidden(idx, pos), self.model.head_weight(), tgt,
                          tgt if self.cp.cp_size == 1 else targets.to(self.device, non_blocking=True))
            out.loss.backward(torch.full_like(out.loss, scale))
        if last:
            self.reducer.finish()
        return out._replace(loss=out.loss.detach())

    def policy_forward_backward(self, tokens, targets, old_logp, advantages, weights=None, ref_logp=None, clip=(0.2, 0.2), kl_coef: float = 0.0,
                                accum: int = 1, last: bool = True) -> objectives.PolicyLoss:
        """One micro-batch of ``objectives.linear_policy_loss`` in the place of ``forward_backward``; the update is ``optimizer_step``.

        ``tokens`` and ``targets`` are whole sequences ``[B, T]`` as for a training step, targets negative where a token does not count.
        Constants are ``[B, T]``, the local shards of ``token_logprobs``, or one value per sequence (``[B]``).  ``weights``: what a token
        counts in the sum over the batch (None: the mean over its counted tokens).  Loss and terms are, averaged over the ranks as
        ``global_loss`` does, those of the whole batch."""
        def loss_of(h, w, tgt, whole):
            wt = self._local_values("weights", weights, tgt.shape)
            if wt is None:
                wt = (1.0 / (whole >= 0).sum().clamp(min=1)).float().view(1, 1)
            return objectives.linear_policy_loss(
                h, w, tgt, self._local_values("old_logp", old_logp, tgt.shape), self._local_values("advantages", advantages, tgt.shape),
                wt * self.cp.cp_size, self._local_values("ref_logp", ref_logp, tgt.shape), clip, kl_coef, self.cfg.vocab_size)
        return self._objective(tokens, targets, last, 1.0 / accum, loss_of)

    def preference_forward_backward(self, tokens, targets, ref_logp, weights=None, beta: float = 0.1, smoothing: float = 0.0, accum: int = 1,
                                    last: bool = True) -> objectives.PreferenceLoss:
        """One micro-batch of ``objectives.linear_preference_loss``: ``tokens`` ``[2 P, T]`` are the chosen answers, then the rejected ones in the
        same order.  ``ref_logp`` as above.  ``weights`` ``[P]`` (None: the mean over the pairs).  The loss is that of the whole pairs on every
        rank of a context-parallel group."""
        def loss_of(h, w, tgt, whole):
            pairs = tgt.shape[0] // 2
            wt = (torch.full((pairs,), 1.0 / max(1, pairs), device=self.device) if weights is None
                  else self._taken(weights).to(self.device, torch.float32, non_blocking=True))
            group = None
            if self.cp.cp_size > 1:
                group = [self.cp.cp_group] if self.cp.cp_group is not None else [g for g in (self.cp.ring_group, self.cp.ulysses_group) if g is not None]
            return objectives.linear_preference_loss(h, w, tgt, self._local_values("ref_logp", ref_logp, tgt.shape), wt, beta, smoothing,
                                                     self.cfg.vocab_size, group)
        return self._objective(tokens, targets, last, self.cp.cp_size / accum, loss_of)

    def optimizer_step(self) -> torch.Tensor:
        lr = self.lr_at(self.step_idx)
        norm = self.opt.step(lr, self.cfg.grad_clip)
        self.opt.zero_grad()
        self.step_idx += 1
        self._micro = 0
        self.last_grad_norm = norm
        return norm

    def train_step(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        loss = self.forward_backward(tokens, targets, 1, True)
        self.optimizer_step()
        return loss

    def global_loss(self, local_loss: torch.Tensor) -> torch.Tensor:
        if self.world == 1:
            return local_loss
        t = local_loss.detach().clone().float().reshape(1)
        dist.all_reduce(t)
        return (t / self.world).squeeze(0)

    @torch.no_grad()
    def eval_loss(self, tokens, targets) -> torch.Tensor:
        idx, tgt, pos = self.shard_batch(tokens, targets)
        return self.model.loss_sum(idx, tgt, pos, 0.0) / idx.numel()

    def finish_step(self) -> None:
        """Host-side end of a step's device work, called by the trainers before the optimiser runs: wait for the
        stream with the ``CP_WATCHDOG_S`` deadline (a polling wait on a watched work handle, so a stuck collective
        raises ``StepTimeout`` instead of hanging the job), then turn any bounded-wait expiry or bounds failure the
        kernels reported into an exception, so that an update is never applied on top of stale data."""
        if self.device.type == "cuda":
            from .parallel.work import wait_for_stream
            wait_for_stream(self.device, self.cfg.watchdog_s, f"step {self.step_idx}")
        self.check_kernels()

    def check_kernels(self) -> None:
        """Raise if any kernel reported a bounded-wait expiry or a bounds failure (one small D2H read)."""
        if self.device.type == "cuda":
            from . import _native as nv
            nv.status_for(self.device).check("train step")

    def close(self) -> None:
        self.model.graphs.clear()
        if self.native_pg is not None:
            from .parallel import rotators
            torch.cuda.synchronize(self.device)
            rotators.NATIVE_GROUPS.pop(id(self.cp.ring_group), None)
            self.native_pg.close()
            self.native_pg = None
        if self.cp.fused is not None:
            self.cp.fused.close()
            self.cp.fused = None


def dropout_seed(*parts: int) -> int:
    """The parts mixed into 64 bits, signed (the steps of splitmix64, Steele, Lea, Flood 2014, once per part)."""
    mask, h = (1 << 64) - 1, 0
    for part in parts:
        h = (h + part + 0x9E3779B97F4A7C15) & mask
        h = ((h ^ h >> 30) * 0xBF58476D1CE4E5B9) & mask
        h = ((h ^ h >> 27) * 0x94D049BB133111EB) & mask
        h ^= h >> 31
    return h - (1 << 64) if h >> 63 else h


class _null:
    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False
