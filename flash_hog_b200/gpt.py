"""Gradient-norm-penalty training step on a pre-LN GPT, attention on the sm_100a kernels.

The benchmarked workload is a random-init 12-layer pre-LN GPT (d_model 768, 12 heads
of 64, causal, MLP 3072, vocab 32000, sequence 1024, 4 sequences per GPU) trained on
the objective

    L_total = L + lam * || dL/dtheta ||^2

whose gradient needs the double backward of every layer. Attention's double
backward runs on this package's kernels through ``dot_product_attention`` (two
nested autograd Functions, the analogue of the reference's nested custom_vjp).
With ``fused=True`` (the default for the "flash" model) LayerNorm, the MLP's GELU
and the cross-entropy loss run on the fused kernels of ``flash_hog_b200.fused`` --
forward, backward and double backward one kernel each -- as do the embeddings, dropout
with the residual additions and, for ``policy_objective``, the clipped policy loss; the
MLP's contractions run on cuBLAS (plain GEMMs). Data
parallelism: each rank computes the full step on its own token batch and the
parameter gradients (penalty terms included) are averaged with one NCCL
all-reduce over a flat buffer.

The reference repository has no model code; it only differentiates the attention
op twice (flash_hog/jax/attention.py:100-130). The same model with
``attention="naive"`` (torch math attention) is the parity reference in tests.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from flash_hog_b200 import _capi
from flash_hog_b200 import fused as fused_ops
from flash_hog_b200.attention import dot_product_attention


@dataclass
class GPTConfig:
    n_layer: int = 12
    d_model: int = 768
    n_head: int = 12
    d_mlp: int = 3072
    vocab: int = 32000
    seq_len: int = 1024
    dropout: float = 0.0       # after the embeddings and on both residual branches, in training mode
    embed_scale: float = 1.0   # factor on the token embeddings
    window: int | None = None  # sliding-window length of the attention (None: all earlier tokens)
    sinks: int = 0             # first tokens that stay visible behind the window


def naive_attention(q, k, v, is_causal=True, sliding_window_length=None, sink_tokens=0):
    """softmax(q k^T / sqrt(D) + causal mask) v in torch ops (BTNH), for reference runs."""
    scale = q.shape[-1] ** -0.5
    s = torch.einsum("bqhd,bkhd->bhqk", q.float(), k.float()) * scale
    if is_causal:
        keep = torch.ones(q.shape[1], k.shape[1], dtype=torch.bool, device=q.device).tril()
        if sliding_window_length is not None:
            far = torch.ones_like(keep).tril(-sliding_window_length)
            far[:, :sink_tokens] = False
            keep &= ~far
        s = s.masked_fill(~keep, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("bhqk,bkhd->bqhd", p, v.float()).to(q.dtype)


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig, attention, fused: bool):
        super().__init__()
        ln = fused_ops.LayerNorm if fused else nn.LayerNorm
        self.cfg, self.attention, self.fused = cfg, attention, fused
        self.mask = {} if cfg.window is None else dict(sliding_window_length=cfg.window, sink_tokens=cfg.sinks)
        self.act = fused_ops.gelu if fused else F.gelu
        self.ln1 = ln(cfg.d_model)
        self.qkv = nn.Linear(cfg.d_model, 3 * cfg.d_model)
        self.proj = nn.Linear(cfg.d_model, cfg.d_model)
        self.ln2 = ln(cfg.d_model)
        self.fc1 = nn.Linear(cfg.d_model, cfg.d_mlp)
        self.fc2 = nn.Linear(cfg.d_mlp, cfg.d_model)

    def _add(self, x, branch, seed, subsequence):
        """x + dropout(branch); ``seed`` None: without dropout."""
        if seed is None:
            return x + branch
        if self.fused:
            return fused_ops.dropout(branch, self.cfg.dropout, seed, subsequence=subsequence, residual=x)
        return x + F.dropout(branch, self.cfg.dropout)

    def forward(self, x, seed=None, index=0):
        b, t, d = x.shape
        h = self.cfg.n_head
        # One projection, then one copy to (3, b, t, h, dh): q, k and v come out contiguous,
        # so the attention op (and its backward and double backward) copies none of them.
        qkv = self.qkv(self.ln1(x)).view(b, t, 3, h, d // h).permute(2, 0, 1, 3, 4).contiguous()
        q, k, v = qkv.unbind(0)
        attn = self.attention(q, k, v, is_causal=True, **self.mask).reshape(b, t, d)
        x = self._add(x, self.proj(attn), seed, 2 * index + 1)
        return self._add(x, self.fc2(self.act(self.fc1(self.ln2(x)))), seed, 2 * index + 2)


class GPT(nn.Module):
    """Pre-LN GPT; ``attention`` is "flash" (the sm_100a op) or "naive" (torch math);
    ``fused`` (default: with "flash") puts the embeddings, LayerNorm, GELU and dropout on
    the fused kernels.

    With ``cfg.dropout`` each forward in training mode takes the next seed of the buffer
    ``dropout_seed`` (an int64 tensor of one element, from 0; give data-parallel ranks
    different starts): the masks of a step are a function of it, and steps replayed as a
    CUDA graph advance it too. It is not part of the state dict: save and restore it with a
    checkpoint, or a resumed run draws its first masks again.

    On the fused kernels a token outside the vocabulary does not stop the program, as
    ``nn.Embedding``'s check on the device does: its row is NaN, and with it the loss."""

    def __init__(self, cfg: GPTConfig, attention: str = "flash", fused: bool | None = None):
        super().__init__()
        if cfg.sinks and cfg.window is None:
            raise ValueError("GPTConfig.sinks apply to a window")
        fn = {"flash": dot_product_attention, "naive": naive_attention}[attention]
        fused = attention == "flash" if fused is None else fused
        self.cfg, self.fused = cfg, fused
        if fused:
            self.wte = fused_ops.Embedding(cfg.vocab, cfg.d_model, scale=cfg.embed_scale)
            self.wpe = fused_ops.Embedding(cfg.seq_len, cfg.d_model)
        else:
            self.wte = nn.Embedding(cfg.vocab, cfg.d_model)
            self.wpe = nn.Embedding(cfg.seq_len, cfg.d_model)
        if cfg.dropout > 0:
            self.register_buffer("dropout_seed", torch.zeros(1, dtype=torch.long), persistent=False)
        self.blocks = nn.ModuleList(Block(cfg, fn, fused) for _ in range(cfg.n_layer))
        self.ln_f = (fused_ops.LayerNorm if fused else nn.LayerNorm)(cfg.d_model)
        self.apply(self._init)
        for blk in self.blocks:  # GPT-2 style scaled init of the residual projections
            for lin in (blk.proj, blk.fc2):
                nn.init.normal_(lin.weight, std=0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, tokens):
        t = tokens.shape[1]
        if t > self.cfg.seq_len:  # the fused lookup would give rows of NaN
            raise IndexError(f"{t} tokens a row, but the model has {self.cfg.seq_len} positions")
        x = self.wte(tokens)
        if not self.fused and self.cfg.embed_scale != 1.0:
            x = x * self.cfg.embed_scale
        x = x + self.wpe(torch.arange(t, device=tokens.device))
        seed = None
        if self.training and self.cfg.dropout > 0:
            seed = self.dropout_seed.clone()  # the backward passes draw the masks of this step again
            self.dropout_seed += 1
            x = fused_ops.dropout(x, self.cfg.dropout, seed) if self.fused else F.dropout(x, self.cfg.dropout)
        for i, blk in enumerate(self.blocks):
            x = blk(x, seed, i)
        return self.ln_f(x) @ self.wte.weight.t()  # tied LM head


def penalty_objective(model: GPT, tokens: torch.Tensor, lam: float):
    """(L + lam ||dL/dtheta||^2, L, ||dL/dtheta||^2) for next-token cross-entropy L
    on ``tokens`` (B, T+1); the gradient is kept in the graph (create_graph)."""
    logits = model(tokens[:, :-1])
    if getattr(model, "fused", False):  # one kernel per pass, gradient in the logits' dtype
        loss = fused_ops.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())
    else:
        loss = F.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())
    params = [p for p in model.parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, params, create_graph=True)
    if getattr(model, "fused", False):  # multi-tensor kernels instead of three per parameter
        penalty = fused_ops.sum_of_squares(grads)
    else:
        penalty = sum((g.float() ** 2).sum() for g in grads)
    return loss + lam * penalty, loss.detach(), penalty.detach()


def _weight_share(weights, rows: int, device) -> torch.Tensor:
    """ranks / (the sum of the policy weights over all ranks), fp32 on ``device``; 0 where that
    sum is 0. One all-reduce of a scalar, no host synchronisation."""
    import torch.distributed as dist

    if weights is None:
        total = torch.full((), float(rows), dtype=torch.float64, device=device)
    else:
        total = weights.sum(dtype=torch.float64)
    dist.all_reduce(total)
    return torch.where(total == 0, 0.0, dist.get_world_size() / total).float()


def policy_objective(model: GPT, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                     lam: float = 0.0, distributed: bool = False, **kwargs):
    """(L + lam ||dL/dtheta||^2, L, log probabilities) for the clipped policy loss L of the
    tokens' own successors: ``tokens`` (B, T+1), everything else (B, T) over the T
    predictions (``weights`` of 0 for prompt and padding). ``kwargs`` are those of
    ``fused.policy_loss``. With ``lam`` 0 no gradient is taken here.

    ``distributed``: L is normalised by the mean over the ranks of their sums of weights
    (unless ``normalizer`` is given), so that the ranks' average of L, and of its gradient,
    is the weighted mean over all ranks' rows, also where one has few of them or none."""
    b, t = tokens.shape[0], tokens.shape[1] - 1
    rows = {n: v.reshape(b * t) if isinstance(v, torch.Tensor) else v for n, v in kwargs.items()}
    share = None
    if distributed and rows.get("normalizer") is None:
        share = _weight_share(rows.get("weights"), b * t, tokens.device)
        rows["normalizer"] = 1.0
    loss, logprobs = fused_ops.policy_loss(model(tokens[:, :-1]).flatten(0, 1), tokens[:, 1:].reshape(b * t),
                                           old_logprobs.reshape(b * t), advantages.reshape(b * t), **rows)
    if share is not None:
        loss = loss * share
    total = loss
    if lam:
        grads = torch.autograd.grad(loss, [p for p in model.parameters() if p.requires_grad], create_graph=True)
        total = loss + lam * fused_ops.sum_of_squares(grads)
    return total, loss.detach(), logprobs.view(b, t)


def allreduce_grads(model: nn.Module, group=None) -> None:
    """Averages parameter gradients over the ranks of ``group``: one all-reduce over
    a flat buffer (NCCL over NVLink on GPUs)."""
    import torch.distributed as dist

    params = [p for p in model.parameters() if p.grad is not None]
    if not params:
        return
    flat = torch.cat([p.grad.reshape(-1) for p in params])
    dist.all_reduce(flat, group=group)
    flat /= dist.get_world_size(group)
    off = 0
    for p in params:
        n = p.grad.numel()
        p.grad.copy_(flat[off:off + n].view_as(p.grad))
        off += n


class PenaltyStepGraph:
    """The compute of one grad-norm-penalty step -- forward, ``autograd.grad`` with
    ``create_graph``, the penalty and ``backward()`` into the parameters' ``.grad`` --
    captured once as a CUDA graph and replayed for each new token batch.

    The step launches thousands of small kernels (every layer differentiated twice),
    so launched one by one from Python it is bound by host launch latency; replayed
    as one graph it runs at the GPU's pace. Shapes, parameters and ``.grad`` tensors
    stay fixed (the graph writes the gradients in place: do not reset them with
    ``zero_grad(set_to_none=True)`` between replays); the data-parallel gradient
    all-reduce and the optimizer update run after the replay, outside the graph.
    With ``flat_grads`` (default: when a multi-rank process group is initialised) every
    ``.grad`` is a view of one flat fp32 buffer, which the graph zeroes first and the
    backward accumulates into, so the all-reduce runs on it in place (no gather or
    scatter copies); on one GPU the backward's own gradient tensors are kept instead
    (no zeroing, no accumulation pass). Autocast runs with its cast cache off, as graph
    capture requires.
    """

    def __init__(self, model: GPT, batch: int, lam: float, autocast: bool = True, warmup: int = 3,
                 flat_grads: bool | None = None):
        dev = next(model.parameters()).device
        self.model, self.lam, self.autocast = model, lam, autocast
        self.tokens = torch.zeros((batch, model.cfg.seq_len + 1), dtype=torch.long, device=dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):  # warm-up off the capture stream (allocator and library set-up)
            for _ in range(warmup):
                model.zero_grad(set_to_none=True)
                self._compute()
        torch.cuda.current_stream(dev).wait_stream(side)
        if flat_grads is None:
            import torch.distributed as dist

            flat_grads = dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1
        self.flat = None
        model.zero_grad(set_to_none=True)
        if flat_grads:
            params = [p for p in model.parameters() if p.requires_grad]
            if any(p.dtype != torch.float32 for p in params):
                raise ValueError("flat_grads keeps the gradients in one fp32 buffer: fp32 parameters only")
            self.flat = torch.zeros(sum(p.numel() for p in params), dtype=torch.float32, device=dev)
            off = 0
            for p in params:
                p.grad = self.flat[off:off + p.numel()].view_as(p)
                off += p.numel()
        self.graph = torch.cuda.CUDAGraph()
        n0 = _capi.launch_count()
        # thread_local: calls from other threads (NCCL's watchdog under torchrun) cannot
        # invalidate the capture.
        with torch.cuda.graph(self.graph, capture_error_mode="thread_local"):
            self.loss, self.penalty = self._compute()
        self.kernels_per_step = _capi.launch_count() - n0  # this library's kernels in one replay

    def _compute(self):
        if getattr(self, "flat", None) is not None:
            self.flat.zero_()  # the backward accumulates into the flat gradient views
        with torch.autocast(device_type="cuda", dtype=torch.bfloat16, enabled=self.autocast, cache_enabled=False):
            total, loss, penalty = penalty_objective(self.model, self.tokens, self.lam)
        total.backward()
        return loss, penalty

    def step(self, tokens: torch.Tensor, optimizer=None, distributed: bool = False):
        """Copies ``tokens`` into the graph's input, replays the step, then averages the
        gradients over the ranks (``distributed``) and applies ``optimizer``. Returns the
        (loss, penalty) device scalars, overwritten by the next replay."""
        self.tokens.copy_(tokens, non_blocking=True)
        self.graph.replay()
        if distributed and self.flat is not None:
            import torch.distributed as dist

            dist.all_reduce(self.flat)
            self.flat /= dist.get_world_size()
        elif distributed:
            allreduce_grads(self.model)
        if optimizer is not None:
            optimizer.step()
        return self.loss, self.penalty


def policy_step(model: GPT, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                lam: float = 0.0, optimizer=None, distributed: bool = False, autocast: bool = True, **kwargs):
    """One step on ``policy_objective``: its gradient, the data-parallel gradient average and
    the optimizer update. Returns (loss, log probabilities of the tokens (B, T)); with
    ``distributed`` the loss is this rank's share, whose average over the ranks is the loss.
    A ``normalizer`` given with ``distributed`` divides each rank's own sum."""
    with torch.autocast(device_type=tokens.device.type, dtype=torch.bfloat16,
                        enabled=autocast and tokens.device.type == "cuda"):
        total, loss, logprobs = policy_objective(model, tokens, old_logprobs, advantages, lam, distributed, **kwargs)
    if optimizer is not None:
        optimizer.zero_grad(set_to_none=True)
    total.backward()
    if distributed:
        allreduce_grads(model)
    if optimizer is not None:
        optimizer.step()
    return loss, logprobs


def train_step(model: GPT, tokens: torch.Tensor, lam: float, optimizer=None, distributed: bool = False,
               autocast: bool = True):
    """One grad-norm-penalty step: objective, its gradient (double backward), the
    data-parallel gradient average and the optimizer update. Returns (loss, penalty)."""
    dev = tokens.device.type
    with torch.autocast(device_type=dev, dtype=torch.bfloat16, enabled=autocast and dev == "cuda"):
        total, loss, penalty = penalty_objective(model, tokens, lam)
    if optimizer is not None:
        optimizer.zero_grad(set_to_none=True)
    total.backward()
    if distributed:
        allreduce_grads(model)
    if optimizer is not None:
        optimizer.step()
    return loss, penalty
