"""The ops of a GPT training step around attention, with fused first- and second-order
backward kernels.

The grad-norm-penalty step (L + lam ||dL/dtheta||^2, configuration 5) differentiates
every layer's backward once more. In torch autograd the double backward of
LayerNorm and of GELU is a composite of many elementwise and reduction kernels;
here each pass is one kernel of ``csrc/ln_gelu.cu`` through the C ABI
(``fh_layernorm_*``, ``fh_gelu``), with two nested autograd Functions per op in the
same pattern as the attention op (``flash_hog/jax/attention.py:52-60, 100-130``):
the outer Function's backward is the inner Function, whose backward is the
double backward. Third-order derivatives raise.

Embedding and dropout are linear and differentiable to any order.

* ``LayerNorm`` (module) / ``layer_norm(x, w, b, eps)``: fp32 arithmetic; under
  autocast the inputs are cast to fp32, as autocast does for torch's layer_norm.
* ``gelu(x)``: exact GELU (x Phi(x)) in the input dtype (fp32 or bf16; fp32
  arithmetic), as ``torch.nn.functional.gelu`` under autocast.
* ``cross_entropy(logits, targets)``: the mean cross entropy of (rows, vocab) logits
  (fp32 or bf16, fp32 arithmetic) as ``torch.nn.functional.cross_entropy`` on the
  logits cast to fp32; its gradient comes back in the logits' dtype, as autocast
  would cast it for the head's matmul (``csrc/xent.cu``, ``fh_xent_*``).
* ``embedding(tokens, weight, scale, padding_idx)`` / ``Embedding`` (module): the scaled
  lookup, its gradient by sorted tokens (``csrc/embed.cu``, ``fh_embed_*``).
* ``dropout(x, p, seed, subsequence, residual)``: dropout from a counter-based generator,
  the mask never stored, with the residual addition (``csrc/dropout.cu``, ``fh_dropout``).
* ``policy_loss(logits, actions, old_logprobs, advantages, ...)``: the clipped policy loss
  with a KL term, beside ``cross_entropy`` (``csrc/policy.cu``, ``fh_policy_*``).
* ``sum_of_squares(tensors)``: the penalty sum_i ||t_i||^2 with torch's multi-tensor
  kernels (one norm pass forward, one scaled copy backward), differentiable once.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from flash_hog_b200 import _capi


def _contig(t):
    return t if t.is_contiguous() else t.contiguous()


class _LayerNormBwd(torch.autograd.Function):
    """(dx, dw, db) of LayerNorm from (x, w, mean, rstd, dy); its backward is the double backward."""

    @staticmethod
    def forward(ctx, x, w, mean, rstd, dy):
        dy = _contig(dy.float())
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        _capi.layernorm_bwd(x, w, mean, rstd, dy, dx, dw, db)
        ctx.save_for_backward(x, w, mean, rstd, dy)
        return dx, dw, db

    @staticmethod
    def backward(ctx, gdx, gdw, gdb):
        x, w, mean, rstd, dy = ctx.saved_tensors
        if any(ctx.needs_input_grad) and torch.is_grad_enabled():
            raise NotImplementedError("third-order derivatives of the fused LayerNorm are not supported")
        gx, gw, gdy = torch.empty_like(x), torch.empty_like(w), torch.empty_like(dy)
        _capi.layernorm_bwd_bwd(x, w, mean, rstd, dy, None if gdx is None else _contig(gdx.float()),
                                None if gdw is None else _contig(gdw.float()),
                                None if gdb is None else _contig(gdb.float()), gx, gw, gdy)
        return gx, gw, None, None, gdy


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, mean, rstd = torch.empty_like(x), x.new_empty(x.shape[:-1]), x.new_empty(x.shape[:-1])
        _capi.layernorm_fwd(x, w, b, eps, y, mean, rstd)
        ctx.save_for_backward(x, w, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        dx, dw, db = _LayerNormBwd.apply(x, w, mean, rstd, dy)
        return dx, dw, db, None


def layer_norm(x, weight, bias, eps: float = 1e-5):
    """LayerNorm over the last dimension in fp32 (fused kernels, differentiable twice)."""
    cast = lambda t: _contig(t.float())
    with torch.autocast(device_type="cuda", enabled=False):
        return _LayerNorm.apply(cast(x), cast(weight), cast(bias), float(eps))


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same parameters and state dict) on the fused kernels."""

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class _GeluBwd(torch.autograd.Function):
    """dh gelu'(a); its backward is the double backward (one kernel for both cotangents)."""

    @staticmethod
    def forward(ctx, a, dh):
        ctx.dh_dtype = dh.dtype
        dh = _contig(dh.to(a.dtype))
        da = torch.empty_like(a)
        _capi.gelu(1, a, dh, None, da, None)
        ctx.save_for_backward(a, dh)
        return da

    @staticmethod
    def backward(ctx, c):
        a, dh = ctx.saved_tensors
        if any(ctx.needs_input_grad) and torch.is_grad_enabled():
            raise NotImplementedError("third-order derivatives of the fused GELU are not supported")
        c = _contig(c.to(a.dtype))
        gdh, ga = torch.empty_like(a), torch.empty_like(a)
        _capi.gelu(2, a, dh, c, gdh, ga)
        return ga, gdh.to(ctx.dh_dtype)


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a):
        h = torch.empty_like(a)
        _capi.gelu(0, a, None, None, h, None)
        ctx.save_for_backward(a)
        return h

    @staticmethod
    def backward(ctx, dh):
        (a,) = ctx.saved_tensors
        return _GeluBwd.apply(a, dh)


def gelu(x):
    """Exact GELU in the input dtype (fp32 or bf16), differentiable twice on the fused kernels."""
    return _Gelu.apply(_contig(x))


class _CrossEntropyBwd(torch.autograd.Function):
    """dz = g (softmax(z) - onehot(t)) / rows; its backward is the double backward."""

    @staticmethod
    def forward(ctx, z, t, lse, g):
        g32 = _contig(g.detach().float().reshape(1))
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        _capi.xent_bwd(z, t, lse, g32, 1.0 / z.shape[0], dz)
        ctx.save_for_backward(z, t, lse, g32)
        ctx.g_shape, ctx.g_dtype = g.shape, g.dtype
        return dz

    @staticmethod
    def backward(ctx, u):
        z, t, lse, g32 = ctx.saved_tensors
        if any(ctx.needs_input_grad) and torch.is_grad_enabled():
            raise NotImplementedError("third-order derivatives of the fused cross entropy are not supported")
        u = _contig(u.to(z.dtype))
        gz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        gg = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
        _capi.xent_bwd_bwd(z, t, lse, g32, 1.0 / z.shape[0], u, gz, gg)
        return gz, None, None, gg.sum().to(ctx.g_dtype).reshape(ctx.g_shape)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, t):
        lse = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
        loss = torch.empty_like(lse)
        _capi.xent_fwd(z, t, lse, loss)
        ctx.save_for_backward(z, t, lse)
        return loss.mean()

    @staticmethod
    def backward(ctx, g):
        z, t, lse = ctx.saved_tensors
        return _CrossEntropyBwd.apply(z, t, lse, g), None


def cross_entropy(logits, targets):
    """Mean cross entropy of (rows, vocab) logits against int64 targets, differentiable
    twice on the fused kernels (fp32 result; the logits' gradient in their dtype)."""
    if logits.stride(-1) != 1:
        logits = logits.contiguous()
    return _CrossEntropy.apply(logits, _contig(targets.long()))


def embedding(tokens, weight, scale: float = 1.0, padding_idx: int | None = None):
    """``scale * weight[tokens]`` for integer ``tokens`` of any shape and a (vocab, dim)
    fp32 or bf16 ``weight``, in the weight's dtype; differentiable to any order.

    The gradient sums equal tokens' rows in fp32 in a fixed order (the same result every
    run) and is zero for ``padding_idx``. A token outside [0, vocab) gives a row of NaN
    and no gradient.
    """
    return _capi.torch_ops().embedding(tokens, weight, scale, padding_idx)


class Embedding(nn.Embedding):
    """``nn.Embedding`` (same parameters and state dict) on the fused kernels, its output
    multiplied by ``scale``. ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are refused."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, scale: float = 1.0,
                 **kwargs):
        super().__init__(num_embeddings, embedding_dim, padding_idx, **kwargs)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = float(scale)

    def forward(self, tokens):
        return embedding(tokens, self.weight, self.scale, self.padding_idx)


def dropout(x, p: float, seed, *, subsequence: int = 0, residual=None):
    """``residual + keep * x / (1 - p)`` (without ``residual``: 0) for fp32 or bf16 tensors,
    differentiable to any order; in ``x``'s dtype, or with a residual in the promoted one.

    The mask is a function of ``seed``, ``subsequence`` and each element's index in ``x``
    alone (Philox4x32-10; ``csrc/dropout.cu``) and is drawn again in the backward passes,
    never stored. ``seed`` is an int64 tensor of one element on ``x``'s device, read when
    the kernel runs, so a captured graph draws a new mask on replay when its value has
    changed; it must keep its value until the backward of the same call has run.
    ``subsequence`` in [0, 2^32) separates calls that share a seed (one per layer). ``p``
    in [0, 1] is rounded to a multiple of 2^-16; at p = 1 everything is dropped.
    """
    return _capi.torch_ops().dropout(x, p, seed, subsequence, residual)


def policy_loss(logits, actions, old_logprobs, advantages, *, ref_logprobs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, normalizer: float | None = None):
    """Clipped policy loss with a KL term over (rows, vocab) logits (fp32 or bf16; fp32
    result), differentiable twice by the logits. Returns ``(loss, logprobs)``.

    Per row, with lp the log probability of ``actions`` under the logits and
    rho = exp(lp - old_logprobs): -min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) +
    kl_coef (exp(ref - lp) - (ref - lp) - 1). ``loss`` is the sum of weights * row loss over
    ``normalizer`` (default: the sum of the weights; 0 where that is 0). Rows of weight 0
    (prompt, padding) are not read: no loss and no gradient whatever they hold.
    ``weights`` (default: all 1) may be a boolean mask. Every input but the logits is a
    constant. ``logprobs`` (fp32, detached) are the lp, 0 in rows of weight 0.
    An action outside [0, vocab) in a weighted row gives NaN.

    The per-row inputs, the clip bounds and ``kl_coef`` are taken in fp32, 64-bit ones
    rounded to it. The exponentials and their sum are fp32: a log probability is accurate
    to about 1e-5, and a ratio closer than that to a clip border may be counted on either
    side of it.
    """
    return _capi.torch_ops().policy_loss(logits, actions, old_logprobs, advantages, ref_logprobs, weights, clip_low,
                                         clip_high, kl_coef, normalizer)


class _SumOfSquares(torch.autograd.Function):
    """sum_i ||t_i||^2 over a list of tensors with multi-tensor kernels: one pass for the
    norms forward, one scaled copy of every tensor backward (instead of a square, a
    reduction and their gradients per tensor)."""

    @staticmethod
    def forward(ctx, *ts):
        ctx.save_for_backward(*ts)
        return torch.stack(torch._foreach_norm(list(ts), 2)).float().square().sum()

    @staticmethod
    def backward(ctx, g):
        ts = ctx.saved_tensors
        return tuple(torch._foreach_mul(list(ts), 2.0 * g))


def sum_of_squares(tensors):
    """sum_i ||t_i||^2 (fp32), differentiable once (the penalty term of the step)."""
    return _SumOfSquares.apply(*tensors)
