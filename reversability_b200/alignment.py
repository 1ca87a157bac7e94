"""Post-training losses on token log-probabilities, with the logits' gradients
(csrc/token_loss.cu): what a preference- or reward-tuning step computes between
the model's logits and its reversible backward.

    token_logprobs          log-probabilities (and entropies) of given tokens
    policy_loss             clipped policy loss with KL and entropy terms
    preference_loss         paired preference loss (sigmoid, hinge, squared)
    *_and_grad              the same with the gradient in the call, for explicit
                            hidden.backward(...) training steps

logits are CUDA fp32, bf16 or fp16 [..., vocab] with evenly strided rows; all
statistics are fp32. Tokens labelled `ignore_index` are not read, contribute
nothing and get zero gradient rows. Labels are the targets of the same position
(no shift inside). Only the logits are differentiated: old, reference and
advantage inputs are constants, and asking for their gradients raises.

The autograd forms save the logits and two numbers a row and form the gradient
in the backward, with the upstream factor applied before the one rounding, so a
loss scaler works with fp16 logits; the *_and_grad forms may write the gradient over
them (`out=logits`), and that of the policy loss reads them once instead of
twice (a preference pair's factor is known only after all its rows are read).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import functional as fn
from .optimized import _accumulate_grad, amp_context, compute_dtype, hidden_states


class PolicyLoss(NamedTuple):
    """loss: scalar; logprobs, kl, entropy: per token (kl without a reference and entropy without a request are
    None); clip_fraction: weighted share of tokens whose clamped branch is taken."""
    loss: torch.Tensor
    logprobs: torch.Tensor
    kl: torch.Tensor | None
    entropy: torch.Tensor | None
    clip_fraction: torch.Tensor


class PreferenceLoss(NamedTuple):
    """loss: scalar; rewards [2 * pairs]: beta times each sequence's log ratio, chosen first; logprobs: per token."""
    loss: torch.Tensor
    rewards: torch.Tensor
    logprobs: torch.Tensor


def _check_rows(temperature: float, ignore_index: int) -> None:
    if not 1e-30 <= temperature <= 1e30:  # its reciprocal is an fp32 number
        raise ValueError("temperature must be finite and positive")
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise ValueError("ignore_index must fit 32 bits")


def _check_constants(**tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is a constant of the loss; detach it")


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, temperature, ignore_index, entropy):
        lp, h, stats = fn.token_logprob_fwd(logits, labels, temperature, ignore_index, entropy)
        ctx.save_for_backward(logits, labels, stats, h)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.set_materialize_grads(False)
        return (lp, h) if entropy else lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_h=None):
        logits, labels, stats, h = ctx.saved_tensors
        if g_lp is None and g_h is None:
            return None, None, None, None, None
        g_lp = torch.zeros(labels.shape, device=logits.device) if g_lp is None else g_lp.contiguous()
        g_h = None if g_h is None else g_h.contiguous()
        d = fn.token_logprob_bwd(logits, labels, stats, g_lp, None if g_h is None else h, g_h, ctx.temperature,
                                 ctx.ignore_index)
        return d, None, None, None, None


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                   entropy: bool = False):
    """ln softmax(logits / temperature) at labels, fp32 in the shape of labels (0 at ignore_index); with `entropy`
    the pair (log-probabilities, entropies of the rows). Differentiable with respect to the logits."""
    _check_rows(temperature, ignore_index)
    fn.require_cuda(logits, labels, what="token log-probabilities")
    if not (logits.requires_grad and torch.is_grad_enabled()):
        lp, h, _ = fn.token_logprob_fwd(logits, labels, temperature, ignore_index, entropy, want_stats=False)
        return (lp, h) if entropy else lp
    return _TokenLogprobs.apply(logits, labels, float(temperature), int(ignore_index), bool(entropy))


class _Policy(torch.autograd.Function):
    """The loss alone, formed before: what carries no gradient stays out of autograd, which costs it time for each tensor."""

    @staticmethod
    def forward(ctx, logits, made):
        loss, actions, pairs, h, ctx.temperature, ctx.ignore_index = made
        ctx.save_for_backward(logits, actions, pairs, h)
        return loss.data  # no view of the metrics: they, and the loss itself, may be changed in place

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, actions, pairs, h = ctx.saved_tensors
        coef = pairs.data_ptr() + 2 * pairs.numel()  # behind the statistics: half of the array's bytes
        d = fn.token_logprob_bwd_at(logits, actions, pairs.data_ptr(), coef, 2, h, None if h is None else coef + 4,
                                    ctx.temperature, ctx.ignore_index, g.float())
        return d, None


def _policy_args(ref_logprobs, weights, clip_low, clip_high, kl_coef, entropy_coef, temperature, ignore_index, entropy,
                 denominator):
    _check_rows(temperature, ignore_index)
    if not (0.0 <= clip_low and 0.0 <= clip_high):
        raise ValueError("clip_low and clip_high must not be negative")
    if kl_coef != 0 and ref_logprobs is None:
        raise ValueError("kl_coef needs ref_logprobs")
    return dict(ref_logprobs=ref_logprobs, weights=weights, clip_low=float(clip_low), clip_high=float(clip_high),
                kl_coef=float(kl_coef), entropy_coef=float(entropy_coef), temperature=float(temperature),
                ignore_index=int(ignore_index), entropy=bool(entropy), denominator=denominator)


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: torch.Tensor | None = None, weights: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                ignore_index: int = -100, entropy: bool = False,
                denominator: torch.Tensor | None = None) -> PolicyLoss:
    """Clipped policy loss over the tokens `actions` [...] of logits [..., V]:

        ratio = exp(lp - old),  kl = exp(ref - lp) - 1 - (ref - lp)
        l     = -min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef kl - entropy_coef H
        loss  = sum w l / denominator

    advantages: one a token, or one a sequence (the leading dimensions of actions). weights: one a token (default
    1); the denominator is the sum of the weights over the tokens that count unless a device scalar is given (a
    token count over several microbatches, say). `entropy` returns H even without a bonus."""
    args = _policy_args(ref_logprobs, weights, clip_low, clip_high, kl_coef, entropy_coef, temperature, ignore_index,
                        entropy, denominator)
    _check_constants(old_logprobs=old_logprobs, advantages=advantages, ref_logprobs=ref_logprobs, weights=weights,
                     denominator=denominator)
    fn.require_cuda(logits, actions, old_logprobs, advantages, what="the policy loss")
    if not (logits.requires_grad and torch.is_grad_enabled()):
        loss, clip, lp, kl, h, _, _ = fn.policy_loss(logits, actions, old_logprobs, advantages, want_grad=False, **args)
        return PolicyLoss(loss, lp, kl, h, clip)
    loss, clip, lp, kl, h, _, pairs = fn.policy_loss(logits, actions, old_logprobs, advantages, want_grad=False,
                                                     want_coef=True, **args)
    loss = _Policy.apply(logits, (loss, actions, pairs, h if args["entropy_coef"] != 0 else None, args["temperature"],
                                  args["ignore_index"]))
    return PolicyLoss(loss, lp, kl, h, clip)


def _scale(grad_scale):
    return (1.0, grad_scale) if isinstance(grad_scale, torch.Tensor) else (float(grad_scale), None)


def policy_loss_and_grad(logits: torch.Tensor, actions: torch.Tensor, old_logprobs: torch.Tensor,
                         advantages: torch.Tensor, *, ref_logprobs: torch.Tensor | None = None,
                         weights: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                         kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                         ignore_index: int = -100, entropy: bool = False, denominator: torch.Tensor | None = None,
                         grad_scale: float | torch.Tensor = 1.0, out: torch.Tensor | None = None):
    """policy_loss outside autograd with its gradient: (PolicyLoss, d (grad_scale * loss) / d logits) in one pass
    over the logits. grad_scale: a number or a device scalar. `out` receives the gradient and may be the logits."""
    args = _policy_args(ref_logprobs, weights, clip_low, clip_high, kl_coef, entropy_coef, temperature, ignore_index,
                        entropy, denominator)
    fn.require_cuda(logits, actions, old_logprobs, advantages, what="the policy loss")
    scale, scale_dev = _scale(grad_scale)
    loss, clip, lp, kl, h, d, _ = fn.policy_loss(logits, actions, old_logprobs, advantages, grad_scale=scale,
                                                 grad_scale_dev=scale_dev, out=out, **args)
    return PolicyLoss(loss, lp, kl, h, clip), d


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, made):
        loss, labels, rows, ctx.temperature, ctx.ignore_index = made
        ctx.save_for_backward(logits, labels, rows)
        return loss.data

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, labels, rows = ctx.saved_tensors
        coef = rows.data_ptr() + 8 * (rows.numel() // 3)  # behind the statistics
        d = fn.token_logprob_bwd_at(logits, labels, rows.data_ptr(), coef, 1, None, None, ctx.temperature,
                                    ctx.ignore_index, g.float())
        return d, None


def _preference_args(kind, beta, label_smoothing, average, temperature, ignore_index):
    _check_rows(temperature, ignore_index)
    if not (math.isfinite(beta) and beta > 0):
        raise ValueError("beta must be finite and positive")
    if not 0.0 <= label_smoothing < 0.5:
        raise ValueError("label_smoothing must be in [0, 0.5)")
    if label_smoothing and kind != "sigmoid":
        raise ValueError("label_smoothing belongs to the sigmoid loss")
    return dict(kind=kind, beta=float(beta), label_smoothing=float(label_smoothing), average=bool(average),
                temperature=float(temperature), ignore_index=int(ignore_index))


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logprobs: torch.Tensor | None, *,
                    kind: str = "sigmoid", beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False,
                    temperature: float = 1.0, ignore_index: int = -100) -> PreferenceLoss:
    """Paired preference loss over logits [2 * pairs, length, V], the chosen sequences of all pairs first, then the
    rejected ones in the same order; labels likewise, with ignore_index on prompt and padding. ref_logprobs: the
    reference model's log-probabilities of the same tokens, or None for a loss without a reference. Per sequence
    gap = sum (lp - ref) over its labelled tokens (their mean with `average`), and with u = beta (gap_chosen -
    gap_rejected): 'sigmoid' -(1 - e) ln sigma(u) - e ln sigma(-u) with e = label_smoothing, 'hinge' max(0, 1 - u),
    'squared' (gap_chosen - gap_rejected - 1 / (2 beta))^2; the loss is the mean over the pairs."""
    args = _preference_args(kind, beta, label_smoothing, average, temperature, ignore_index)
    _check_constants(ref_logprobs=ref_logprobs)
    fn.require_cuda(logits, labels, ref_logprobs, what="the preference loss")
    if not (logits.requires_grad and torch.is_grad_enabled()):
        loss, lp, rewards, _, _ = fn.preference_loss(logits, labels, ref_logprobs, want_grad=False, **args)
        return PreferenceLoss(loss, rewards, lp)
    loss, lp, rewards, _, rows = fn.preference_loss(logits, labels, ref_logprobs, want_grad=False, **args)
    loss = _Preference.apply(logits, (loss, labels, rows, args["temperature"], args["ignore_index"]))
    return PreferenceLoss(loss, rewards, lp)


def preference_loss_and_grad(logits: torch.Tensor, labels: torch.Tensor, ref_logprobs: torch.Tensor | None, *,
                             kind: str = "sigmoid", beta: float = 0.1, label_smoothing: float = 0.0,
                             average: bool = False, temperature: float = 1.0, ignore_index: int = -100,
                             grad_scale: float | torch.Tensor = 1.0, out: torch.Tensor | None = None):
    """preference_loss outside autograd with its gradient: (PreferenceLoss, d (grad_scale * loss) / d logits).
    `out` receives the gradient and may be the logits."""
    args = _preference_args(kind, beta, label_smoothing, average, temperature, ignore_index)
    fn.require_cuda(logits, labels, ref_logprobs, what="the preference loss")
    scale, scale_dev = _scale(grad_scale)
    loss, lp, rewards, d, _ = fn.preference_loss(logits, labels, ref_logprobs, grad_scale=scale,
                                                    grad_scale_dev=scale_dev, out=out, **args)
    return PreferenceLoss(loss, rewards, lp), d


def backward_through_head(model, ids: torch.Tensor, loss_and_grad, precision: str = "bf16", reuse: bool = False):
    """One forward and backward of a language model around a loss on its logits, without autograd over the
    vocabulary: hidden states, the head GEMM into one logits buffer, `loss_and_grad(logits, out)` -> (loss, d logits)
    writing the gradient over the logits (the *_and_grad functions above), then the head's two gradient GEMMs and
    the model's backward (the reversible reconstruction for a ReversibleLM). ids [B, T]; the logits given to the
    loss are [B, T, V] in the compute type. Adds to the parameters' .grad and returns the loss."""
    with amp_context(ids.device, precision):
        hidden = hidden_states(model, ids, reuse)
    weight = model.lm_head.weight
    compute = compute_dtype(ids.device, precision, weight.dtype)
    x = hidden.detach().reshape(-1, hidden.shape[-1]).to(compute).contiguous()
    w = weight.detach().to(compute).contiguous()
    logits = fn.head_logits_buffer(x.shape[0], w.shape[0], x.device, compute)
    fn.linear_fwd(x, w, out=logits)
    logits = logits.unflatten(0, ids.shape)
    loss, d = loss_and_grad(logits, logits)
    d = d.flatten(0, 1)
    dx = fn.linear_dgrad(d, w)
    _accumulate_grad(weight, fn.linear_wgrad(d, x))
    del logits, d
    with amp_context(ids.device, precision):
        hidden.backward(dx.view(hidden.shape).to(hidden.dtype))
    return loss
