"""autograd.Functions over librevk for the module-level API (nn.Linear,
scaled-dot-product attention, RMSNorm and SwiGLU of the reference model).

Autocast: librevk kernels are not ATen ops, so autocast cannot cast around
them. `linear` and `attention` apply the CUDA autocast policy explicitly (the
same policy the reference relies on, train_baseline.py:205-207): under an
enabled autocast context their inputs are cast to the autocast dtype with
ordinary (differentiable) torch casts, so gradients flow back through the
casts exactly as they do for F.linear / F.scaled_dot_product_attention.
RMSNorm and SwiGLU run in their input dtype, as nn.RMSNorm and silu*value do.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import functional as fn


def autocast_dtype(device_type: str = "cuda") -> torch.dtype | None:
    if torch.is_autocast_enabled(device_type):
        return torch.get_autocast_dtype(device_type)
    return None


class LinearFn(torch.autograd.Function):
    """y = x @ w.T with x, w in one dtype (bf16/f16 on tensor cores, fp32 on CUDA cores)."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return fn.linear_fwd(x, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w = ctx.saved_tensors
        gy = gy.to(x.dtype).contiguous()
        gx = fn.linear_dgrad(gy, w) if ctx.needs_input_grad[0] else None
        gw = fn.linear_wgrad(gy, x).to(w.dtype) if ctx.needs_input_grad[1] else None
        return gx, gw


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """nn.Linear forward on librevk GEMMs (replaces F.linear at model.py:37,45,55-56)."""
    fn.require_cuda(x, w)
    low = autocast_dtype(x.device.type)
    if low is not None:
        with torch.autocast(x.device.type, enabled=False):
            x, w = x.to(low), w.to(low)
            bias = bias.to(low) if bias is not None else None
    elif x.dtype != w.dtype:
        raise ValueError(f"linear: input {x.dtype} and weight {w.dtype} differ outside autocast")
    y = LinearFn.apply(x.contiguous(), w.contiguous())
    return y if bias is None else y + bias


class AttentionFn(torch.autograd.Function):
    """Causal attention over packed qkv [B, T, 3D] -> [B, T, D]."""

    @staticmethod
    def forward(ctx, qkv, n_heads):
        o, lse = fn.attention_fwd(qkv, n_heads)
        ctx.n_heads = n_heads
        ctx.save_for_backward(qkv, o, lse)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        qkv, o, lse = ctx.saved_tensors
        return fn.attention_bwd(qkv, o, go.contiguous(), lse, ctx.n_heads), None


def attention(qkv: torch.Tensor, n_heads: int) -> torch.Tensor:
    """F.scaled_dot_product_attention(q, k, v, is_causal=True) on the packed qkv projection."""
    fn.require_cuda(qkv)
    low = autocast_dtype(qkv.device.type)
    if low is not None and qkv.dtype != low:
        with torch.autocast(qkv.device.type, enabled=False):
            qkv = qkv.to(low)
    return AttentionFn.apply(qkv.contiguous(), n_heads)


class RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        y, rstd = fn.rmsnorm_fwd(x, w, eps)
        ctx.save_for_backward(x, w, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w, rstd = ctx.saved_tensors
        dx, dw = fn.rmsnorm_bwd(x, w, rstd, gy.contiguous())
        return dx, dw, None


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float | None) -> torch.Tensor:
    """nn.RMSNorm forward; eps None means finfo(x.dtype).eps (kernels_v3.py:78-80)."""
    fn.require_cuda(x, w)
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    return RMSNormFn.apply(x.contiguous(), w, float(eps))


def once(backward):
    """once_differentiable, whose context costs some microseconds, only where a graph of the backward is recorded."""
    recorded = once_differentiable(backward)

    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def differentiated(x: torch.Tensor, a: torch.Tensor | None = None, b: torch.Tensor | None = None) -> bool:
    """Whether a derivative of these is to be had: one of them requires a gradient, or carries a tangent of forward-mode
    differentiation (which a Function refuses; past it, the result would have lost the tangent without a word)."""
    if torch.is_grad_enabled() and (x.requires_grad or (a is not None and a.requires_grad) or
                                    (b is not None and b.requires_grad)):
        return True
    if forward_ad._current_level < 0:  # no level is open (asking each tensor takes 0.6 us)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, a, b))


class LayerNormFn(torch.autograd.Function):
    """Keeps the input and two numbers a row."""

    @staticmethod
    def forward(ctx, x, w, b, eps, out_dtype):
        y, stats, xr, weight = fn.layernorm_fwd_kept(x, w, b, eps, out_dtype)
        ctx.save_for_backward(xr, weight, stats)
        ctx.param_dtype = torch.float32 if w is None and b is None else (b if w is None else w).dtype
        return y

    @staticmethod
    @once
    def backward(ctx, gy):
        xr, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = fn.layernorm_bwd_kept(xr, weight, stats, gy, ctx.param_dtype, need[0], need[1], need[2])
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """F.layer_norm over the last dimension (at most 16384 wide, 16377 if the width is no multiple of 8): statistics in
    fp32, weight and bias (each may be None) in fp32 or x's type, the output in x's type unless out_dtype says otherwise
    (any type for fp32 x, fp32 for 16-bit x). Rows of unit stride, an even distance apart, are read where they lie if they
    start as far from 16-byte boundaries as rows side by side would (x[..., :width] of wider rows, both widths multiples of
    8, do); others are copied. Like the other norms it runs in its input's type under autocast. The gradients of weight
    and bias are sums in a fixed order."""
    if differentiated(x, weight, bias):
        return LayerNormFn.apply(x, weight, bias, float(eps), out_dtype)
    return fn.layernorm_fwd_kept(x, weight, bias, float(eps), out_dtype, False)[0]


class DropoutFn(torch.autograd.Function):
    """Keeps no mask: the backward generates it anew from (seed, offset)."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        y = fn.dropout(x, p, seed, offset, residual)
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
            seed = None
        ctx.args = p, seed, int(offset), x.dtype
        return y

    @staticmethod
    @once
    def backward(ctx, gy):
        p, seed, offset, dtype = ctx.args
        need = ctx.needs_input_grad
        dx = None
        if need[0]:
            dx = fn.dropout_checked(gy, p, ctx.saved_tensors[0] if seed is None else int(seed), offset, None, dtype)
        return dx, gy if need[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, *, offset: int = 0,
            residual: torch.Tensor | None = None, training: bool = True) -> torch.Tensor:
    """Dropout whose mask is a function of (seed, offset) and the element's position and is never stored: a
    recompute, an inverse or a backward with the same two numbers drops the same elements. Each is dropped with
    probability round(p 2^32) / 2^32, the others scaled by 1 / (1 - p); with `residual` (x's shape, its type or fp32)
    the result is added to it, in its type. Give every call of a step its own offset and every step its own seed (or
    the other way round). seed may be an int64 scalar on the device, which a captured step's replays read anew;
    change it in place only after the backward. What is dropped is not used: NaN there does not spread."""
    if not training:
        p = 0.0
    if differentiated(x, residual):
        return DropoutFn.apply(x, residual, float(p), seed, offset)
    return fn.dropout(x, float(p), seed, offset, residual)


class SwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u):
        ctx.save_for_backward(u)
        return fn.swiglu_fwd(u)

    @staticmethod
    @once_differentiable
    def backward(ctx, gh):
        u, = ctx.saved_tensors
        return fn.swiglu_bwd(u, gh.contiguous())


def swiglu(u: torch.Tensor) -> torch.Tensor:
    """silu(gate) * value over u = [gate | value] (model.py:55-56)."""
    fn.require_cuda(u)
    return SwiGLUFn.apply(u.contiguous())


class LinearCrossEntropyFn(torch.autograd.Function):
    """Keeps the inputs and one number a row; the backward forms the logits again, a piece of the vocabulary at a time."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        loss, kept = fn.linear_ce_fwd(hidden, weight, labels, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, kept)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once
    def backward(ctx, g):
        hidden, weight, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw = fn.linear_ce_bwd(hidden, weight, kept, g, ctx.reduction, need[0], need[1])
        return dx, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """F.cross_entropy(F.linear(hidden, weight), labels) without the logits (model.py:104, train_baseline.py:262): hidden
    [..., d], weight [V, d] of one type, int64 labels [...]; the loss in fp32, 'mean' over the labels that count (0 if
    none does), 'sum', or 'none' (one a label). What lies in a row labelled ignore_index does not spread and its gradients
    are zero; in 16 bits such rows are not read and cost nothing. A label outside [0, V) sets the library's device status
    and counts as ignored. The gradients come in the inputs' types, rounded once from fp32 sums over 16-bit softmax terms
    (fp16: scaled inside, so a mean over many rows does not underflow before the gradients themselves do; with 'none' one
    power of two serves all rows, and a row whose gradient is 2^-k of the largest keeps terms down to 2^(k - 37)). fp32
    inputs stay fp32 throughout, in pieces of the rows. Under autocast both inputs are cast as F.linear's are."""
    low = autocast_dtype("cuda")
    if low is not None:
        with torch.autocast("cuda", enabled=False):
            hidden, weight = hidden.to(low), weight.to(low)
    if differentiated(hidden, weight):
        return LinearCrossEntropyFn.apply(hidden, weight, labels, int(ignore_index), reduction)
    return fn.linear_ce_fwd(hidden, weight, labels, int(ignore_index), reduction)[0]
