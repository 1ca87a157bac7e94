"""Tensor-level wrappers over librevk: argument checks, output allocation and
the current-stream launch. These are the only functions that touch the C ABI
directly; autograd Functions and the fused engine build on them.

All inputs must be CUDA tensors; a CPU tensor raises ValueError mentioning
CUDA (the reference's error convention, kernels.py:59-60, kernels_v3.py:54-57).
"""
from __future__ import annotations

import functools

import torch

from . import _lib

_TC_DTYPES = (torch.bfloat16, torch.float16)


def require_cuda(*tensors: torch.Tensor, what: str = "librevk kernels") -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError(f"{what} require CUDA tensors; no CPU fallback exists")


def _row_major_2d(t: torch.Tensor, name: str) -> tuple[torch.Tensor, int]:
    """Returns (t viewed as 2-D, leading dimension); the last dim must be unit-stride."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() > 2:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        t = t.reshape(-1, t.shape[-1])
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have a unit-stride last dimension")
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


# ------------------------------------------------------------------ RMSNorm
def rmsnorm_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float, out_dtype: torch.dtype | None = None,
                want_rstd: bool = True, out: torch.Tensor | None = None):
    """y = x * rsqrt(mean(x^2) + eps) * weight over the last dim; returns (y, rstd)."""
    require_cuda(x, weight)
    if weight.dtype != torch.float32 or weight.dim() != 1 or weight.numel() != x.shape[-1]:
        raise ValueError("RMSNorm weight must be fp32 [width] matching the input width")
    x2, ldx = _row_major_2d(x, "x")
    rows, width = x2.shape
    out_dtype = out_dtype or x.dtype
    y = out if out is not None else torch.empty(x.shape, device=x.device, dtype=out_dtype)
    y2, ldy = _row_major_2d(y, "out")
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if want_rstd else None
    _lib.call("rk_rmsnorm_fwd", x2.data_ptr(), _lib.code(x.dtype), ldx, weight.contiguous().data_ptr(),
              y2.data_ptr(), _lib.code(out_dtype), ldy, _lib.ptr(rstd), rows, width, float(eps), _lib.stream_ptr())
    return y, rstd


def rmsnorm_bwd(x: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, dy: torch.Tensor,
                dx_dtype: torch.dtype | None = None, dw: torch.Tensor | None = None, accumulate_dw: bool = False):
    """Returns (dx, dw) for y = rmsnorm(x) * weight; dw is fp32 [width]."""
    require_cuda(x, weight, rstd, dy)
    x2, ldx = _row_major_2d(x, "x")
    g2, ldg = _row_major_2d(dy, "dy")
    rows, width = x2.shape
    dx = torch.empty(x.shape, device=x.device, dtype=dx_dtype or x.dtype)
    dx2, lddx = _row_major_2d(dx, "dx")
    if dw is None:
        dw = torch.empty(width, device=x.device, dtype=torch.float32)
        accumulate_dw = False
    ws_bytes = _lib.lib().rk_rmsnorm_bwd_workspace(rows, width)
    ws = torch.empty(max(ws_bytes // 4, 1), device=x.device, dtype=torch.float32)
    _lib.call("rk_rmsnorm_bwd", x2.data_ptr(), _lib.code(x.dtype), ldx, weight.contiguous().data_ptr(),
              rstd.data_ptr(), g2.data_ptr(), _lib.code(dy.dtype), ldg, dx2.data_ptr(), _lib.code(dx.dtype), lddx,
              dw.data_ptr(), int(accumulate_dw), ws.data_ptr(), ws_bytes, rows, width, _lib.stream_ptr())
    return dx, dw


# ------------------------------------------------------------------ layer norm
def _on_current_device(t: torch.Tensor, name: str, *others: torch.Tensor | None) -> None:
    index = t.get_device()
    if index != torch.cuda.current_device():
        raise ValueError(f"{name} must be on the current CUDA device")
    for o in others:
        if o is not None and o.get_device() != index:
            raise ValueError(f"all tensors must be on {name}'s device")


def _new(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous uninitialised tensor of t's shape (the cheapest call for it: they are most of a small pass's time)."""
    if t.dtype is dtype and t.is_contiguous():
        return torch.empty_like(t)
    return t.new_empty(t.shape, dtype=dtype)


def even_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """(t or a contiguous copy of it, rows, width, row stride): rows of unit-stride elements an even distance apart
    are taken as they lie, anything else is copied."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // width if width else 0, width, width
    rows, ld = 1, None
    even = width == 1 or t.stride(-1) == 1
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size != 1:
            if ld is None:
                ld = stride
            even = even and stride == ld * rows
            rows *= size
    if even and (ld is None or ld >= width):
        return t, rows, width, width if ld is None else ld
    return t.contiguous(), rows, width, width


def _norm_rows(t: torch.Tensor, per: int) -> tuple[torch.Tensor, int, int, int]:
    """even_rows of a tensor whose rows start as far from multiples of `per` elements as those of a new contiguous one
    (what the layer norm's vectors need); others are copied."""
    rows_of = even_rows(t)
    r, rows, width, ld = rows_of
    if r.data_ptr() // t.element_size() % per == 0 and (rows <= 1 or (ld - width) % per == 0):
        return rows_of
    return t.clone(memory_format=torch.contiguous_format), rows, width, width


def _norm_param(x: torch.Tensor, t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != x.shape[-1] or (t.dtype is not torch.float32 and t.dtype != x.dtype):
        raise ValueError(f"layer norm {name} must be [width] in fp32 or the input's type")
    return t if t.is_contiguous() else t.contiguous()


def _norm_params(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None):
    """(weight, bias, dtype code): contiguous [width] vectors of one type, fp32 or x's."""
    if weight is not None:
        weight = _norm_param(x, weight, "weight")
    if bias is not None:
        bias = _norm_param(x, bias, "bias")
        if weight is not None and bias.dtype != weight.dtype:
            raise ValueError("layer norm weight and bias must share a type")
    one = bias if weight is None else weight
    return weight, bias, 0 if one is None else _lib.code(one.dtype)


def _fast_rows(t: torch.Tensor, per: int) -> tuple[torch.Tensor, int, int, int]:
    if t.is_contiguous() and t.data_ptr() % 32 == 0:
        width = t.size(-1)
        if width:
            return t, t.numel() // width, width, width
    return _norm_rows(t, per)


def layernorm_fwd_kept(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
                       out_dtype: torch.dtype | None = None, want_stats: bool = True):
    """layernorm_fwd that also returns what its backward can use again: (y, stats, x in rows it can read, weight)."""
    require_cuda(x, weight, bias, what="layer norm kernels")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("layer norm needs a non-empty last dimension")
    if out_dtype is None:
        out_dtype = x.dtype
    elif x.dtype is not torch.float32 and out_dtype not in (x.dtype, torch.float32):
        raise ValueError("layer norm of 16-bit inputs gives their type or fp32")
    _on_current_device(x, "the input", weight, bias)
    weight, bias, pcode = _norm_params(x, weight, bias)
    xr, rows, width, ld = _fast_rows(x, 16 // x.element_size())
    y = _new(x, out_dtype)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    _lib.call("rk_layernorm_fwd", xr.data_ptr(), _lib.code(x.dtype), ld, _lib.ptr(weight), _lib.ptr(bias), pcode,
              y.data_ptr(), _lib.code(out_dtype), width, _lib.ptr(stats), rows, width, eps, _lib.stream_ptr())
    return y, stats, xr, weight


def layernorm_fwd(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
                  out_dtype: torch.dtype | None = None, want_stats: bool = True):
    """y = (x - mean) * rsqrt(var + eps) * weight + bias over the last dim; returns (y, stats [rows, 2] or None)."""
    return layernorm_fwd_kept(x, weight, bias, float(eps), out_dtype, want_stats)[:2]


@functools.lru_cache(maxsize=64)
def _layernorm_workspace(rows: int, width: int) -> int:
    return _lib.lib().rk_layernorm_bwd_workspace(rows, width)


def layernorm_bwd_kept(x: torch.Tensor, weight: torch.Tensor | None, stats: torch.Tensor, dy: torch.Tensor,
                       param_dtype: torch.dtype, want_dx: bool, want_dw: bool, want_db: bool):
    """layernorm_bwd of what layernorm_fwd_kept returned. Rows, strides, sizes and devices are looked at anew: hooks on saved
    tensors need not hand back the strides that the forward saw."""
    per, device = 16 // x.element_size(), dy.get_device()
    xr, rows, width, ldx = _fast_rows(x, per)
    if dy.numel() != rows * width or stats.numel() != 2 * rows or stats.dtype is not torch.float32 or \
            not stats.is_contiguous() or x.get_device() != device or stats.get_device() != device:
        raise ValueError("layer norm backward takes dy of the input's shape and the forward's stats")
    if weight is not None and (weight.numel() != width or weight.dtype is not param_dtype or not weight.is_contiguous() or
                               weight.get_device() != device):
        raise ValueError("layer norm backward takes the forward's weight")
    dyr, _, _, lddy = _fast_rows(dy, per)
    dx = _new(xr, x.dtype) if want_dx else None
    dw = (x.new_empty(width, dtype=param_dtype) if weight is None else torch.empty_like(weight)) if want_dw else None
    db = (x.new_empty(width, dtype=param_dtype) if weight is None else torch.empty_like(weight)) if want_db else None
    n_ws = _layernorm_workspace(rows, width) if want_dw or want_db else 0
    ws = stats.new_empty(n_ws // 4) if n_ws else None
    _lib.call("rk_layernorm_bwd", xr.data_ptr(), _lib.code(x.dtype), ldx, _lib.ptr(weight), _lib.code(param_dtype),
              stats.data_ptr(), dyr.data_ptr(), _lib.code(dy.dtype), lddy, _lib.ptr(dx), width, _lib.ptr(dw), _lib.ptr(db),
              _lib.ptr(ws), n_ws, rows, width, _lib.stream_ptr())
    return dx, dw, db


def layernorm_bwd(x: torch.Tensor, weight: torch.Tensor | None, stats: torch.Tensor, dy: torch.Tensor,
                  param_dtype: torch.dtype = torch.float32, want_dx: bool = True, want_dw: bool = True,
                  want_db: bool = True):
    """(dx in x's type, dweight, dbias in param_dtype; None where not wanted) of layernorm_fwd."""
    require_cuda(x, weight, stats, dy, what="layer norm kernels")
    _on_current_device(x, "the input", weight, stats, dy)
    weight, _, _ = _norm_params(x, weight, None)
    if weight is not None and weight.dtype != param_dtype:
        raise ValueError("parameter gradients come in the weight's type")
    if dy.shape != x.shape:
        raise ValueError("layer norm backward takes dy of the input's shape and the forward's stats")
    return layernorm_bwd_kept(x, weight, stats, dy, param_dtype, want_dx, want_dw, want_db)


# ------------------------------------------------------------------ dropout
def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, offset: int = 0, residual: torch.Tensor | None = None,
            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """residual + (kept ? x / (1 - p) : 0) with the mask of (seed, offset), a function of the element's position in
    row-major order. seed: a whole number or an int64 device scalar."""
    require_cuda(x, residual, what="dropout kernels")
    if not 0.0 <= p <= 1.0:
        raise ValueError("the dropout probability must be in [0, 1]")
    offset, on_device = int(offset), isinstance(seed, torch.Tensor)
    if not 0 <= offset < 2 ** 64:
        raise ValueError("the dropout offset must fit 64 bits")
    if on_device:
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError("a dropout seed on the device must be one int64 number")
    else:
        seed = int(seed)
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError("the dropout seed must fit 64 bits")
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        raise ValueError("the dropout residual must have the input's shape and its type or fp32")
    _on_current_device(x, "the input", residual, seed if on_device else None)
    out_dtype = out_dtype or (x.dtype if residual is None else residual.dtype)
    if residual is not None and out_dtype != residual.dtype:
        raise ValueError("dropout with a residual gives the residual's type")
    return dropout_checked(x, float(p), seed, offset, residual, out_dtype)


def dropout_checked(x: torch.Tensor, p: float, seed: int | torch.Tensor, offset: int, residual: torch.Tensor | None,
                    out_dtype: torch.dtype) -> torch.Tensor:
    """dropout of arguments that were checked."""
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    on_device = isinstance(seed, torch.Tensor)
    y = _new(x, out_dtype)
    _lib.call("rk_dropout", x.data_ptr(), _lib.code(x.dtype), _lib.ptr(residual), y.data_ptr(), _lib.code(out_dtype),
              x.numel(), p, 0 if on_device else seed & 0xFFFFFFFFFFFFFFFF, seed.data_ptr() if on_device else None, offset,
              _lib.stream_ptr())
    return y


# ------------------------------------------------------------------ SwiGLU
def swiglu_fwd(u: torch.Tensor) -> torch.Tensor:
    require_cuda(u)
    if not u.is_contiguous() or u.shape[-1] % 2:
        raise ValueError("SwiGLU input must be contiguous with an even last dimension")
    width = u.shape[-1] // 2
    rows = u.numel() // u.shape[-1] if u.numel() else 0
    h = torch.empty((*u.shape[:-1], width), device=u.device, dtype=u.dtype)
    _lib.call("rk_swiglu_fwd", u.data_ptr(), h.data_ptr(), _lib.code(u.dtype), rows, width, _lib.stream_ptr())
    return h


def swiglu_bwd(u: torch.Tensor, dh: torch.Tensor) -> torch.Tensor:
    require_cuda(u, dh)
    dh = dh.to(u.dtype).contiguous()
    width = u.shape[-1] // 2
    rows = u.numel() // u.shape[-1] if u.numel() else 0
    du = torch.empty_like(u)
    _lib.call("rk_swiglu_bwd", u.data_ptr(), dh.data_ptr(), du.data_ptr(), _lib.code(u.dtype), rows, width,
              _lib.stream_ptr())
    return du


# ------------------------------------------------------------------ reconstruct
def reconstruct_midpoint(x_next: torch.Tensor, force: torch.Tensor, coeff: float,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """x_prev = x_next - round_force_dtype(coeff * force) (fp32 state)."""
    require_cuda(x_next, force)
    if x_next.dtype != torch.float32 or not x_next.is_contiguous() or not force.is_contiguous():
        raise ValueError("reconstruct expects a contiguous fp32 state and a contiguous force")
    if x_next.numel() != force.numel():
        raise ValueError("state and force sizes differ")
    out = out if out is not None else torch.empty_like(x_next)
    _lib.call("rk_reconstruct_midpoint", x_next.data_ptr(), force.data_ptr(), _lib.code(force.dtype), float(coeff),
              out.data_ptr(), x_next.numel(), _lib.stream_ptr())
    return out


def reconstruct_euler(state: torch.Tensor, sublayer_out: torch.Tensor, out: torch.Tensor | None = None):
    require_cuda(state, sublayer_out)
    if state.dtype != torch.float32 or not state.is_contiguous() or not sublayer_out.is_contiguous():
        raise ValueError("reconstruct expects a contiguous fp32 state and a contiguous sublayer output")
    out = out if out is not None else torch.empty_like(state)
    _lib.call("rk_reconstruct_euler", state.data_ptr(), sublayer_out.data_ptr(), _lib.code(sublayer_out.dtype),
              out.data_ptr(), state.numel(), _lib.stream_ptr())
    return out


# ------------------------------------------------------------------ GEMMs
def _tma_ready(t: torch.Tensor) -> torch.Tensor:
    """Tensor-core operands are read by TMA, which needs 16-byte aligned rows.
    A 2-D bf16/f16 operand whose row stride or base breaks that is staged into
    a zero-padded copy (row stride rounded up to 8 elements); the returned view
    has the original shape, and the padding is never read as data."""
    if t.dtype not in _TC_DTYPES:
        return t
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if (ld * 2) % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    rows, cols = t.shape
    padded = torch.zeros((rows, (cols + 7) // 8 * 8), device=t.device, dtype=t.dtype)
    padded[:, :cols].copy_(t)
    return padded[:, :cols]


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else (t.stride(0) if t.stride(0) >= t.shape[1] else t.shape[1])


def _gemm_dtype(*ts: torch.Tensor) -> int:
    dts = {t.dtype for t in ts}
    if len(dts) != 1:
        raise ValueError(f"GEMM operands must share a dtype, got {dts}")
    return _lib.code(dts.pop())


def linear_fwd(x: torch.Tensor, w: torch.Tensor, out_dtype: torch.dtype | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x @ w.T (nn.Linear without bias); x [..., K], w [N, K]."""
    require_cuda(x, w)
    x2, _ = _row_major_2d(x, "x")
    w2, _ = _row_major_2d(w, "weight")
    x2, w2 = _tma_ready(x2), _tma_ready(w2)
    ldx, ldw = _ld(x2), _ld(w2)
    M, K = x2.shape
    N = w2.shape[0]
    if w2.shape[1] != K:
        raise ValueError("linear: weight in_features mismatch")
    out_dtype = out_dtype or x.dtype
    y = out if out is not None else torch.empty((*x.shape[:-1], N), device=x.device, dtype=out_dtype)
    y2, ldy = _row_major_2d(y, "out")
    _lib.call("rk_gemm_fprop", x2.data_ptr(), ldx, w2.data_ptr(), ldw, y2.data_ptr(), ldy, M, N, K,
              _gemm_dtype(x2, w2), _lib.code(y.dtype), _lib.stream_ptr())
    return y


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dx = dy @ w; dy [..., N], w [N, K]."""
    require_cuda(dy, w)
    g2, _ = _row_major_2d(dy, "dy")
    w2, _ = _row_major_2d(w, "weight")
    g2, w2 = _tma_ready(g2), _tma_ready(w2)
    ldg, ldw = _ld(g2), _ld(w2)
    M, N = g2.shape
    K = w2.shape[1]
    dx = torch.empty((*dy.shape[:-1], K), device=dy.device, dtype=out_dtype or dy.dtype)
    dx2, lddx = _row_major_2d(dx, "dx")
    _lib.call("rk_gemm_dgrad", g2.data_ptr(), ldg, w2.data_ptr(), ldw, dx2.data_ptr(), lddx, M, N, K,
              _gemm_dtype(g2, w2), _lib.code(dx.dtype), _lib.stream_ptr())
    return dx


def linear_dgrad_dsum(dy: torch.Tensor, w: torch.Tensor, o: torch.Tensor, n_heads: int, length: int):
    """(do, dsum) with do = dy @ w (16-bit, as linear_dgrad) and the attention
    backward's D = rowsum(do * o) per head (32 or 64 wide), [B, H, T] fp32,
    formed in the GEMM epilogue; None when the shapes do not fit that epilogue.
    dy [M, N], w [N, K], o [M, K] with K = n_heads * (32 or 64), M = B * length."""
    require_cuda(dy, w, o)
    M, N = dy.shape
    K = w.shape[1]
    if dy.dtype not in _TC_DTYPES or w.dtype != dy.dtype or o.dtype != dy.dtype or \
            K not in (32 * n_heads, 64 * n_heads) or \
            M % length or not (dy.is_contiguous() and w.is_contiguous() and o.is_contiguous()):
        return None
    do = torch.empty((M, K), device=dy.device, dtype=dy.dtype)
    dsum = torch.empty((M // length, n_heads, length), device=dy.device, dtype=torch.float32)
    st = _lib.lib().rk_gemm_dgrad_dsum(dy.data_ptr(), N, w.data_ptr(), K, do.data_ptr(), K, M, N, K,
                                       _lib.code(dy.dtype), o.data_ptr(), K, dsum.data_ptr(), length, n_heads,
                                       _lib.stream_ptr())
    if st == _lib.ERR_UNSUPPORTED:
        return None
    _lib.check(st, "rk_gemm_dgrad_dsum")
    return do, dsum


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor | None = None,
                 accumulate: bool = False) -> torch.Tensor:
    """dw (+)= dy^T @ x in fp32; dy [..., N], x [..., K] -> dw [N, K]."""
    require_cuda(dy, x)
    g2, _ = _row_major_2d(dy, "dy")
    x2, _ = _row_major_2d(x, "x")
    g2, x2 = _tma_ready(g2), _tma_ready(x2)
    ldg, ldx = _ld(g2), _ld(x2)
    M, N = g2.shape
    K = x2.shape[1]
    if dw is None:
        dw = torch.empty((N, K), device=dy.device, dtype=torch.float32)
        accumulate = False
    if dw.dtype != torch.float32:
        raise ValueError("weight gradients accumulate in fp32")
    ws_bytes = _lib.lib().rk_gemm_wgrad_workspace(M, N, K)
    ws = torch.empty(max(ws_bytes // 4, 1), device=dy.device, dtype=torch.float32)
    _lib.call("rk_gemm_wgrad", g2.data_ptr(), ldg, x2.data_ptr(), ldx, dw.data_ptr(), dw.stride(0), M, N, K,
              _gemm_dtype(g2, x2), int(accumulate), ws.data_ptr(), ws_bytes, _lib.stream_ptr())
    return dw


# ------------------------------------------------------------------ softmax head (fused cross-entropy)
def head_logits_buffer(rows: int, vocab: int, device, dtype) -> torch.Tensor:
    """[rows, vocab] view of a buffer whose row stride is vocab rounded up to 64
    (TMA needs 16-byte aligned rows)."""
    vpad = (vocab + 63) // 64 * 64
    return torch.empty((rows, vpad), device=device, dtype=dtype)[:, :vocab]


class HeadState:
    """What the softmax-head backward needs from the forward: expo [M, V]
    (exp(x - m_b), 16-bit), stats [M, width, 2] ((m_b, sum exp) per 128-column
    block), labels [M], and after head_loss rowc [M, 4] and the per-block
    factors fcoef [width, M]."""

    def __init__(self, expo, stats, xlabel, labels):
        self.expo, self.stats, self.xlabel, self.labels = expo, stats, xlabel, labels
        self.rowc = None
        self.fcoef = None


def head_fprop(hidden: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, expo: torch.Tensor | None = None,
               stats: torch.Tensor | None = None, xlabel: torch.Tensor | None = None) -> HeadState:
    """The head GEMM x = hidden @ w.T with the cross-entropy's log-sum-exp
    partials in its epilogue. hidden [M, K], w [V, K] (bf16/f16), labels [M]."""
    require_cuda(hidden, w)
    M, K = hidden.shape
    V = w.shape[0]
    if expo is None:
        expo = head_logits_buffer(M, V, hidden.device, hidden.dtype)
    width = _lib.lib().rk_head_stats_width(V)
    if stats is None:
        stats = torch.empty((M, width, 2), device=hidden.device, dtype=torch.float32)
    if xlabel is None:
        xlabel = torch.empty(M, device=hidden.device, dtype=torch.float32)
    _lib.call("rk_head_fprop", hidden.data_ptr(), _ld(hidden), w.data_ptr(), _ld(w), labels.data_ptr(),
              expo.data_ptr(), _ld(expo), stats.data_ptr(), xlabel.data_ptr(), M, V, K, _gemm_dtype(hidden, w),
              _lib.stream_ptr())
    return HeadState(expo, stats, xlabel, labels)


def head_loss(st: HeadState, grad_scale: float = 1.0, grad_scale_dev: torch.Tensor | None = None,
              ignore_index: int = -100, loss_rows: torch.Tensor | None = None,
              rowc: torch.Tensor | None = None, fcoef: torch.Tensor | None = None) -> torch.Tensor:
    """Per-row cross-entropy loss (0 for ignore_index); fills st.rowc and
    st.fcoef for the backward."""
    M, V = st.expo.shape
    dev = st.expo.device
    if loss_rows is None:
        loss_rows = torch.empty(M, device=dev, dtype=torch.float32)
    if rowc is None:
        rowc = torch.empty((M, 4), device=dev, dtype=torch.float32)
    if fcoef is None:
        fcoef = torch.empty((st.stats.shape[1], M), device=dev, dtype=torch.float32)
    _lib.call("rk_head_loss", st.stats.data_ptr(), st.stats.shape[1], st.xlabel.data_ptr(), st.labels.data_ptr(), M,
              V, float(grad_scale), _lib.ptr(grad_scale_dev), loss_rows.data_ptr(), rowc.data_ptr(),
              fcoef.data_ptr(), fcoef.stride(0), int(ignore_index), _lib.stream_ptr())
    st.rowc, st.fcoef = rowc, fcoef
    return loss_rows


def head_dgrad(st: HeadState, w: torch.Tensor, out_dtype: torch.dtype | None = None,
               split: bool = True) -> torch.Tensor:
    """dhidden = dlogits @ w, dlogits = (softmax - onehot) * scale formed inside the GEMM.
    With split (the default) the vocabulary reduction is sliced across all SMs
    when the output alone has fewer tiles than SMs (rk_head_dgrad_ws)."""
    M, V = st.expo.shape
    K = w.shape[1]
    dx = torch.empty((M, K), device=w.device, dtype=out_dtype or w.dtype)
    args = (st.expo.data_ptr(), _ld(st.expo), st.fcoef.data_ptr(), st.fcoef.stride(0), st.rowc.data_ptr(),
            st.labels.data_ptr(), w.data_ptr(), _ld(w), dx.data_ptr(), K, M, V, K, _gemm_dtype(st.expo, w),
            _lib.code(dx.dtype))
    ws_bytes = _lib.lib().rk_head_dgrad_workspace(M, V, K) if split else 0
    if ws_bytes > 0:
        ws = torch.empty(ws_bytes // 4, device=w.device, dtype=torch.float32)
        _lib.call("rk_head_dgrad_ws", *args, ws.data_ptr(), ws_bytes, _lib.stream_ptr())
    else:
        _lib.call("rk_head_dgrad", *args, _lib.stream_ptr())
    return dx


def head_wgrad(st: HeadState, hidden: torch.Tensor, dw: torch.Tensor | None = None,
               accumulate: bool = False) -> torch.Tensor:
    """dw (+)= dlogits^T @ hidden in fp32, dlogits formed inside the GEMM."""
    M, V = st.expo.shape
    K = hidden.shape[1]
    if dw is None:
        dw = torch.empty((V, K), device=hidden.device, dtype=torch.float32)
        accumulate = False
    _lib.call("rk_head_wgrad", st.expo.data_ptr(), _ld(st.expo), st.fcoef.data_ptr(), st.fcoef.stride(0),
              st.rowc.data_ptr(), st.labels.data_ptr(), hidden.data_ptr(), _ld(hidden), dw.data_ptr(), dw.stride(0),
              M, V, K, _gemm_dtype(st.expo, hidden), int(accumulate), _lib.stream_ptr())
    return dw


# ------------------------------------------------------------------ cross-entropy in pieces of the vocabulary
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_PIECE_BYTES = 512 << 20  # fp32: logits of the rows taken at a time


def _linear_ce_check_inputs(hidden, weight, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or 0 in weight.shape:
        raise ValueError("the head loss takes hidden [..., d] and a non-empty weight [vocabulary, d]")
    if hidden.dtype != weight.dtype or hidden.dtype not in _lib.DTYPE_CODE:
        raise ValueError("hidden and weight must share a type: fp32, bf16 or fp16")


def _linear_ce_check(hidden, weight, labels, reduction):
    require_cuda(hidden, weight, labels, what="the head loss")
    _linear_ce_check_inputs(hidden, weight, reduction)
    if labels.dtype is not torch.int64 or labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels must be int64 of shape {tuple(hidden.shape[:-1])}")
    _on_current_device(hidden, "hidden", weight, labels)


@functools.lru_cache(maxsize=64)
def _linear_ce_bytes(M: int, V: int, K: int, copy_w: bool) -> tuple[int, int]:
    lib = _lib.lib()
    return lib.rk_linear_ce_kept(M), lib.rk_linear_ce_fwd_workspace(M, V, K, copy_w)


@functools.lru_cache(maxsize=64)
def _linear_ce_bwd_bytes(M: int, V: int, K: int, copy_w: bool, dx: bool, dw: bool) -> int:
    flags = copy_w + (0 if dx else 2) + (0 if dw else 4)  # RK_LINEAR_CE_NO_DX, RK_LINEAR_CE_NO_DW
    return _lib.lib().rk_linear_ce_bwd_workspace(M, V, K, flags)


def _head_weight(weight: torch.Tensor) -> tuple[torch.Tensor, int, bool]:
    """(weight with unit-stride rows, row stride, whether the library has to copy it to rows that TMA can read)."""
    if weight.stride(1) != 1 or (weight.stride(0) < weight.shape[1] and weight.shape[0] > 1):
        weight = weight.contiguous()
    ld = weight.stride(0) if weight.shape[0] > 1 else weight.shape[1]
    return weight, ld, weight.data_ptr() % 16 != 0 or (weight.shape[0] > 1 and ld % 8 != 0)


def linear_ce_fwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                  reduction: str = "mean"):
    """(loss, kept): the cross-entropy of hidden [..., d] @ weight[V, d].T at labels [...] without its logits, fp32; kept
    is what linear_ce_bwd needs beside the inputs."""
    _linear_ce_check(hidden, weight, labels, reduction)
    labels = labels.contiguous()
    V, K = weight.shape
    loss = hidden.new_empty(labels.shape if reduction == "none" else (), dtype=torch.float32)
    if hidden.dtype == torch.float32:
        return _linear_ce_fwd_f32(hidden, weight, labels, ignore_index, reduction, loss)
    x, M, _, ld = even_rows(hidden)
    w, ldw, copy_w = _head_weight(weight)
    n_kept, n_ws = _linear_ce_bytes(M, V, K, copy_w)
    kept = labels.new_empty(n_kept // 4, dtype=torch.int32)
    ws = labels.new_empty(n_ws, dtype=torch.uint8)
    _lib.call("rk_linear_ce_fwd", x.data_ptr(), ld, w.data_ptr(), ldw, labels.data_ptr(), int(ignore_index), M, V, K,
              _lib.code(hidden.dtype), _REDUCTIONS[reduction], loss.data_ptr(), kept.data_ptr(), ws.data_ptr(), n_ws,
              _lib.stream_ptr())
    return loss, kept


def linear_ce_bwd(hidden: torch.Tensor, weight: torch.Tensor, kept: torch.Tensor, grad: torch.Tensor,
                  reduction: str = "mean", want_dx: bool = True, want_dw: bool = True,
                  dx_dtype: torch.dtype | None = None, dw_dtype: torch.dtype | None = None):
    """(d hidden, d weight) for the loss's gradient (a device scalar; one a row with reduction "none"), in the inputs'
    types unless others are given; None where not wanted."""
    _linear_ce_check_inputs(hidden, weight, reduction)
    V, K = weight.shape
    rows, f32 = hidden.shape[:-1].numel(), hidden.dtype is torch.float32
    if kept.dtype is not (torch.int64 if f32 else torch.int32) or kept.numel() != (rows if f32 else 4 + 4 * rows) or \
            not kept.is_contiguous():
        raise ValueError("kept must be what linear_ce_fwd returned for hidden")
    if grad.dtype is not torch.float32 or not grad.is_contiguous():
        grad = grad.detach().float().contiguous()
    if grad.get_device() != hidden.get_device() or grad.numel() != (rows if reduction == "none" else 1):
        raise ValueError("the loss's gradient must be on hidden's device, one number or one a row")
    _on_current_device(hidden, "hidden", weight, kept)
    dx = _new(hidden, dx_dtype or hidden.dtype) if want_dx else None
    dw = _new(weight, dw_dtype or weight.dtype) if want_dw else None
    if hidden.dtype == torch.float32:
        return _linear_ce_bwd_f32(hidden, weight, kept, grad, reduction, dx, dw)
    x, M, _, ld = even_rows(hidden)
    w, ldw, copy_w = _head_weight(weight)
    n_ws = _linear_ce_bwd_bytes(M, V, K, copy_w, want_dx, want_dw)
    ws = hidden.new_empty(n_ws, dtype=torch.uint8)
    _lib.call("rk_linear_ce_bwd", x.data_ptr(), ld, w.data_ptr(), ldw, kept.data_ptr(), M, V, K,
              _lib.code(hidden.dtype), _REDUCTIONS[reduction], grad.data_ptr(), _lib.ptr(dx), K,
              _lib.code(dx.dtype) if want_dx else 0, _lib.ptr(dw), K, _lib.code(dw.dtype) if want_dw else 0,
              ws.data_ptr(), n_ws, _lib.stream_ptr())
    return dx, dw


def _f32_chunks(hidden: torch.Tensor, labels: torch.Tensor, V: int):
    """(first row, rows, logits buffer) of the row chunks whose fp32 logits fit _PIECE_BYTES."""
    rows = labels.numel()
    step = min(rows, max(1, _PIECE_BYTES // (4 * V)))
    logits = torch.empty((step, V), device=hidden.device, dtype=torch.float32)
    for s in range(0, rows, max(step, 1)):
        yield s, min(step, rows - s), logits


def _linear_ce_fwd_f32(hidden, weight, labels, ignore_index, reduction, loss):
    """fp32 parity configuration: pieces of the rows, on the CUDA-core GEMM and the token-loss kernels."""
    V = weight.shape[0]
    x, y = hidden.reshape(-1, hidden.shape[-1]), labels.view(-1)
    ignored = y == ignore_index
    valid = ~ignored & (y >= 0) & (y < V)
    marks = torch.where(valid, y, torch.where(ignored, -100, -1))  # -1: outside the vocabulary, whatever ignore_index is
    rows = torch.empty(y.shape, device=x.device, dtype=torch.float32)
    w = weight.contiguous()
    for s, n, logits in _f32_chunks(x, y, V):
        linear_fwd(x[s:s + n].contiguous(), w, out=logits[:n])
        rows[s:s + n] = token_logprob_fwd(logits[:n], marks[s:s + n], want_stats=False)[0]
    rows.neg_()
    if reduction == "none":
        loss.copy_(rows.view(loss.shape))
    else:
        total = rows.sum(dtype=torch.float64)
        loss.copy_(total / valid.sum().clamp(min=1) if reduction == "mean" else total)
    return loss, torch.where(valid, y, -100)


def _linear_ce_bwd_f32(hidden, weight, kept, grad, reduction, dx, dw):
    V, K = weight.shape
    x, w = hidden.reshape(-1, K), weight.contiguous()
    valid = kept >= 0
    up = grad.view(-1) if reduction == "none" else grad.expand(kept.shape)
    up = torch.where(valid, -up / valid.sum().clamp(min=1) if reduction == "mean" else -up, 0.0)
    total = None if dw is None else torch.zeros((V, K), device=x.device, dtype=torch.float32)
    for s, n, logits in _f32_chunks(x, kept, V):
        xc = x[s:s + n].masked_fill(~valid[s:s + n, None], 0.0)  # what lies in an ignored row does not spread
        z = linear_fwd(xc, w, out=logits[:n])
        stats = token_logprob_fwd(z, kept[s:s + n])[2]
        d = token_logprob_bwd(z, kept[s:s + n], stats, up[s:s + n].contiguous(), out=z)
        if dx is not None:
            part = linear_dgrad(d, w)
            dx.view(-1, K)[s:s + n] = part.masked_fill_(~valid[s:s + n, None], 0.0)  # 0 times an infinite weight is none
        if total is not None:
            linear_wgrad(d, xc, dw=total, accumulate=True)
    return dx, total if dw is None or dw.dtype == torch.float32 else total.to(dw.dtype)


# ------------------------------------------------------------------ attention
def attention_fwd(qkv: torch.Tensor, n_heads: int, out: torch.Tensor | None = None):
    """Causal attention over packed qkv [B, T, 3*D]; returns (o [B, T, D], lse [B, H, T])."""
    require_cuda(qkv)
    if qkv.dim() != 3 or qkv.shape[-1] % (3 * n_heads) or qkv.stride(-1) != 1:
        raise ValueError("attention expects qkv [batch, length, 3*d_model] with a unit-stride last dim")
    B, T, three_d = qkv.shape
    D = three_d // 3
    HD = D // n_heads
    if qkv.stride(0) != T * qkv.stride(1):
        raise ValueError("qkv rows must be evenly strided")
    o = out if out is not None else torch.empty((B, T, D), device=qkv.device, dtype=qkv.dtype)
    lse = torch.empty((B, n_heads, T), device=qkv.device, dtype=torch.float32)
    _lib.call("rk_attn_fwd", qkv.data_ptr(), qkv.stride(1), o.data_ptr(), o.stride(1), lse.data_ptr(), B, n_heads,
              HD, T, _lib.code(qkv.dtype), _lib.stream_ptr())
    return o, lse


def attention_bwd(qkv: torch.Tensor, o: torch.Tensor, do: torch.Tensor, lse: torch.Tensor, n_heads: int,
                  dkv_stream: "torch.cuda.Stream | None" = None, dsum: torch.Tensor | None = None):
    """Returns dqkv [B, T, 3*D] for the causal attention of attention_fwd.
    With `dkv_stream` (16-bit inputs) the dK/dV kernel runs on that stream
    beside the dQ kernel, after D = rowsum(dO*O) is in place: `dsum`
    [B, H, T] when the caller formed it (linear_dgrad_dsum), else a small
    kernel writes it; the current stream waits for both before returning."""
    require_cuda(qkv, o, do, lse)
    B, T, three_d = qkv.shape
    D = three_d // 3
    do = do.to(o.dtype)
    if do.stride() != o.stride():
        do = do.contiguous()
        if do.stride() != o.stride():
            raise ValueError("dout must share the layout of out")
    dqkv = torch.empty_like(qkv)
    have_dsum = dsum is not None and dkv_stream is not None and qkv.dtype in _TC_DTYPES
    if not have_dsum:
        dsum = torch.empty((B, n_heads, T), device=qkv.device, dtype=torch.float32)
    args = (qkv.data_ptr(), qkv.stride(1), o.data_ptr(), do.data_ptr(), o.stride(1), lse.data_ptr(), dsum.data_ptr(),
            dqkv.data_ptr(), dqkv.stride(1), B, n_heads, D // n_heads, T, _lib.code(qkv.dtype))
    if dkv_stream is None or qkv.dtype not in _TC_DTYPES:
        _lib.call("rk_attn_bwd", *args, _lib.stream_ptr())
        return dqkv
    main = torch.cuda.current_stream()
    if not have_dsum:
        _lib.call("rk_attn_bwd_piece", 0, *args, main.cuda_stream)
    ready = torch.cuda.Event()
    ready.record(main)
    dkv_stream.wait_event(ready)
    _lib.call("rk_attn_bwd_piece", 2, *args, dkv_stream.cuda_stream)
    _lib.call("rk_attn_bwd_piece", 1, *args, main.cuda_stream)
    done = torch.cuda.Event()
    done.record(dkv_stream)
    main.wait_event(done)
    return dqkv


# ------------------------------------------------------------------ embedding
def embedding_fwd(ids: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor, out: torch.Tensor | None = None):
    """x[b, t] = tok[ids[b, t]] + pos[t] (fp32) for ids [B, T]; returns [B*T, d]."""
    require_cuda(ids, tok, pos)
    B, T = ids.shape
    d = tok.shape[1]
    ids = ids.contiguous()
    out = out if out is not None else torch.empty((B * T, d), device=tok.device, dtype=torch.float32)
    _lib.call("rk_embedding_fwd", ids.data_ptr(), tok.data_ptr(), pos.data_ptr(), out.data_ptr(), B * T, T, d,
              tok.shape[0], _lib.stream_ptr())
    return out


def embedding_bwd(ids: torch.Tensor, dx: torch.Tensor, g_tok: torch.Tensor, g_pos: torch.Tensor,
                  dx2: torch.Tensor | None = None):
    """Deterministically accumulates dx (+ dx2) [B*T, d] into g_tok[ids] and g_pos[t]."""
    require_cuda(ids, dx, g_tok, g_pos)
    B, T = ids.shape
    d = g_tok.shape[1]
    ids = ids.contiguous()
    ws_bytes = _lib.lib().rk_embedding_bwd_workspace(B * T, g_tok.shape[0])
    ws = torch.empty(max(ws_bytes, 1), device=dx.device, dtype=torch.uint8)
    _lib.call("rk_embedding_bwd", ids.data_ptr(), dx.contiguous().data_ptr(),
              None if dx2 is None else dx2.contiguous().data_ptr(), g_tok.data_ptr(), g_pos.data_ptr(),
              B * T, T, d, g_tok.shape[0], ws.data_ptr(), ws_bytes, _lib.stream_ptr())


def embedding_bwd_sort(ids: torch.Tensor, vocab: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """The first phase of embedding_bwd: the rows of ids [B, T] grouped by id,
    into a uint8 buffer that embedding_bwd_sorted reads. It depends on the ids
    alone, so it can be issued early, on another stream."""
    require_cuda(ids)
    rows = ids.numel()
    nbytes = _lib.lib().rk_embedding_bwd_sort_bytes(rows, vocab)
    if out is None:
        out = torch.empty(max(nbytes, 1), device=ids.device, dtype=torch.uint8)
    _lib.call("rk_embedding_bwd_sort", ids.contiguous().data_ptr(), rows, vocab, out.data_ptr(), out.numel(),
              _lib.stream_ptr())
    return out


def embedding_bwd_sorted(sorted_rows: torch.Tensor, dx: torch.Tensor, g_tok: torch.Tensor, g_pos: torch.Tensor,
                         T: int, dx2: torch.Tensor | None = None):
    """The rest of embedding_bwd from embedding_bwd_sort's result (same ids):
    accumulates dx (+ dx2) [B*T, d] into g_tok and g_pos, bit for bit as
    embedding_bwd does."""
    require_cuda(sorted_rows, dx, g_tok, g_pos)
    rows, d = dx.shape
    ws_bytes = _lib.lib().rk_embedding_bwd_sorted_workspace(rows, d)
    ws = torch.empty(max(ws_bytes, 1), device=dx.device, dtype=torch.uint8)
    _lib.call("rk_embedding_bwd_sorted", sorted_rows.data_ptr(), sorted_rows.numel(), dx.contiguous().data_ptr(),
              None if dx2 is None else dx2.contiguous().data_ptr(), g_tok.data_ptr(), g_pos.data_ptr(), rows, T, d,
              g_tok.shape[0], ws.data_ptr(), ws_bytes, _lib.stream_ptr())


# ------------------------------------------------------------------ fused reversible-step helpers
def add_rmsnorm_fwd(x: torch.Tensor, a: torch.Tensor, weight: torch.Tensor, eps: float, out_dtype: torch.dtype,
                    want_sum: bool = False, want_rstd: bool = True):
    """s = x + a; y = rmsnorm(s) * weight. Returns (y, s or None, rstd or None); rows contiguous."""
    require_cuda(x, a, weight)
    rows, width = x.shape
    y = torch.empty((rows, width), device=x.device, dtype=out_dtype)
    ssum = torch.empty((rows, width), device=x.device, dtype=torch.float32) if want_sum else None
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if want_rstd else None
    _lib.call("rk_add_rmsnorm_fwd", x.data_ptr(), a.data_ptr(), _lib.code(a.dtype), weight.data_ptr(), y.data_ptr(),
              _lib.code(out_dtype), _lib.ptr(ssum), _lib.ptr(rstd), rows, width, float(eps), _lib.stream_ptr())
    return y, ssum, rstd


def rmsnorm_bwd_fused(x: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, dy: torch.Tensor,
                      dw: torch.Tensor, residual: torch.Tensor | None = None, lp_add: torch.Tensor | None = None,
                      lp_dtype: torch.dtype | None = None, dx_out: torch.Tensor | None = None,
                      lp_out: torch.Tensor | None = None, accumulate_dw: bool = True, lp_scale: float = 1.0):
    """dx_out = rmsnorm_bwd(dy) + residual (fp32); lp_out = round(lp_add + round(dx)) if lp_add else
    round(round(dx_out) * lp_scale) (cast_scale of the total) when lp_dtype is given. dw
    accumulates. Returns (dx_out, lp_out)."""
    dx_out, lp_out, _ = _rmsnorm_bwd_fused(x, weight, rstd, dy, dw, residual, lp_add, lp_dtype, dx_out, lp_out,
                                           accumulate_dw, lp_scale)
    return dx_out, lp_out


def rmsnorm_bwd_fused_deferred(x: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, dy: torch.Tensor,
                               residual: torch.Tensor | None = None, lp_add: torch.Tensor | None = None,
                               lp_dtype: torch.dtype | None = None, lp_scale: float = 1.0):
    """rmsnorm_bwd_fused without the weight-gradient reduction: returns
    (dx_out, lp_out, partials); rmsnorm_dw_reduce(partials, rows, width, dw)
    finishes dw later (on any stream ordered after this one)."""
    return _rmsnorm_bwd_fused(x, weight, rstd, dy, None, residual, lp_add, lp_dtype, None, None, True, lp_scale)


def rmsnorm_dw_reduce(partials: torch.Tensor, rows: int, width: int, dw: torch.Tensor, accumulate: bool = True):
    """dw (+)= the fixed-order sum of the partials a deferred rmsnorm_bwd_fused left."""
    require_cuda(partials, dw)
    _lib.call("rk_rmsnorm_dw_reduce", partials.data_ptr(), rows, width, dw.data_ptr(), int(accumulate),
              _lib.stream_ptr())


def _rmsnorm_bwd_fused(x, weight, rstd, dy, dw, residual, lp_add, lp_dtype, dx_out, lp_out, accumulate_dw, lp_scale):
    require_cuda(x, weight, rstd, dy)
    rows, width = x.shape
    dx_out = dx_out if dx_out is not None else torch.empty((rows, width), device=x.device, dtype=torch.float32)
    if lp_dtype is not None and lp_out is None:
        lp_out = torch.empty((rows, width), device=x.device, dtype=lp_dtype)
    ws_bytes = _lib.lib().rk_rmsnorm_bwd_workspace(rows, width)
    ws = torch.empty(max(ws_bytes // 4, 1), device=x.device, dtype=torch.float32)
    _lib.call("rk_rmsnorm_bwd_fused", x.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dy.data_ptr(),
              _lib.code(dy.dtype), _lib.ptr(residual), _lib.ptr(lp_add), _lib.ptr(lp_out),
              _lib.code(lp_out.dtype) if lp_out is not None else _lib.code(dy.dtype), float(lp_scale), dx_out.data_ptr(),
              _lib.ptr(dw), int(accumulate_dw), ws.data_ptr(), ws_bytes, rows, width, _lib.stream_ptr())
    return dx_out, lp_out, ws


def reconstruct_midpoint_sum(x_next: torch.Tensor, a: torch.Tensor, m: torch.Tensor, coeff: float,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """x_prev = x_next - round(coeff * round(a + m)); coeff = -2h gives the forward update."""
    require_cuda(x_next, a, m)
    if a.dtype != m.dtype:
        raise ValueError("force parts must share a dtype")
    out = out if out is not None else torch.empty_like(x_next)
    _lib.call("rk_reconstruct_midpoint_sum", x_next.data_ptr(), a.data_ptr(), m.data_ptr(), _lib.code(a.dtype),
              float(coeff), out.data_ptr(), x_next.numel(), _lib.stream_ptr())
    return out


def linear_reconstruct(x: torch.Tensor, w: torch.Tensor, state: torch.Tensor, coeff: float,
                       addend: torch.Tensor | None = None, out: torch.Tensor | None = None, norm=None,
                       low: torch.Tensor | None = None):
    """out = state - round(coeff * round(round(x @ w^T) + addend)) with the
    sublayer output x @ w^T only in the GEMM epilogue (rk_gemm_fprop_reconstruct);
    bitwise equal to linear_fwd followed by reconstruct_midpoint_sum (addend) or
    reconstruct_midpoint. With norm = (weight, eps, y, rstd or None) the RMSNorm
    forward of `out` runs in the same pass (rk_gemm_fprop_reconstruct_norm,
    N == 256), bitwise equal to rmsnorm_fwd / add_rmsnorm_fwd; with `low` the
    rounded x @ w^T is stored there too. None when the shapes or dtypes do not
    fit the fused epilogue (the caller runs the separate steps)."""
    require_cuda(x, w, state)
    M, K = x.shape
    N = w.shape[0]
    if x.dtype not in _TC_DTYPES or w.dtype != x.dtype or state.dtype != torch.float32 or \
            tuple(state.shape) != (M, N) or (addend is not None and addend.dtype != x.dtype) or N % 32 or \
            not (x.is_contiguous() and w.is_contiguous() and state.is_contiguous()) or \
            (addend is not None and not addend.is_contiguous()):
        return None
    if norm is not None or low is not None:
        nw, eps, y, rstd = norm if norm is not None else (None, 0.0, None, None)
        if N != 256 or (nw is not None and (nw.dtype != torch.float32 or not nw.is_contiguous() or
                                            y.dtype != x.dtype or tuple(y.shape) != (M, N) or not y.is_contiguous())) \
                or (low is not None and (low.dtype != x.dtype or tuple(low.shape) != (M, N) or
                                         not low.is_contiguous())) or nw is None:
            return None
    out = out if out is not None else torch.empty_like(state)
    if norm is None:
        st = _lib.lib().rk_gemm_fprop_reconstruct(x.data_ptr(), K, w.data_ptr(), K, state.data_ptr(), N,
                                                  _lib.ptr(addend), N, float(coeff), out.data_ptr(), N, M, N, K,
                                                  _lib.code(x.dtype), _lib.stream_ptr())
        name = "rk_gemm_fprop_reconstruct"
    else:
        st = _lib.lib().rk_gemm_fprop_reconstruct_norm(x.data_ptr(), K, w.data_ptr(), K, state.data_ptr(), N,
                                                       _lib.ptr(addend), N, float(coeff), out.data_ptr(), N,
                                                       _lib.ptr(low), N, nw.data_ptr(), float(eps), y.data_ptr(), N,
                                                       _lib.ptr(rstd), M, N, K, _lib.code(x.dtype),
                                                       _lib.stream_ptr())
        name = "rk_gemm_fprop_reconstruct_norm"
    if st in (_lib.ERR_UNSUPPORTED, _lib.ERR_ALIGN):
        return None
    _lib.check(st, name)
    return out


def cast_scale(x: torch.Tensor, dtype: torch.dtype, scale: float) -> torch.Tensor:
    """round(round(x) * scale) in dtype (x fp32)."""
    require_cuda(x)
    out = torch.empty(x.shape, device=x.device, dtype=dtype)
    _lib.call("rk_cast_scale", x.data_ptr(), out.data_ptr(), _lib.code(dtype), float(scale), x.numel(),
              _lib.stream_ptr())
    return out


def linear_swiglu_fwd(x: torch.Tensor, w_up: torch.Tensor, save_u: bool = False):
    """h = silu(gate) * value of u = x @ w_up.T computed in the GEMM epilogue
    (u never written unless save_u). x [M, K], w_up [2ff, K] (gate rows first).
    Returns (h [M, ff], u [M, 2ff] or None)."""
    require_cuda(x, w_up)
    M, K = x.shape
    ff = w_up.shape[0] // 2
    h = torch.empty((M, ff), device=x.device, dtype=x.dtype)
    u = torch.empty((M, 2 * ff), device=x.device, dtype=x.dtype) if save_u else None
    _lib.call("rk_gemm_fprop_swiglu", x.data_ptr(), x.stride(0), w_up.data_ptr(), w_up.stride(0), h.data_ptr(), ff,
              _lib.ptr(u), 2 * ff, M, ff, K, _gemm_dtype(x, w_up), _lib.stream_ptr())
    return h, u


def linear_dgrad_swiglu(dy: torch.Tensor, w_down: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """du = swiglu_bwd(u, linear_dgrad(dy, w_down)) in one GEMM (the SwiGLU
    backward in the epilogue; dh never written). dy [M, d], w_down [d, ff],
    u [M, 2ff] (gate columns first). Returns du like u."""
    require_cuda(dy, w_down, u)
    M, d = dy.shape
    ff = w_down.shape[1]
    du = torch.empty_like(u)
    _lib.call("rk_gemm_dgrad_swiglu", dy.data_ptr(), dy.stride(0), w_down.data_ptr(), w_down.stride(0), u.data_ptr(),
              u.stride(0), du.data_ptr(), du.stride(0), M, ff, d, _gemm_dtype(dy, w_down), _lib.stream_ptr())
    return du


def dgrad_swiglu_fusable(dy: torch.Tensor, w_down: torch.Tensor, u: torch.Tensor) -> bool:
    return dy.dtype in _TC_DTYPES and w_down.dtype == dy.dtype and u.dtype == dy.dtype and \
        w_down.shape[1] % 64 == 0 and dy.is_contiguous() and w_down.is_contiguous() and u.is_contiguous() and \
        u.shape[1] == 2 * w_down.shape[1] and (dy.shape[1] * 2) % 16 == 0 and \
        all(t.data_ptr() % 16 == 0 for t in (dy, w_down, u))


def swiglu_fusable(x: torch.Tensor, w_up: torch.Tensor) -> bool:
    return x.dtype in _TC_DTYPES and w_up.dtype == x.dtype and (w_up.shape[0] // 2) % 128 == 0 and \
        x.is_contiguous() and w_up.is_contiguous() and (x.shape[1] * 2) % 16 == 0


# ------------------------------------------------------------------ token log-probabilities and their losses
def token_rows(logits: torch.Tensor, labels: torch.Tensor, name: str = "labels") -> tuple[int, int, int, torch.Tensor]:
    """Checks logits [..., V] against labels [...] and returns (rows, V, row stride, contiguous labels). The rows
    must be evenly strided (any stride of at least V, no alignment rule) and the last dimension unit-stride."""
    require_cuda(logits, labels)
    if logits.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"logits must be fp32, bf16 or fp16, got {logits.dtype}")
    if labels.dtype is not torch.int64 or labels.get_device() != logits.get_device() or logits.dim() < 1 or \
            labels.shape != logits.shape[:-1]:
        raise ValueError(f"{name} must be int64 on the logits' device with shape {tuple(logits.shape[:-1])}")
    V = logits.shape[-1]
    if logits.get_device() != torch.cuda.current_device():
        raise ValueError("logits must be on the current CUDA device")
    if V and logits.is_contiguous():
        return labels.numel(), V, V, labels if labels.is_contiguous() else labels.contiguous()
    if V < 1 or (V > 1 and logits.stride(-1) != 1):
        raise ValueError("logits must have a non-empty, unit-stride last dimension")
    rows, ld = 1, None
    for size, stride in zip(reversed(logits.shape[:-1]), reversed(logits.stride()[:-1])):
        if size != 1:
            if ld is None:
                ld = stride
            elif stride != ld * rows and logits.numel():
                raise ValueError("logits rows must be evenly strided (pass a contiguous tensor)")
            rows *= size
    if ld is None or rows <= 1:
        ld = V
    if ld < V and rows:
        raise ValueError("logits rows overlap")
    return rows, V, max(ld, V), labels.contiguous()


def like_rows(logits: torch.Tensor, rows: int, ld: int) -> torch.Tensor:
    """An uninitialised tensor of logits' shape and row stride (so both sides share their 16-byte phase)."""
    V = logits.shape[-1]
    if ld == V:
        return torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    return torch.empty((rows, ld), device=logits.device, dtype=logits.dtype)[:, :V].view(logits.shape)


def row_values(t: torch.Tensor | None, like: torch.Tensor, name: str) -> torch.Tensor | None:
    """An fp32 contiguous array of one value a row (None passes)."""
    if t is None:
        return None
    if t.get_device() != like.get_device() or t.shape != like.shape:
        raise ValueError(f"{name} must be on the logits' device with shape {tuple(like.shape)}")
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


def device_scalar(t, device, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.device != device or t.numel() != 1:
        raise ValueError(f"{name} must be a scalar tensor on the logits' device")
    return t.detach().float()


def token_logprob_fwd(logits: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0, ignore_index: int = -100,
                      entropy: bool = False, want_stats: bool = True):
    """(logprob, entropy or None, stats or None) of logits [..., V] at labels [...], fp32 in the shape of labels;
    0 at ignore_index. stats [rows, 2]: what token_logprob_bwd needs of a row (its reference value and sum)."""
    rows, V, ld, labels = token_rows(logits, labels)
    logprob = torch.empty(labels.shape, device=logits.device, dtype=torch.float32)
    h = torch.empty_like(logprob) if entropy else None
    stats = torch.empty((rows, 2), device=logits.device, dtype=torch.float32) if want_stats else None
    n_ws = _lib.lib().rk_token_logprob_workspace(rows)
    ws = torch.empty(n_ws, device=logits.device, dtype=torch.uint8) if n_ws else None
    _lib.call("rk_token_logprob_fwd", logits.data_ptr(), ld, V, labels.data_ptr(), rows, 1.0 / temperature,
              int(ignore_index), _lib.code(logits.dtype), logprob.data_ptr(), _lib.ptr(h), _lib.ptr(stats), _lib.ptr(ws),
              n_ws, _lib.stream_ptr())
    return logprob, h, stats


def token_logprob_bwd(logits: torch.Tensor, labels: torch.Tensor, stats: torch.Tensor, d_logprob: torch.Tensor,
                      entropy: torch.Tensor | None = None, d_entropy: torch.Tensor | None = None,
                      temperature: float = 1.0, ignore_index: int = -100, scale: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """d loss / d logits (in the logits' dtype, rounded once) from contiguous fp32 d loss / d logprob and, with
    `entropy`, d loss / d entropy, times the device scalar `scale`. `out` may be the logits themselves."""
    return token_logprob_bwd_at(logits, labels, stats.data_ptr(), d_logprob.data_ptr(), 1, entropy, _lib.ptr(d_entropy),
                                temperature, ignore_index, scale, out)


def token_logprob_bwd_at(logits, labels, stats: int, d_logprob: int, coef_stride: int, entropy, d_entropy: int | None,
                         temperature, ignore_index, scale, out=None) -> torch.Tensor:
    """token_logprob_bwd with its row factors given by address (they may be interleaved)."""
    rows, V, ld, labels = token_rows(logits, labels)
    out, ldd = gradient_rows(logits, out, rows, ld)
    _lib.call("rk_token_logprob_bwd", logits.data_ptr(), ld, V, labels.data_ptr(), rows, 1.0 / temperature,
              ignore_index, _lib.code(logits.dtype), stats, _lib.ptr(entropy), d_logprob, d_entropy, coef_stride,
              _lib.ptr(scale), out.data_ptr(), ldd, _lib.stream_ptr())
    return out


def gradient_rows(logits: torch.Tensor, out: torch.Tensor | None, rows: int, ld: int) -> tuple[torch.Tensor, int]:
    """(gradient tensor, its row stride): a new one laid out like the logits, or a checked `out`, of which autograd is
    told that it is written (a loss that saved it must not take the gradients for its logits)."""
    if out is None:
        return like_rows(logits, rows, ld), ld
    if out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise ValueError("out must match the logits' shape, dtype and device")
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError("out must have a unit-stride last dimension")
    V = logits.shape[-1]
    ldd = token_rows(out, torch.empty(out.shape[:-1], device=out.device, dtype=torch.int64))[2]
    if out.data_ptr() == logits.data_ptr() and rows and ldd != ld:  # strides of dimensions of size 1 say nothing
        raise ValueError("out may alias the logits only with the same strides")
    gap = (out.data_ptr() - logits.data_ptr()) // out.element_size()
    first = (rows - 1) * (ld if gap > 0 else ldd) + V  # elements from the start of the one that lies first to its end
    if rows and gap and abs(gap) < first and not (ld == ldd and V <= abs(gap) % ld <= ld - V):
        raise ValueError("out overlaps the logits without being the same rows")
    torch.autograd.graph.increment_version(out)
    return out, ldd


@functools.lru_cache(maxsize=64)
def _policy_workspace(rows: int) -> int:
    return _lib.lib().rk_policy_workspace(rows)


@functools.lru_cache(maxsize=64)
def _preference_workspace(pairs: int, length: int) -> int:
    return -(-_lib.lib().rk_preference_workspace(pairs, length) // 16) * 16


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                ref_logprobs: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                temperature: float = 1.0, ignore_index: int = -100, entropy: bool = False,
                denominator: torch.Tensor | None = None, grad_scale: float = 1.0,
                grad_scale_dev: torch.Tensor | None = None, want_grad: bool = True, want_coef: bool = False,
                out: torch.Tensor | None = None):
    """rk_policy_loss: (loss, clip fraction, logprob, kl or None, entropy or None, dlogits or None, pairs or None), pairs
    [2, rows, 2] being the rows' statistics and factors for the backward. advantages has the shape of actions or of its
    leading dimensions (one a sequence)."""
    rows, V, ld, actions = token_rows(logits, actions, "actions")
    dev = logits.device
    old = row_values(old_logprobs, actions, "old_logprobs")
    ref = row_values(ref_logprobs, actions, "ref_logprobs")
    w = row_values(weights, actions, "weights")
    lead, group = advantages.dim(), 1
    if advantages.get_device() != actions.get_device() or advantages.shape != actions.shape[:lead]:
        raise ValueError("advantages must be on the logits' device with the shape of actions or of its leading "
                         "dimensions")
    if lead < actions.dim():
        group = max(1, actions.shape[lead:].numel())
    adv = row_values(advantages, advantages, "advantages")
    denominator = device_scalar(denominator, dev, "denominator")
    grad_scale_dev = device_scalar(grad_scale_dev, dev, "grad_scale")
    want_h = entropy or entropy_coef != 0
    # metrics and workspace in one allocation; what the backward keeps, apart from them, in another
    n_ws = _policy_workspace(rows)
    aux = torch.empty(4 + n_ws // 4, device=dev, dtype=torch.float32)
    pairs = torch.empty(4 * rows, device=dev, dtype=torch.float32) if want_coef else None
    at, pairs_at = aux.data_ptr(), _lib.ptr(pairs)
    logprob = torch.empty(actions.shape, device=dev, dtype=torch.float32)
    kl = torch.empty_like(logprob) if ref is not None else None
    h = torch.empty_like(logprob) if want_h else None
    dlogits, ldd = gradient_rows(logits, out, rows, ld) if want_grad else (None, V)
    terms = _lib.POLICY_TERMS.pack(old.data_ptr(), adv.data_ptr(), _lib.ptr(ref) or 0, _lib.ptr(w) or 0,
                                   _lib.ptr(denominator) or 0, _lib.ptr(grad_scale_dev) or 0, group, clip_low, clip_high,
                                   kl_coef, entropy_coef, 1.0 / temperature, grad_scale)
    _lib.call("rk_policy_loss", logits.data_ptr(), ld, V, actions.data_ptr(), rows, int(ignore_index),
              _lib.code(logits.dtype), terms, logprob.data_ptr(), _lib.ptr(kl), _lib.ptr(h), at,
              pairs_at, pairs_at + 8 * rows if pairs_at else None, _lib.ptr(dlogits), ldd, at + 16, n_ws,
              _lib.stream_ptr())
    return aux[0], aux[2], logprob, kl, h, dlogits, pairs


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logprobs: torch.Tensor | None, kind: str,
                    beta: float, label_smoothing: float = 0.0, average: bool = False, temperature: float = 1.0,
                    ignore_index: int = -100, grad_scale: float = 1.0, grad_scale_dev: torch.Tensor | None = None,
                    want_grad: bool = True, out: torch.Tensor | None = None):
    """rk_preference_loss: (loss, logprob, rewards [2 * pairs], dlogits or None, rows' statistics [2 * rows] and factors
    [rows] in one array) for logits [2 * pairs, length, V], chosen sequences first."""
    if logits.dim() != 3 or logits.shape[0] % 2 or logits.shape[0] == 0:
        raise ValueError("preference logits must be [2 * pairs, length, vocabulary], chosen sequences first")
    if kind not in _lib.PREFERENCE_KINDS:
        raise ValueError(f"kind must be one of {sorted(_lib.PREFERENCE_KINDS)}")
    rows, V, ld, labels = token_rows(logits, labels)
    dev = logits.device
    seqs, length = labels.shape
    ref = row_values(ref_logprobs, labels, "ref_logprobs")
    grad_scale_dev = device_scalar(grad_scale_dev, dev, "grad_scale")
    n_ws = _preference_workspace(seqs // 2, length)
    # loss and workspace in one allocation; what the backward keeps, apart from them, in another
    aux = torch.empty(4 + n_ws // 4, device=dev, dtype=torch.float32)
    kept = torch.empty(3 * rows, device=dev, dtype=torch.float32)
    logprob = torch.empty(labels.shape, device=dev, dtype=torch.float32)
    rewards = torch.empty(seqs, device=dev, dtype=torch.float32)
    at = aux.data_ptr()
    stats_at = kept.data_ptr()
    dlogits, ldd = gradient_rows(logits, out, rows, ld) if want_grad else (None, V)
    terms = _lib.PREFERENCE_TERMS.pack(_lib.ptr(ref) or 0, _lib.ptr(grad_scale_dev) or 0, beta, label_smoothing,
                                       1.0 / temperature, grad_scale, _lib.PREFERENCE_KINDS[kind], int(average))
    _lib.call("rk_preference_loss", logits.data_ptr(), ld, V, labels.data_ptr(), seqs // 2, length, int(ignore_index),
              _lib.code(logits.dtype), terms, logprob.data_ptr(), rewards.data_ptr(), at,
              stats_at, stats_at + 8 * rows, _lib.ptr(dlogits), ldd, at + 16, n_ws, _lib.stream_ptr())
    return aux[0], logprob, rewards, dlogits, kept
