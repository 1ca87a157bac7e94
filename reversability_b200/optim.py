"""AdamW over a module's own tensors (csrc/adamw_multi.cu): one launch for up to
64 parameters of a kind, moments in 32 or 8 bits, global-norm clipping fused in.

The trainer (train.py) keeps its parameters in one flat buffer and updates them
with rk_adamw_step; this optimizer is for models trained through autograd, whose
parameters and gradients lie where PyTorch put them.
"""
from __future__ import annotations

import ctypes
import itertools
import math

import torch

from . import _lib
from . import functional as fn

QUANT_BLOCK = 256  # elements that share a scale in 8-bit moments
_FIELDS = 7        # 8-byte fields of rk_adamw_tensor


def _table(entries) -> tuple:
    """rk_adamw_tensor array (every field is 8 bytes) from tuples of seven integers."""
    flat = list(itertools.chain.from_iterable(entries))
    return (ctypes.c_uint64 * len(flat))(*flat), len(flat) // _FIELDS


class AdamW(torch.optim.Optimizer):
    """Decoupled-weight-decay Adam (torch.optim.AdamW's update and defaults) for CUDA fp32, bf16 or fp16 parameters
    with gradients of any of these types, moments held in fp32 or in 8 bits.

    state_bits (a group option): 32, or 8 for block-wise codes of 256 elements (2 + 2/64 bytes a parameter instead
    of 8). Small, sensitive tensors such as norm weights can be given a group of their own with 32.
    max_norm: clip the gradients' global norm over all groups to it (torch.nn.utils.clip_grad_norm_ without its
    rescaling pass over the gradients); the norm of the last step is `grad_norm`, a device scalar.

    A group counts one step for each step() that finds a gradient in it. Step count, learning rate and the derived constants live on the device, so a captured graph that contains
    step() counts on when it is replayed; a learning rate changed in param_groups is copied there by the next
    step() outside a graph, or by sync_lr()."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_norm: float | None = None):
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be positive")
        self.max_norm = max_norm
        self.grad_norm = None  # the gradients' global norm before clipping in the last step (device scalar)
        self._lr = {}  # group index -> the learning rate its device scalars hold
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      scalars=None))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            b1, b2 = group["betas"]
            if group["state_bits"] not in (8, 32):
                raise ValueError("state_bits must be 8 or 32")
            if not (0 <= b1 < 1 and 0 <= b2 < 1):
                raise ValueError("betas must be in [0, 1)")
            if not (float(group["lr"]) >= 0 and group["eps"] >= 0 and math.isfinite(group["weight_decay"])):
                raise ValueError("lr and eps must not be negative and weight_decay must be finite")
            for p in group["params"]:
                fn.require_cuda(p, what="AdamW parameters")
                if p.dtype not in _lib.DTYPE_CODE or not p.is_contiguous():
                    raise ValueError("AdamW parameters must be contiguous fp32, bf16 or fp16")
        except ValueError:
            self.param_groups.pop()
            raise

    # ---- device scalars
    def _group_scalars(self, index: int) -> torch.Tensor:
        """fp32[8] of the group on its device: [0] lr, [1] steps taken, [2] gradient norm, [3] clip coefficient."""
        group = self.param_groups[index]
        dev = group["params"][0].device
        scalars = group["scalars"]
        if scalars is None:
            scalars = torch.zeros(8, device=dev, dtype=torch.float32)
        elif scalars.device != dev:
            scalars = scalars.to(dev)
        if scalars is not group["scalars"]:
            group["scalars"] = scalars
            self._lr.pop(index, None)
        lr = group["lr"]
        if isinstance(lr, torch.Tensor):
            scalars[0].copy_(lr)
        elif self._lr.get(index) != lr:
            scalars[0].fill_(lr)
            self._lr[index] = lr
        return scalars

    def sync_lr(self) -> None:
        """Copies the groups' learning rates to the device (for graph replays; step() does it by itself)."""
        for i, group in enumerate(self.param_groups):
            if group["params"]:
                self._group_scalars(i)

    def set_step(self, step: int) -> None:
        """Sets the number of steps already taken (bias correction), as when moments come from elsewhere."""
        for i, group in enumerate(self.param_groups):
            if group["params"]:
                self._group_scalars(i)[1].fill_(float(step))

    # ---- state
    def _moments_of(self, p: torch.Tensor, bits: int) -> dict:
        state = self.state[p]
        if "exp_avg" not in state:
            if bits == 32:
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            else:
                blocks = -(-p.numel() // QUANT_BLOCK)
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.int8)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8)
                state["exp_avg_scale"] = torch.zeros(blocks, device=p.device, dtype=torch.float32)
                state["exp_avg_sq_scale"] = torch.zeros(blocks, device=p.device, dtype=torch.float32)
        return state

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim.Optimizer.load_state_dict, but the moments keep their saved types (the base class would
        cast codes and fp32 moments to the parameters' type)."""
        super().load_state_dict(state_dict)
        saved = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        own = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(saved, own):
            if key in state_dict["state"]:
                self.state[p] = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in state_dict["state"][key].items()}
        self._lr.clear()

    def _entry(self, p: torch.Tensor, g: torch.Tensor, bits: int) -> tuple:
        st = self._moments_of(p, bits)
        m, v = st["exp_avg"], st["exp_avg_sq"]
        if bits == 8:
            if m.dtype != torch.int8 or v.dtype != torch.uint8:
                raise ValueError("8-bit moments must be int8 and uint8 codes")
            return (p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), st["exp_avg_scale"].data_ptr(),
                    st["exp_avg_sq_scale"].data_ptr(), p.numel())
        if m.dtype != torch.float32 or v.dtype != torch.float32:
            raise ValueError("32-bit moments must be fp32")
        return p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0, p.numel()

    # ---- the step
    @torch.no_grad()
    def step(self, closure=None, *, grads=None):
        """One update. grads: gradients in the order of the parameters over all groups (None where there is none),
        instead of the parameters' .grad; they may have another floating type than the parameters."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        given = None if grads is None else iter(grads)
        launches = []  # (group index, p dtype, g dtype, entries)
        keep = []      # contiguous copies, alive until the launches are queued
        for index, group in enumerate(self.param_groups):
            bits, kinds = group["state_bits"], {}
            for p in group["params"]:
                g = p.grad if given is None else next(given, None)
                if g is None:
                    continue
                if g.layout != torch.strided or g.dtype not in _lib.DTYPE_CODE or g.device != p.device or \
                        g.shape != p.shape:
                    raise ValueError("AdamW gradients must be dense fp32, bf16 or fp16 in the parameters' shape and "
                                     "on their device")
                if not g.is_contiguous():
                    g = g.contiguous()
                    keep.append(g)
                if p.numel():
                    kinds.setdefault((p.dtype, g.dtype), []).append(self._entry(p, g, bits))
            launches += [(index, pd, gd, *_table(entries)) for (pd, gd), entries in kinds.items()]
        if not launches:
            return loss
        stream, lib = _lib.stream_ptr(), _lib.lib()
        partials, parts = None, 0
        if self.max_norm is not None:
            counts = [lib.rk_adamw_multi_parts(n) for *_, n in launches]
            parts = sum(counts)
            partials = torch.empty(parts, device=self.param_groups[launches[0][0]]["params"][0].device,
                                   dtype=torch.float32)
            at = partials.data_ptr()
            for (_, _, gd, table, n), count in zip(launches, counts):
                _lib.call("rk_adamw_multi_sumsq", table, n, _lib.code(gd), at, stream)
                at += 4 * count
        scalars = {}
        for index in dict.fromkeys(i for i, *_ in launches):
            group, scalars[index] = self.param_groups[index], self._group_scalars(index)
            b1, b2 = group["betas"]
            _lib.call("rk_adamw_multi_prepare", _lib.ptr(partials), parts, self.max_norm or 0.0, b1, b2,
                      group["weight_decay"], scalars[index].data_ptr(), stream)
        if self.max_norm is not None:
            self.grad_norm = scalars[launches[0][0]][2]
        for index, pd, gd, table, n in launches:
            group = self.param_groups[index]
            b1, b2 = group["betas"]
            _lib.call("rk_adamw_multi_step", table, n, _lib.code(pd), _lib.code(gd), group["state_bits"],
                      scalars[index].data_ptr(), b1, b2, group["eps"], stream)
        return loss

    @torch.no_grad()
    def moments(self, out=None, dtype: torch.dtype = torch.float32) -> list:
        """The values that the 8-bit moments stand for: a pair (exp_avg, exp_avg_sq) for each parameter with 8-bit
        state, in the order of the parameters. out: pairs of contiguous tensors of one type to write into."""
        params = [p for g in self.param_groups if g["state_bits"] == 8 for p in g["params"] if "exp_avg" in self.state[p]]
        if out is None:
            out = [(torch.empty_like(p, dtype=dtype), torch.empty_like(p, dtype=dtype)) for p in params]
        if len(out) != len(params):
            raise ValueError(f"out must hold {len(params)} pairs")
        entries, kinds = [], set()
        for p, (m, v) in zip(params, out):
            if m.shape != p.shape or v.shape != p.shape or m.device != p.device or v.device != p.device or \
                    not (m.is_contiguous() and v.is_contiguous()):
                raise ValueError("out pairs must be contiguous in the parameters' shapes and on their device")
            kinds |= {m.dtype, v.dtype}
            st = self.state[p]
            entries.append((m.data_ptr(), v.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(),
                            st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_scale"].data_ptr(), p.numel()))
        if not entries:
            return out
        if len(kinds) != 1:
            raise ValueError("out tensors must share one type")
        table, n = _table(entries)
        _lib.call("rk_adamw_multi_moments", table, n, _lib.code(kinds.pop()), _lib.stream_ptr())
        return out
