"""AdamW over a module's own tensors (csrc/adamw_multi.cu): one launch for up to
64 parameters of a kind, moments in 32 or 8 bits, global-norm clipping fused in.

The trainer (train.py) keeps its parameters in one flat buffer and updates them
with rk_adamw_step; this optimizer is for models trained through autograd, whose
parameters and gradients lie where PyTorch put them.
"""
from __future__ import annotations

import array
import ctypes
import itertools
import math
import operator

import torch

from . import _lib
from . import functional as fn

QUANT_BLOCK = 256  # elements that share a scale in 8-bit moments
_FIELDS = 7        # 8-byte fields of rk_adamw_tensor
_NO_RATE = (None, None)


def _seen(state) -> tuple[list, list]:
    """The parameters and their entries in an optimizer's state."""
    return list(state), list(state.values())


def _same(seen, state) -> bool:
    """Whether these are still the same objects in the same order (a comparison would look into the tensors)."""
    return len(seen[0]) == len(state) and all(map(operator.is_, seen[0], state)) and \
        all(map(operator.is_, seen[1], state.values()))


class _Launch:
    """The tensors of one group with one parameter and one gradient type and one count of steps: their rk_adamw_tensor
    array, whose moment addresses and sizes stay from step to step while p and g are written anew in each."""

    def __init__(self, index: int, bits: int, p_dtype: torch.dtype, g_dtype: torch.dtype, block: torch.Tensor | None = None):
        self.index, self.bits, self.p_dtype, self.g_dtype = index, bits, p_dtype, g_dtype
        self.block, self.counter = block, (index, id(block))  # the scalars that count their steps, None for the group's
        self.p_code, self.g_code = _lib.code(p_dtype), _lib.code(g_dtype)
        self.entries = []  # (parameter, elements, place among all parameters)
        self.flat = []
        # of each entry its state, of all entries the moments (held, so that nothing else can lie there) and their addresses
        self.names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")[:4 if bits == 8 else 2]
        self.of_state = operator.itemgetter(*self.names)
        self.states, self.moments, self.at = [], [], []

    def add(self, p: torch.Tensor, g: torch.Tensor, state: dict, place: int) -> None:
        n, blocks = p.numel(), -(-p.numel() // QUANT_BLOCK)
        kinds = ((torch.int8, n), (torch.uint8, n), (torch.float32, blocks), (torch.float32, blocks)) if self.bits == 8 else \
            ((torch.float32, n), (torch.float32, n))
        for name, (dtype, size) in zip(self.names, kinds):
            t = state.get(name)
            if t is None or t.dtype is not dtype or t.numel() != size or not t.is_contiguous() or \
                    t.get_device() != p.get_device():
                raise ValueError(f"{self.bits}-bit moments: {name} must be a contiguous {dtype} tensor of {size} elements "
                                 "on the parameter's device")
        moments = self.of_state(state)
        at = [t.data_ptr() for t in moments]
        self.entries.append((p, n, place))
        self.states.append(state)
        self.moments += moments
        self.at += at
        self.flat += (p.data_ptr(), g.data_ptr(), *at, *(0,) * (4 - len(at)), n)

    def finish(self) -> "_Launch":
        self.parts = _lib.lib().rk_adamw_multi_parts(len(self.entries))  # of the norm's partial sums
        self.words = array.array("Q", self.flat)
        self.table = (ctypes.c_uint64 * len(self.flat)).from_buffer(self.words) if self.flat else None
        return self

    def moved(self) -> bool:
        """Whether a moment lies elsewhere than when the table was made."""
        of_state = self.of_state
        try:
            return [t.data_ptr() for state in self.states for t in of_state(state)] != self.at
        except KeyError:
            return True

    def refill(self, grads, device: int) -> bool:
        """Writes the addresses of parameters and gradients into the table; False if it does not fit them or the
        moments have moved."""
        if self.moved():
            return False
        words, field, g_dtype = self.words, 0, self.g_dtype
        for p, n, i in self.entries:
            g = p.grad if grads is None else grads[i]  # autograd holds .grad to the parameter's shape
            if g is None or g.dtype is not g_dtype or p.numel() != n or g.get_device() != device or \
                    not g.is_contiguous() or not p.is_contiguous():
                return False
            if grads is not None and g.shape != p.shape or grads is None and g.numel() != n:
                return False
            at = p.data_ptr()
            if at != words[field]:  # memory that it did not leave is of one type, and no two devices share an address
                if p.dtype is not self.p_dtype or p.get_device() != device:
                    return False
                words[field] = at
            words[field + 1] = g.data_ptr()
            field += _FIELDS
        return True


class AdamW(torch.optim.Optimizer):
    """Decoupled-weight-decay Adam (torch.optim.AdamW's update and defaults) for CUDA fp32, bf16 or fp16 parameters
    with gradients of any of these types, moments held in fp32 or in 8 bits.

    state_bits (a group option): 32, or 8 for block-wise codes of 256 elements (2 + 2/64 bytes a parameter instead
    of 8). Small, sensitive tensors such as norm weights can be given a group of their own with 32.
    max_norm: clip the gradients' global norm over all groups to it (torch.nn.utils.clip_grad_norm_ without its
    rescaling pass over the gradients); the norm of the last step is `grad_norm`, a device scalar.

    Each tensor counts the steps that found a gradient for it. Tensors that have always stepped together share their
    scalars: the group's (param_groups[i]["scalars"], which hold its learning rate too) or, for those that came in late
    or were left out of a step, a copy of their own (state[p]["scalars"]), with a launch of its own. A captured graph
    counts the tensors together that it was captured with.

    Step count, learning rate and the derived constants live on the device, so a captured graph that contains step()
    counts on when it is replayed; a learning rate changed in param_groups is copied there by the next step() outside a
    graph, or by sync_lr(), and never by a capture, except that a rate given as a tensor on the device is read from that
    tensor by each replay. What a step() makes for itself cannot be captured: take a first step, with the same
    gradients, outside the graph."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_norm: float | None = None):
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be positive")
        self.max_norm = max_norm
        self.grad_norm = None  # the gradients' global norm before clipping in the last step (device scalar)
        self._captured = {}    # by id, what captured graphs go on reading and writing
        self._partials = []    # workspaces of the norm, the last one in use
        self._reset()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      scalars=None))

    def _reset(self) -> None:
        self._launches = None  # the last step's plan
        self._made_of = []     # (state_bits, parameters) of each group then
        self._state_of = ()    # the optimizer's state then
        self._idle = []        # (place, parameter) outside it
        self._updated = []     # the parameters in it
        self._parts = None     # (address, size) of the norm's workspace for it
        self._coded = None     # the table of the parameters with 8-bit moments
        self._coded_of = ()    # the optimizer's state when it was made
        self._norm_of = None   # the address of the scalars that grad_norm is a view of
        self._lr = {}          # by id, device scalars and the learning rate that they hold
        self._counted = {}     # by id, the groups' scalars that steps have counted in

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self.grad_norm = None
        self.__dict__.setdefault("_captured", {})  # load_state_dict comes here too
        self.__dict__.setdefault("_partials", [])
        self._reset()

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
        scalars, first = group["scalars"], group["params"][0]
        if scalars is None or scalars.get_device() != first.get_device():
            self._uncaptured()
            dev = first.device
            scalars = torch.zeros(8, device=dev, dtype=torch.float32) if scalars is None else scalars.to(dev)
            group["scalars"] = scalars
        return self._with_rate(scalars, group["lr"])

    def _with_rate(self, scalars: torch.Tensor, lr) -> torch.Tensor:
        """The scalars, holding this learning rate."""
        if isinstance(lr, torch.Tensor):
            capturing = torch.cuda.is_current_stream_capturing()
            if not capturing or lr.device == scalars.device:
                scalars[0].copy_(lr.detach())
            if capturing:
                self._captured[id(lr)] = lr
            self._lr.pop(id(scalars), None)
        elif self._lr.get(id(scalars), _NO_RATE)[1] != lr and not torch.cuda.is_current_stream_capturing():
            scalars[0].fill_(lr)  # in a graph it would put this rate back with every replay
            self._lr[id(scalars)] = scalars, lr
        return scalars

    def _all_scalars(self, index: int) -> list[torch.Tensor]:
        """The group's scalars and those that its tensors have of their own."""
        group = self.param_groups[index]
        own = (self.state[p]["scalars"] for p in group["params"] if p in self.state and "scalars" in self.state[p])
        blocks = {id(t): t for t in (self._group_scalars(index), *own)}
        return [self._with_rate(t, group["lr"]) for t in blocks.values()]

    def _count(self, found) -> None:
        """Parts the counts of tensors that no longer step together, before a step with these (group index, parameter,
        gradient, place) tuples: those of a block that are left out go on with a copy of it; those without moments start
        from zero, on the group's scalars if none has stepped there."""
        live = {id(p) for _, p, _, _ in found}
        for index, group in enumerate(self.param_groups):
            blocks, new = {}, []
            for p in group["params"]:
                state = self.state.get(p)
                if state and "exp_avg" in state:
                    block = state.get("scalars")
                    blocks.setdefault(id(block), (block, [], []))[1 if id(p) in live else 2].append(state)
                elif id(p) in live:
                    new.append(p)
            for block, steps, rests in blocks.values():
                if steps and rests:
                    self._uncaptured()
                    copy = (self._group_scalars(index) if block is None else block).clone()
                    for state in rests:
                        state["scalars"] = copy
            if new and group["scalars"] is not None:
                if blocks:
                    self._uncaptured()
                    block = torch.zeros(8, device=new[0].device, dtype=torch.float32)
                    for p in new:
                        self.state[p]["scalars"] = block
                elif id(group["scalars"]) in self._counted:  # all moments have been dropped
                    self._uncaptured()
                    group["scalars"] = None

    def _uncaptured(self) -> None:
        """Moments and scalars made in a capture would start anew with every replay."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a first step cannot be captured; take one with these gradients outside the graph")

    def sync_lr(self) -> None:
        """Copies the groups' learning rates to the device (for graph replays; step() does it by itself)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.sync_lr: a captured copy would put these rates back with every replay")
        for i, group in enumerate(self.param_groups):
            if group["params"]:
                self._all_scalars(i)

    def set_step(self, step: int) -> None:
        """Sets the number of steps already taken (bias correction), as when moments come from elsewhere."""
        for i, group in enumerate(self.param_groups):
            if group["params"]:
                for scalars in self._all_scalars(i):
                    scalars[1].fill_(float(step))
        self._counted, self._launches = {}, None  # no step has counted on from here

    # ---- state
    def _moments_of(self, p: torch.Tensor, bits: int) -> dict:
        state = self.state[p]
        if "exp_avg" not in state:
            self._uncaptured()
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
        cast codes and fp32 moments to the parameters' type). Refuses the state of another optimizer."""
        for group in state_dict["param_groups"]:
            missing = {"lr", "betas", "eps", "weight_decay", "state_bits", "scalars"} - set(group)
            if missing:
                raise ValueError("not the state of an optim.AdamW of this package: its groups have no " +
                                 ", ".join(sorted(missing)) + ". To take over moments from another optimizer, put them into "
                                 "state[p] as fp32 exp_avg and exp_avg_sq and call set_step()")
        super().load_state_dict(state_dict)
        saved = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        own = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        copies = {}  # what tensors share stays shared

        def copy(v, device):
            if not isinstance(v, torch.Tensor):
                return v
            return copies.setdefault((id(v), device), v.detach().to(device, copy=True))
        for key, p in zip(saved, own):
            if key in state_dict["state"]:
                self.state[p] = {k: copy(v, p.device) for k, v in state_dict["state"][key].items()}
        self._reset()
        for group in self.param_groups:
            if group["scalars"] is not None and any("exp_avg" in self.state.get(p, ()) for p in group["params"]):
                group["scalars"] = scalars = group["scalars"].to(group["params"][0].device)
                self._counted[id(scalars)] = scalars

    def _plan(self, found) -> list[_Launch]:
        """The launches for (group index, parameter, gradient, place) tuples."""
        launches = {}
        for index, p, g, i in found:
            if p.dtype not in _lib.DTYPE_CODE or not p.is_contiguous():
                raise ValueError("AdamW parameters must be contiguous fp32, bf16 or fp16")
            bits = self.param_groups[index]["state_bits"]
            if bits not in (8, 32):
                raise ValueError("state_bits must be 8 or 32")
            block = self.state[p].get("scalars")
            if block is not None and block.device != p.device:
                raise ValueError("scalars must be on the parameter's device")
            key = index, id(block), p.dtype, g.dtype
            if key not in launches:
                launches[key] = _Launch(index, bits, p.dtype, g.dtype, block)
            launches[key].add(p, g, self._moments_of(p, bits), i)
        return [launch.finish() for launch in launches.values()]

    def _refill(self, launches, grads) -> bool:
        """Writes the addresses of parameters and gradients into the last plan's tables; False if the plan does not fit
        (other groups or parameters, another set of gradients, other types or sizes, moments replaced, a gradient that
        needs a copy)."""
        if len(self._made_of) != len(self.param_groups):
            return False
        for group, (bits, params) in zip(self.param_groups, self._made_of):
            now = group["params"]
            if group["state_bits"] != bits or len(now) != len(params) or not all(map(operator.is_, now, params)):
                return False
        if not _same(self._state_of, self.state):
            return False
        for i, p in self._idle:
            if (p.grad if grads is None else grads[i]) is not None and p.numel():
                return False
        device = torch.cuda.current_device()
        for launch in launches:
            if not launch.refill(grads, device):
                return False
        return True

    @torch.no_grad()
    def _collect(self, grads) -> list:
        """Checks the gradients and plans the launches for them; returns what has to live until those are queued."""
        found = []  # (group index, parameter, gradient, the parameter's place among all)
        self._launches, self._idle, self._coded = None, [], None
        device = torch.cuda.current_device()
        places = itertools.count()
        for index, group in enumerate(self.param_groups):
            for p in group["params"]:
                i = next(places)
                g = p.grad if grads is None else grads[i]
                if g is not None and (g.layout is not torch.strided or g.dtype not in _lib.DTYPE_CODE or
                                      g.get_device() != p.get_device() or g.shape != p.shape):
                    raise ValueError("AdamW gradients must be dense fp32, bf16 or fp16 in the parameters' shape and "
                                     "on their device")
                if g is None or not p.numel():
                    self._idle.append((i, p))
                elif p.get_device() != device:
                    raise ValueError("AdamW parameters with gradients must be on the current CUDA device")
                else:
                    found.append((index, p, g if g.is_contiguous() else g.contiguous(), i))
        self._count(found)
        self._launches = self._plan(found)
        for launch in self._launches:
            if launch.block is None:
                block = self._group_scalars(launch.index)
                self._counted[id(block)] = block
        self._updated, self._parts = [p for _, p, _, _ in found], None
        self._state_of = _seen(self.state)
        self._made_of = [(group["state_bits"], list(group["params"])) for group in self.param_groups]
        return found

    def _norm_workspace(self, parts: int, device: torch.device) -> torch.Tensor:
        """At least `parts` floats. A workspace is never given back: a captured graph or another stream may still write
        to it."""
        if not self._partials or self._partials[-1].numel() < parts or self._partials[-1].device != device:
            self._partials.append(torch.empty(parts, device=device, dtype=torch.float32))
        return self._partials[-1]

    def _keep_for_replays(self, launches, scalars=()) -> None:
        """Holds the moments and scalars whose addresses a capture is about to record: a state that is loaded or put in
        their place must not leave replays with memory that belongs to others. Parameters and gradients are the
        caller's to hold, as with any captured graph."""
        for t in itertools.chain(scalars, *(launch.moments for launch in launches)):
            self._captured[id(t)] = t

    # ---- the step
    def step(self, closure=None, *, grads=None):
        """One update. grads: gradients in the order of the parameters over all groups (None where there is none),
        instead of the parameters' .grad; they may have another floating type than the parameters."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grads is not None:
            grads = list(grads)
            if len(grads) != sum(len(group["params"]) for group in self.param_groups):
                raise ValueError("grads must hold an entry for each parameter")
        keep = None
        if self._launches is None or not self._refill(self._launches, grads):
            keep = self._collect(grads)
        launches = self._launches
        if not launches:
            return loss
        stream = _lib.stream_ptr()
        scalars = {}
        for launch in launches:
            if launch.counter not in scalars:
                scalars[launch.counter] = self._group_scalars(launch.index) if launch.block is None else \
                    self._with_rate(launch.block, self.param_groups[launch.index]["lr"])
        if torch.cuda.is_current_stream_capturing():
            self._keep_for_replays(launches, scalars.values())
        norm = None, 0
        if self.max_norm is not None:
            if self._parts is None:
                parts = sum(launch.parts for launch in launches)
                self._parts = self._norm_workspace(parts, self._updated[0].device).data_ptr(), parts
            norm = self._parts
            at = norm[0]
            for launch in launches:
                _lib.call("rk_adamw_multi_sumsq", launch.table, len(launch.entries), launch.g_code, at, stream)
                at += 4 * launch.parts
        for (index, _), block in scalars.items():
            group = self.param_groups[index]
            b1, b2 = group["betas"]
            _lib.call("rk_adamw_multi_prepare", *norm, self.max_norm or 0.0, b1, b2,
                      group["weight_decay"], block.data_ptr(), stream)
        if self.max_norm is not None:
            block = scalars[launches[0].counter]
            if block.data_ptr() != self._norm_of:
                self._norm_of, self.grad_norm = block.data_ptr(), block[2]
        for launch in launches:
            group = self.param_groups[launch.index]
            b1, b2 = group["betas"]
            _lib.call("rk_adamw_multi_step", launch.table, len(launch.entries), launch.p_code, launch.g_code, launch.bits,
                      scalars[launch.counter].data_ptr(), b1, b2, group["eps"], stream)
        # the kernels wrote past autograd: a graph kept from before must not take the new values for the old ones
        torch.autograd.graph.increment_version(self._updated)
        del keep
        return loss

    @torch.no_grad()
    def moments(self, out=None, dtype: torch.dtype = torch.float32) -> list:
        """The values that the 8-bit moments stand for: a pair (exp_avg, exp_avg_sq) for each parameter with 8-bit
        state, in the order of the parameters. out: pairs of contiguous tensors of one type to write into."""
        coded = self._coded
        if coded is None or not _same(self._coded_of, self.state) or coded.moved():
            coded = _Launch(-1, 8, torch.float32, torch.float32)
            for p in (p for g in self.param_groups if g["state_bits"] == 8 for p in g["params"]):
                if p in self.state and "exp_avg" in self.state[p]:
                    if p.get_device() != torch.cuda.current_device():
                        raise ValueError("AdamW parameters must be on the current CUDA device")
                    coded.add(p, p, self.state[p], 0)
            self._coded, self._coded_of = coded.finish(), _seen(self.state)
        if out is None:
            out = [(torch.empty_like(p, dtype=dtype), torch.empty_like(p, dtype=dtype)) for p, *_ in coded.entries]
        if len(out) != len(coded.entries):
            raise ValueError(f"out must hold {len(coded.entries)} pairs")
        if not out:
            return out
        table, field, kind, device = coded.table, 0, out[0][0].dtype, torch.cuda.current_device()
        for (_, n, *_), (m, v) in zip(coded.entries, out):
            if m.numel() != n or v.numel() != n or m.dtype is not kind or v.dtype is not kind or \
                    m.get_device() != device or v.get_device() != device or \
                    not (m.is_contiguous() and v.is_contiguous()):
                raise ValueError("out pairs must be contiguous CUDA tensors of one type and the parameters' sizes")
            table[field] = m.data_ptr()
            table[field + 1] = v.data_ptr()
            field += _FIELDS
        if torch.cuda.is_current_stream_capturing():
            self._keep_for_replays([coded])
        _lib.call("rk_adamw_multi_moments", table, len(out), _lib.code(kind), _lib.stream_ptr())
        return out
