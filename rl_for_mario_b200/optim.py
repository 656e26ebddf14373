"""The end of a training step: the norm of a model's gradient and AdamW, over all tensors at once.

The reference's trainer clips the gradient's norm and takes an AdamW step
(trainer/train_pretrain.py:121-129).  ``grad_norm`` is that norm, ``AdamW`` a torch
optimizer whose step() is one or two kernels for all of its parameters: clipping is part
of it, the averages are kept in 32 or in 8 bits, and 16-bit weights may have fp32 ones
beside them.  A step reads its learning rate (a tensor, if it is given as one), its
seed and its number on the device, so that a captured step is a step of its own at
each replay.
"""
from __future__ import annotations

import copy
import ctypes
import math
import struct
import sys
from array import array
from operator import attrgetter
from typing import Dict, Iterable, List, Optional, Tuple, Union

import torch

from . import kernels

Tensor = torch.Tensor

BLOCK = 256  # elements of a parameter that share a scale; each parameter starts a new block
_MOST_GROUPS = 16
_GROUP = struct.Struct("5dQ")
_LEAST_FP32, _MOST_FP32 = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _dense(t: Tensor) -> bool:
    """Whether the tensor's elements lie side by side in some order of its dimensions."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


# Each of these looks at one property of many tensors without an interpreted loop: a model has a hundred
# tensors, and a microsecond for each would be more than the kernels take.
_data_ptr, _numel, _contiguous, _on = (getattr(Tensor, n) for n in ("data_ptr", "numel", "is_contiguous", "get_device"))
_dtype_of, _grad_of, _bytes = attrgetter("dtype"), attrgetter("grad"), attrgetter("nbytes")


def _address(values: array) -> int:
    return values.buffer_info()[0]


def grad_norm(tensors: Iterable[Optional[Tensor]]) -> Tensor:
    """The 2-norm of all tensors taken as one, an fp32 number on their device; None among them is passed
    over.  bf16, fp16 or fp32, mixed, any shapes and strides.  fp64 sums in a fixed order."""
    ts = [t for t in tensors if t is not None]
    if not ts:
        raise ValueError("grad_norm needs one tensor at least")
    dev, dt = ts[0].device, ts[0].dtype
    if (dev.type == "cuda" and dt in kernels._DTYPES and set(map(_dtype_of, ts)) == {dt}
            and set(map(_on, ts)) == {dev.index} and all(map(_contiguous, ts))):
        kinds = array("i", [kernels._DTYPES[dt]]) * len(ts)
    else:
        kinds = array("i")
        for i, t in enumerate(ts):
            if t.device != dev or dev.type != "cuda":
                kernels._same_device(*ts)
            if t.layout is not torch.strided:
                raise TypeError("grad_norm takes dense tensors")
            kinds.append(kernels._dtype_code(t))
            if not _dense(t):
                ts[i] = t.contiguous()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = kernels._workspace("dt_grad_norm_workspace", dev.index, len(ts))
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    at, n = array("q", map(_data_ptr, ts)), array("q", map(_numel, ts))
    kernels._launch("dt_grad_norm", dev, len(ts), _address(at), _address(n), _address(kinds), norm.data_ptr(),
                    ws.data_ptr(), size)
    return norm


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over bf16, fp16 and fp32 parameters of one CUDA device, mixed:

        m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    ``state_bits`` 32: averages in fp32.  8: in one byte an element with a power of two for each 256 elements,
    rounded up or down at random (by ``seed``, the step and the element), so that they follow the gradients
    as those in 32 bits do: v to about 10 % of its root, m to about 8 %.  Ranks that hold copies of the same
    parameters take the same seed, which keeps the copies the same.
    ``master``: fp32 weights are kept beside 16-bit parameters; without them a step smaller than half a unit
    in the last place of a 16-bit weight is lost.  They are what a step starts from: reset_master() after the
    parameters were changed from outside.
    ``max_norm``: the gradient is scaled so that its norm over all parameters is at most this; the norm of
    each step is in ``norm``.  A step whose norm is not finite changes nothing and is not counted.

    Groups (16 at most) have lr, betas, eps and weight_decay of their own; lr may be an fp32 tensor of one
    number on the device.  t is the number of steps of the optimizer: a parameter without a gradient is left
    alone in that step.  Parameters may be used in any order of memory as long as they have no gaps.
    ``moments()`` gives the averages; ``state_dict()`` holds them flat, parameter i from element 256 (blocks of
    256 of the parameters before it) on.
    """

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32, master: bool = False,
                 max_norm: Optional[float] = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32 (got {state_bits})")
        if max_norm is not None and not 0.0 < ctypes.c_float(max_norm).value < math.inf:
            raise ValueError(f"max_norm must be positive and finite (got {max_norm})")
        if not -2 ** 63 <= int(seed) < 2 ** 64:
            raise ValueError("seed must fit 64 bits")
        self.state_bits, self.max_norm, self.keeps_master = state_bits, max_norm, bool(master)
        self.seed = int(seed) - 2 ** 64 if int(seed) >= 2 ** 63 else int(seed)
        self._order: List[Tensor] = []  # parameters as they were added: the order of the flat arrays
        self._buffers: Dict[str, Tensor] = {}
        self._built = 0  # parameters that the arrays are made for
        self._packed: List[Tuple[Optional[tuple], bytes]] = []  # of each group: its numbers, and these as bytes
        self.norm: Optional[Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    # --------------------------------------------------------------------- parameters
    def add_param_group(self, param_group) -> None:
        if len(self.param_groups) == _MOST_GROUPS:
            raise ValueError(f"AdamW takes {_MOST_GROUPS} groups at most")
        super().add_param_group(param_group)
        try:
            group = self.param_groups[-1]
            for p in group["params"]:
                self._check_param(p)
            self._pack_group(group, group["params"][0].device if group["params"] else None)
        except BaseException:
            self.param_groups.pop()
            raise
        self._order.extend(group["params"])
        self._packed.append((None, b""))

    def _check_param(self, p: Tensor) -> None:
        if not p.is_cuda:
            raise ValueError("AdamW updates CUDA parameters only (no CPU path)")
        first = self._order[0] if self._order else self.param_groups[-1]["params"][0]
        if p.device != first.device:
            raise ValueError(f"parameters are on different devices ({first.device} and {p.device})")
        if p.dtype not in kernels._DTYPES:
            raise TypeError(f"unsupported dtype {p.dtype}")
        if p.layout is not torch.strided or not _dense(p):
            raise ValueError(f"a parameter of shape {tuple(p.shape)}, strides {tuple(p.stride())} has gaps")

    @staticmethod
    def _pack_group(g: dict, dev: Optional[torch.device] = None) -> bytes:
        """The group's numbers as the entry point takes them, checked."""
        lr, (b1, b2), eps, wd = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        at = 0
        if isinstance(lr, Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != (dev or lr.device) or not lr.is_cuda:
                raise ValueError("an lr tensor must be one fp32 number on the parameters' device")
            at, lr = lr.data_ptr(), 0.0
        if not (0.0 <= lr < math.inf and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and 0.0 <= wd < math.inf):
            raise ValueError(f"lr and weight_decay must not be negative, betas lie in [0, 1) (got lr {lr}, betas "
                             f"{(b1, b2)}, weight_decay {wd})")
        if not _LEAST_FP32 <= eps <= _MOST_FP32:
            raise ValueError(f"eps must be a normal number in fp32 (got {eps})")
        return _GROUP.pack(lr, b1, b2, eps, wd, at)

    def _overlap(self) -> None:
        spans = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in self._order if p.numel())
        for (a, n), (b, _) in zip(spans, spans[1:]):
            if a + n > b:
                raise ValueError("two parameters share memory")

    def _build(self) -> None:
        """(Re)makes the flat arrays for the parameters there are; what was there stays in front."""
        ps = self._order
        self._overlap()
        dev = ps[0].device
        blocks = [(p.numel() + BLOCK - 1) // BLOCK for p in ps]
        total, old = sum(blocks), self._buffers
        shapes = {"exp_avg": total * BLOCK, "exp_avg_sq": total * BLOCK}
        byte = torch.uint8 if self.state_bits == 8 else torch.float32
        new = {k: torch.zeros(n, dtype=byte, device=dev) for k, n in shapes.items()}
        if self.state_bits == 8:
            for k in shapes:
                new[k + "_scale"] = torch.full((total,), 32, dtype=torch.uint8, device=dev)
        if self.keeps_master:
            new["master"] = torch.zeros(total * BLOCK, dtype=torch.float32, device=dev)
            self._fill_master(new["master"], self._built)
        for k, t in old.items():
            if k in new:
                new[k][:t.numel()].copy_(t)
        if "count" not in old:
            self._buffers["count"] = torch.tensor([self.seed, 0], dtype=torch.int64, device=dev)
            self._buffers["ticket"] = torch.zeros(1, dtype=torch.int32, device=dev)
            old = self._buffers
        self._buffers = {**new, "count": old["count"], "ticket": old["ticket"]}
        self._built = len(ps)
        self._blocks = total
        group = {id(p): i for i, g in enumerate(self.param_groups) for p in g["params"]}
        self._dtypes = [p.dtype for p in ps]
        self._numels = [p.numel() for p in ps]
        self._nbytes = list(map(_bytes, ps))
        self._strides = [None if p.is_contiguous() else p.stride() for p in ps]
        self._sizes = array("q", self._numels)
        self._kinds = array("i", [kernels._dtype_code(p) + 256 * group[id(p)] for p in ps])
        self._plain = all(st is None for st in self._strides)
        self._look(list(map(_data_ptr, ps)))

    def _fill_master(self, master: Tensor, first: int) -> None:
        at = 0
        for i, p in enumerate(self._order):
            if i >= first and p.dtype != torch.float32:
                master[at:at + p.numel()].copy_(torch.as_strided(p.detach(), (p.numel(),), (1,)))
            at += (p.numel() + BLOCK - 1) // BLOCK * BLOCK

    @torch.no_grad()
    def reset_master(self) -> None:
        """Takes the fp32 weights from the 16-bit parameters anew: after these were changed from outside (weights loaded
        into the model, say), which the next step would otherwise undo."""
        self._ready()
        if self.keeps_master:
            self._fill_master(self._buffers["master"], 0)

    def _ready(self) -> None:
        if not self._order:
            raise ValueError("AdamW has no parameters")
        if self._built != len(self._order):
            self._build()

    # --------------------------------------------------------------------------- step
    def step(self, closure=None):
        # torch wraps an optimizer's step to run its hooks and mark it for the profiler, which takes 15 us; that
        # wrapper is used where there is a hook or a profiler to serve.
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or any(map(len, _GLOBAL_HOOKS))
                or _profiling()):
            return _hooked_step(self, closure)
        return self._step(closure)

    step.hooked = True  # (tells torch not to wrap it again)

    @torch.no_grad()
    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._ready()
        ps, buf = self._order, self._buffers
        dev = buf["count"].device
        at, to, keep = self._addresses(ps, dev.index)
        if to is None or not self._blocks:
            self.norm = None
            return loss
        size, ws, norm = 0, None, None
        if self.max_norm is not None:
            size = kernels._workspace("dt_grad_norm_workspace", dev.index, len(ps))
            ws = buf.get("parts")
            if ws is None or ws.numel() < size:
                ws = buf["parts"] = torch.empty(size, dtype=torch.uint8, device=dev)
            norm = self.norm = torch.empty((), dtype=torch.float32, device=dev)
        groups = b"".join([self._group_bytes(i, g, dev) for i, g in enumerate(self.param_groups)])
        kernels._launch("dt_adamw_step", dev, len(ps), _address(at), _address(to), _address(self._sizes),
                        _address(self._kinds), len(self.param_groups), groups, self.state_bits,
                        buf["exp_avg"].data_ptr(), buf["exp_avg_sq"].data_ptr(), kernels._ptr(buf.get("exp_avg_scale")),
                        kernels._ptr(buf.get("exp_avg_sq_scale")), kernels._ptr(buf.get("master")),
                        buf["count"].data_ptr(), buf["ticket"].data_ptr(), self.max_norm or 0.0, kernels._ptr(norm),
                        kernels._ptr(ws), size)
        # The launch writes through addresses: PyTorch has to be told, as autograd's check of saved tensors and every
        # weight derived from these (a model's folded norms) go by the version.  (2 us for 53 tensors.)
        torch.autograd.graph.increment_version(ps if all(to) else [p for p, g in zip(ps, to) if g])
        return loss

    def weights_changed(self) -> None:
        """Tells PyTorch that the parameters were written, which step() does by itself.  A replay of a captured step runs
        no Python: call this after it, before the model is used outside the graph, as what is derived from the
        weights (MarioDT.fuse_norms, FastDTAttention) is taken anew when their version has changed."""
        torch.autograd.graph.increment_version(self._order)

    def _addresses(self, ps: List[Tensor], index: int):
        """(addresses of the parameters, of their gradients, tensors to be held until the launch); the second None
        without any gradient.  Every parameter and gradient is looked at in every step."""
        grads = list(map(_grad_of, ps))
        live = [g for g in grads if g is not None]
        if not live:
            return None, None, live
        at = list(map(_data_ptr, ps))
        # Nothing is held of a parameter's memory: other memory may stand at its address of the last look.
        if at != self._seen:
            for i in range(len(ps)):
                self._same(i)
            self._overlap()
            self._look(at)
        if (len(live) == len(ps) and self._plain and list(map(_bytes, ps)) == self._nbytes
                and all(map(_contiguous, ps)) and all(map(_contiguous, grads))
                and list(map(_dtype_of, grads)) == self._dtypes and list(map(_numel, grads)) == self._numels
                and set(map(_on, grads)) == {index}):
            return self._at, array("q", list(map(_data_ptr, grads))), grads
        keep: List[Tensor] = []
        to = array("q", [self._gradient(i, g, keep) for i, g in enumerate(grads)])
        return self._at, to, keep

    def _look(self, at: List[int]) -> None:
        """Notes where the parameters are."""
        self._seen, self._at = at, array("q", at)

    def _same(self, i: int) -> Tensor:
        """Parameter i, whose type, size, order of memory and device have to be those of the flat arrays."""
        p = self._order[i]
        if (p.dtype != self._dtypes[i] or p.numel() != self._numels[i] or p.device != self._buffers["count"].device
                or (None if p.is_contiguous() else p.stride()) != self._strides[i]):
            raise ValueError(f"parameter {i} has changed its type, size, strides or device")
        return p

    def _gradient(self, i: int, g: Optional[Tensor], keep: List[Tensor]) -> int:
        """The address of parameter i's gradient in the parameter's order of memory; 0 without one."""
        p = self._same(i)
        if g is None:
            return 0
        if g.layout is not torch.strided:
            raise TypeError("AdamW takes dense gradients")
        if g.dtype != p.dtype or g.shape != p.shape or g.device != p.device:
            raise ValueError(f"the gradient of parameter {i} does not match it")
        if g.stride() != p.stride() and not (g.is_contiguous() and p.is_contiguous()):
            g = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(g)
            keep.append(g)
        return g.data_ptr()

    def _group_bytes(self, i: int, g: dict, dev: torch.device) -> bytes:
        """_pack_group of group i, taken again when one of its numbers has changed."""
        if isinstance(g["lr"], Tensor):
            return self._pack_group(g, dev)
        key = (g["lr"], *g["betas"], g["eps"], g["weight_decay"])  # (numbers: a list of betas may be changed in place)
        was, packed = self._packed[i]
        if was != key:
            packed = self._pack_group(g, dev)
            self._packed[i] = key, packed
        return packed

    # -------------------------------------------------------------------------- state
    def steps(self) -> Tensor:
        """The number of steps taken, an int64 number on the device."""
        self._ready()
        return self._buffers["count"][1].clone()

    @property
    def master(self) -> Optional[Tensor]:
        """The fp32 weights of 16-bit parameters, flat."""
        self._ready()
        return self._buffers.get("master")

    def moments(self) -> Tuple[Tensor, Tensor]:
        """(m, v), flat: the optimizer's own fp32 arrays, or with 8 bits the numbers that they stand for, as new
        bf16 tensors (bf16 holds each of them)."""
        self._ready()
        b = self._buffers
        if self.state_bits == 32:
            return b["exp_avg"], b["exp_avg_sq"]
        dev = b["count"].device
        m, v = (torch.empty(self._blocks * BLOCK, dtype=torch.bfloat16, device=dev) for _ in range(2))
        if self._blocks:
            kernels._launch("dt_adamw_moments", dev, b["exp_avg"].data_ptr(), b["exp_avg_scale"].data_ptr(),
                            b["exp_avg_sq"].data_ptr(), b["exp_avg_sq_scale"].data_ptr(), self._blocks, m.data_ptr(),
                            v.data_ptr())
        return m, v

    def state_dict(self) -> dict:
        """{"state": seed, step and the flat arrays themselves, "param_groups": as torch's}."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        self._ready()
        number = {id(p): i for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        groups = [{**{k: v for k, v in g.items() if k != "params"}, "params": [number[id(p)] for p in g["params"]]}
                  for g in self.param_groups]
        state = {k: v for k, v in self._buffers.items() if k not in ("count", "ticket", "parts")}
        result = {"state": {"seed": self.seed, "step": self._buffers["count"][1], **state}, "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            other = hook(self, result)
            result = result if other is None else other
        return result

    def load_state_dict(self, state_dict: dict) -> None:
        """Takes copies of what state_dict() gave, from any device; a group's rate that is a tensor here takes the loaded
        value where it is.  Nothing is changed where the state does not fit."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            other = hook(self, state_dict)
            state_dict = state_dict if other is None else other
        self._load(state_dict)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    @torch.no_grad()
    def _load(self, state_dict: dict) -> None:
        self._ready()
        state, groups = state_dict["state"], state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state has other groups of parameters")
        mine = {k: v for k, v in self._buffers.items() if k not in ("count", "ticket", "parts")}
        if set(mine) | {"seed", "step"} != set(state):
            raise ValueError(f"the state has {sorted(state)}, this optimizer {sorted(mine)}, seed and step")
        for k, t in mine.items():
            if state[k].numel() != t.numel() or state[k].dtype != t.dtype:
                raise ValueError(f"{k} of the state does not match: {tuple(state[k].shape)} {state[k].dtype}, "
                                 f"{tuple(t.shape)} {t.dtype} here")
        dev = self._buffers["count"].device
        # What is loaded becomes this optimizer's own; a rate on the device keeps its place, where captured steps read it.
        # (Copied together, and moved once each: groups that share a rate go on sharing it.)
        loaded = copy.deepcopy([{k: v for k, v in new.items() if k != "params"} for new in groups])
        rates = {id(new["lr"]): new["lr"] for new in loaded if isinstance(new["lr"], Tensor)}
        moved = {i: lr.to(dev) for i, lr in rates.items()}
        for g, new in zip(self.param_groups, loaded):
            new["lr"] = moved.get(id(new["lr"]), new["lr"])
            self._pack_group(new, dev)
            new["params"] = g["params"]
        seed, step = int(state["seed"]), torch.as_tensor(state["step"], dtype=torch.int64).reshape(())
        for k, t in mine.items():
            t.copy_(state[k].reshape(-1))
        self.seed = seed
        self._buffers["count"][0].fill_(seed)
        self._buffers["count"][1].copy_(step)
        written: Dict[int, float] = {}
        for g, new in zip(self.param_groups, loaded):
            lr = g["lr"]
            if isinstance(lr, Tensor):
                value = float(new["lr"])
                if written.setdefault(id(lr), value) != value:  # shared here, but not there
                    lr = torch.empty_like(lr)
                new["lr"] = lr.fill_(value)
            g.clear()
            g.update(new)

    def __getstate__(self) -> dict:
        """All but hooks and a step() that a scheduler put in the class's place, which belong to this object: a copy
        starts without them, as a copy of torch's optimizers does."""
        return {k: v for k, v in self.__dict__.items()
                if k != "step" and not (k.startswith("_optimizer_") and k.endswith("_hooks"))}


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)
# Where this torch does not have them under these names, every step goes through torch's wrapper.
_GLOBAL_HOOKS = tuple(getattr(sys.modules[torch.optim.Optimizer.__module__], "_global_optimizer_" + n, (None,))
                      for n in ("pre_hooks", "post_hooks"))
_profiling = getattr(torch.autograd, "_profiler_enabled", lambda: True)
