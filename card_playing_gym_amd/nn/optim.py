"""The optimiser step of an update on the HIP path: the gradients' global norm and AdamW over
a model's tensors at once (csrc/optim.hip), moments in 32 bits or in 8-bit blocks.

After ``loss.backward()`` through the trunk (nn/train.py) an update clips the gradients by their
global norm and steps its optimiser (a fused Adam in cardgym/rl/trainer.py:392-395, which this is
with ``weight_decay=0``).  ``AdamW`` does both in one call with a handful of launches::

    optimizer = AdamW(model.parameters(), lr=3e-4, max_norm=1.0)
    loss.backward()
    optimizer.step()          # optimizer.norm: the gradients' norm, on the device

``AdamWPlan`` is the step without an optimiser around it, over parameters and state tensors
that the caller keeps.  The parameters' handles follow either: ``AdamW.step`` re-derives the
trunk's bf16 copies as any optimiser's does, ``AdamWPlan.step`` moves the version counters, so
the next eager call does.

Step counts live on the device and a step reads them there, so a captured step counts on at
every replay; a learning rate given as a device scalar is read at every replay too.  State is
made at a parameter's first gradient, so take one step before capturing one.

Moments in 8 bits take a quarter of the state's memory: blocks of 256 elements, each with a
float32 scale and a code per element whose value is within 6 % (rounded up or down at random, so
that averages stay where they belong).  Their random numbers come from ``seed``, the step count, the
tensor's place and the element's, so a run repeats bit for bit.
"""

from __future__ import annotations

import array
import ctypes
import operator
from contextlib import nullcontext
from typing import Iterable, Sequence

import torch
from torch.autograd.graph import increment_version

from .. import _native as nat
from .kv_cache import dtype_code, require_device, stream_handle

MOMENT_BLOCK = 256  # elements of a tensor that share a scale

_ptr = torch.Tensor.data_ptr
_numel = torch.Tensor.numel
_contiguous = torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")
_device_index = torch.Tensor.get_device  # -1 on the CPU


def moment_blocks(n: int) -> int:
    """Scales of the 8-bit moments of n elements."""

    return -(-n // MOMENT_BLOCK)


def _on(device: torch.device):
    """The device made current for a launch, where it is not."""

    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _addresses(values: Sequence[int]) -> array.array:
    return array.array("Q", values)


def _dense(grads: Sequence[torch.Tensor | None]) -> list[torch.Tensor | None]:
    """Contiguous gradients (copies of those that are not)."""

    out = []
    for g in grads:
        if g is not None and g.layout != torch.strided:
            raise ValueError("sparse gradients are not supported")
        out.append(g if g is None else g.detach().contiguous())
    return out


def _scalar(value: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if value.dtype != dtype or value.numel() != 1 or value.device != device:
        raise ValueError(f"{name} must be a {dtype} scalar on {device}")
    return value


def _on_host(lr) -> bool:
    return isinstance(lr, torch.Tensor) and lr.device.type == "cpu"


def grad_norm(grads: Iterable[torch.Tensor | None]) -> torch.Tensor:
    """The Euclidean norm of the gradients together (None: skipped), a float64 scalar on their
    device: the norm that ``torch.nn.utils.clip_grad_norm_`` clips by.  The squares are added in
    float64, so neither large nor tiny gradients lose it.  A constant: no derivative goes through it."""

    return _grad_norm(grads, None)


def _grad_norm(grads: Iterable[torch.Tensor | None], out: torch.Tensor | None) -> torch.Tensor:
    """``grad_norm``, into ``out`` where it is given."""

    grads = _dense([g for g in grads if g is not None])
    if not grads:
        raise ValueError("grad_norm needs at least one gradient")
    require_device(*grads)
    device = grads[0].device
    if any(g.device != device for g in grads):
        raise ValueError("gradients must be on one device")
    n = len(grads)
    dtypes = array.array("i", [dtype_code(g.dtype) for g in grads])
    pointers, sizes = _addresses([_ptr(g) for g in grads]), array.array("q", [_numel(g) for g in grads])
    norm = torch.empty((), device=device, dtype=torch.float64) if out is None else out
    size = nat.lib().cg_grad_norm_workspace_size(n)
    workspace = torch.empty(size, device=device, dtype=torch.uint8)
    with _on(device):
        nat.call("cg_grad_norm", pointers.buffer_info()[0], sizes.buffer_info()[0], dtypes.buffer_info()[0], n,
                 norm.data_ptr(), workspace.data_ptr(), size, stream_handle(device))
    return norm


def moment_values(codes: torch.Tensor, scales: torch.Tensor, signed: bool) -> torch.Tensor:
    """What 8-bit moments stand for, in float32: ``signed`` for ``exp_avg``'s codes (uint8 of any
    shape, with the scales of its blocks of 256 elements), not for ``exp_avg_sq``'s."""

    require_device(codes, scales)
    if codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous uint8 tensor")
    blocks = moment_blocks(codes.numel())
    if scales.dtype != torch.float32 or scales.shape != (blocks,) or not scales.is_contiguous() or (
            scales.device != codes.device):
        raise ValueError(f"scales must be contiguous float32 [{blocks}] on the codes' device")
    values = torch.empty(codes.shape, device=codes.device, dtype=torch.float32)
    with _on(codes.device):
        nat.call("cg_moment_values", codes.data_ptr(), scales.data_ptr(), int(bool(signed)), values.data_ptr(),
                 codes.numel(), stream_handle(codes.device))
    return values


def _check_apart(tensors: Iterable[torch.Tensor]) -> None:
    """The step writes every one of these: no two may share memory."""

    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    if any(begin < end for (_, end), (begin, _) in zip(spans, spans[1:])):
        raise ValueError("parameters and their state must not share memory (is a parameter listed twice?)")


class AdamWPlan:
    """AdamW over parameters and state that the caller keeps, checked once.

    ``params``: contiguous tensors of one type (float32, bfloat16 or float16) on one GPU.
    ``exp_avgs`` / ``exp_avg_sqs``: float32 of the parameters' sizes; or, with moments in 8 bits,
    uint8 codes of those sizes beside ``exp_avg_scales`` / ``exp_avg_sq_scales``, float32
    [ceil(size / 256)] each.  All zeros before the first step.  A gradient that is not finite spoils its
    element; with moments in 8 bits, its block.  (Blocks of gradients below 3e-18 lose their second moment in 8 bits:
    keep ``eps`` at 1e-16 or more.)  ``steps``: a float32 scalar each, the
    number of steps taken.  ``seed`` and ``first`` (the place of the first tensor) choose the 8-bit
    moments' random numbers.

    ``step`` updates all of them in place; a tensor without a gradient keeps its parameter, state
    and count.  The plan keeps the storage it was built over alive."""

    def __init__(
        self,
        params: Sequence[torch.Tensor],
        exp_avgs: Sequence[torch.Tensor],
        exp_avg_sqs: Sequence[torch.Tensor],
        steps: Sequence[torch.Tensor],
        *,
        exp_avg_scales: Sequence[torch.Tensor] | None = None,
        exp_avg_sq_scales: Sequence[torch.Tensor] | None = None,
        seed: int = 0,
        first: int = 0,
    ) -> None:
        self.params = list(params)
        if not self.params:
            raise ValueError("a plan needs at least one parameter")
        if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
            raise ValueError("moments in 8 bits need both lists of scales")
        self.state_bits = 32 if exp_avg_scales is None else 8
        kinds = [list(exp_avgs), list(exp_avg_sqs), list(steps)]
        if self.state_bits == 8:
            kinds += [list(exp_avg_scales), list(exp_avg_sq_scales)]
        if any(len(kind) != len(self.params) for kind in kinds):
            raise ValueError("every parameter needs its state: the lists differ in length")
        require_device(*self.params)
        self.device, self.dtype = self.params[0].device, self.params[0].dtype
        self._code = dtype_code(self.dtype)
        moment = torch.float32 if self.state_bits == 32 else torch.uint8
        for i, (p, m, v, t) in enumerate(zip(self.params, *kinds[:3])):
            if p.dtype != self.dtype or p.device != self.device:
                raise ValueError("a plan's parameters must be of one type on one device")
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
            for name, x in (("exp_avgs", m), ("exp_avg_sqs", v)):
                if x.dtype != moment or x.numel() != p.numel() or x.device != self.device or not x.is_contiguous():
                    raise ValueError(f"{name}[{i}] must be contiguous {moment} of its parameter's size and device")
            _scalar(t, f"steps[{i}]", torch.float32, self.device)
            for name, scales in zip(("exp_avg_scales", "exp_avg_sq_scales"), kinds[3:]):
                x, blocks = scales[i], moment_blocks(p.numel())
                if x.dtype != torch.float32 or x.shape != (blocks,) or x.device != self.device or not x.is_contiguous():
                    raise ValueError(f"{name}[{i}] must be contiguous float32 [{blocks}] on its parameter's device")
        if not 0 <= int(first) <= 2**31 - 1 - len(self.params):
            raise ValueError("first is out of range")
        _check_apart([x for kind in (self.params, *kinds) for x in kind])
        self.seed, self.first = int(seed) & 0xFFFFFFFF, int(first)
        self._device_index = self.params[0].get_device()
        self._shapes = [p.shape for p in self.params]
        self._addresses = list(map(_ptr, self.params))
        # Storage that the records below name, alive as long as they are (a captured step too).
        self._storage = [x.detach() for kind in (self.params, *kinds) for x in kind]
        self._tensors = (nat.AdamWTensor * len(self.params))()
        for i, (p, m, v, t) in enumerate(zip(self.params, *kinds[:3])):
            scales = [kind[i].data_ptr() for kind in kinds[3:]] or [None, None]
            self._tensors[i] = nat.AdamWTensor(p.data_ptr(), m.data_ptr(), v.data_ptr(), *scales, t.data_ptr(), p.numel())
        self._workspace_size = nat.lib().cg_adamw_workspace_size(len(self.params))

    def _gradient_addresses(self, grads: list[torch.Tensor | None]) -> tuple[array.array, list]:
        """Addresses of the gradients (0: none), and the tensors they are in."""

        if len(grads) != len(self.params):
            raise ValueError(f"{len(self.params)} parameters but {len(grads)} gradients")
        shapes, present = self._shapes, grads
        try:
            pointers = list(map(_ptr, grads))
        except (TypeError, RuntimeError):  # some are None, or sparse
            shapes = [shape for shape, g in zip(shapes, grads) if g is not None]
            present = [g for g in grads if g is not None]
            pointers = None
        if [g.shape for g in present] != shapes:
            raise ValueError("a gradient differs from its parameter in shape")
        # (sets of types and devices: quicker than comparing them one by one)
        if not set(map(_dtype, present)) <= {self.dtype} or not set(map(_device_index, present)) <= {self._device_index}:
            raise ValueError("a gradient differs from its parameter in type or device")
        try:
            dense = all(map(_contiguous, present))
        except RuntimeError:  # sparse layouts have no strides to ask for
            dense = False
        if not dense:
            grads, pointers = _dense(grads), None
        if pointers is None:
            pointers = [0 if g is None else _ptr(g) for g in grads]
        return _addresses(pointers), grads

    def step(
        self,
        grads: Sequence[torch.Tensor | None],
        *,
        lr: float | torch.Tensor,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        max_norm: float | None = None,
        norm: torch.Tensor | None = None,
    ) -> torch.Tensor | None:
        """One step with these gradients (None: skipped), the parameters' types and shapes.

        ``lr``: a number, or a float32 scalar on the device.  With ``max_norm`` the gradients are
        scaled by min(1, max_norm / (norm + 1e-6)): by ``norm`` (a float64 scalar, ``grad_norm``'s)
        where it is given, else by the norm of these gradients.  Returns the norm it clipped by."""

        if list(map(_ptr, self.params)) != self._addresses:
            raise ValueError("a parameter's data moved since the plan was built: build a new plan")
        return self._step(grads, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm, norm=norm)

    def _step(self, grads, *, lr, betas, eps, weight_decay, max_norm, norm, out=None) -> torch.Tensor | None:
        """``step`` with parameters that are where they were, its own norm written into ``out`` where that is given."""

        pointers, kept = self._gradient_addresses(list(grads))
        if norm is not None and max_norm is None:
            raise ValueError("norm is given without max_norm")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("max_norm must be non-negative")
        clip = nat.CG_CLIP_NONE
        if max_norm is not None:
            clip = nat.CG_CLIP_OWN_NORM if norm is None else nat.CG_CLIP_GIVEN_NORM
            if norm is None:
                norm = torch.empty((), device=self.device, dtype=torch.float64) if out is None else out
            else:
                _scalar(norm, "norm", torch.float64, self.device)
        config = nat.AdamWConfig(
            0.0, betas[0], betas[1], eps, weight_decay, max_norm or 0.0, None, self.seed, self.first, self._code,
            self.state_bits, clip,
        )
        if isinstance(lr, torch.Tensor):
            config.lr_device = _scalar(lr, "lr", torch.float32, self.device).data_ptr()
        else:
            config.lr = lr
        workspace = torch.empty(self._workspace_size, device=self.device, dtype=torch.uint8)
        with _on(self.device):
            nat.call("cg_adamw_step", self._tensors, pointers.buffer_info()[0], len(self.params), ctypes.byref(config),
                     None if norm is None else norm.data_ptr(), workspace.data_ptr(), self._workspace_size,
                     stream_handle(self.device))
        del kept
        increment_version(self.params)
        return norm


_STATE = {32: ("step", "exp_avg", "exp_avg_sq"),
          8: ("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (decoupled weight decay) with clipping by the global norm in the step.

    ``max_norm``: the norm of all groups' gradients together is clipped to it, as
    ``clip_grad_norm_`` before the step would; ``norm`` then holds the last step's norm (a float64
    device scalar; 0 of no gradients): a new one each step until a step is captured, from then on one that
    every step and replay writes.  ``state_bits``: 32, or 8 for moments in blocks of 256 (see
    :class:`AdamWPlan`).  A group's ``lr`` may be a float32 device scalar, which a captured step
    reads at every replay (its other options are captured as they are), or a scalar on the host, which is read
    at each step and not captured.

    Parameters must be contiguous and those of one group and type on one device, all of them with clipping.  No
    step is skipped for gradients that are not finite: with clipping a NaN among them makes every parameter NaN.

    ``state_dict`` has ``torch.optim.AdamW``'s layout, and with ``state_bits=32`` its state dicts
    load (not with options that this step lacks, as far as the dict tells: a coupled decay of ``torch.optim.Adam``
    shows only in dicts with ``decoupled_weight_decay``); 8-bit state holds codes (uint8) and
    ``exp_avg_scale`` / ``exp_avg_sq_scale``.  Loading copies into state, and a learning rate on the
    device, that is already there, so a captured step goes on with what was loaded.
    ``state``'s tensors are taken when a parameter joins: change them in place, or exchange them together with their
    parameter in its group."""

    def __init__(
        self,
        params,
        lr: float | torch.Tensor = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        max_norm: float | None = None,
        state_bits: int = 32,
        seed: int = 0,
    ) -> None:
        if state_bits not in _STATE:
            raise ValueError("state_bits must be 32 or 8")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("max_norm must be non-negative")
        self._options = {"max_norm": max_norm, "state_bits": int(state_bits), "seed": int(seed)}
        self._forget()
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    max_norm = property(lambda self: self._options["max_norm"])
    state_bits = property(lambda self: self._options["state_bits"])

    def _forget(self) -> None:
        self.norm: torch.Tensor | None = None
        self._norm_held: torch.Tensor | None = None  # what captured steps write, and those after them
        self._plans: list[tuple[int, AdamWPlan]] | None = None  # (group, plan); None: to be built
        self._captured: list[tuple] = []  # plans and learning rates: a graph's replays use what these hold
        self._planned: tuple | None = None  # what the plans were built over (_members)
        self._stateless: list[torch.Tensor] = []

    def __getstate__(self):
        return {**super().__getstate__(), "_options": self._options}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        if "_captured" not in self.__dict__:  # copied or unpickled
            self._forget()
        self._plans = None

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        lr, (beta1, beta2) = group["lr"], group["betas"]
        try:
            if not isinstance(lr, torch.Tensor) and not lr >= 0:
                raise ValueError(f"invalid learning rate {lr}")
            if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
                raise ValueError(f"betas must lie in [0, 1): {group['betas']}")
            if not group["eps"] >= 0 or not group["weight_decay"] >= 0:
                raise ValueError("eps and weight_decay must be non-negative")
        except ValueError:
            self.param_groups.pop()
            raise
        self._plans = None

    # -- state -----------------------------------------------------------------------------

    def _new_state(self, p: torch.Tensor) -> dict[str, torch.Tensor]:
        dtype = torch.float32 if self.state_bits == 32 else torch.uint8
        zeros = lambda shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=p.device)  # noqa: E731
        state = {"step": zeros(()), "exp_avg": zeros(p.shape, dtype), "exp_avg_sq": zeros(p.shape, dtype)}
        if self.state_bits == 8:
            blocks = (moment_blocks(p.numel()),)
            state |= {"exp_avg_scale": zeros(blocks), "exp_avg_sq_scale": zeros(blocks)}
        return state

    def load_state_dict(self, state_dict) -> None:
        # Between the caller's hooks: the dict is checked as the last pre-hook leaves it, before anything is loaded, and
        # the state is in place for the first post-hook.
        held = {p: self.state[p] for group in self.param_groups for p in group["params"] if self.state.get(p)}
        rates = [group["lr"] for group in self.param_groups]
        loaded: dict[torch.Tensor, dict] = {}
        hooks = [
            self.register_load_state_dict_pre_hook(lambda _, given: loaded.update(self._checked(given))),
            self.register_load_state_dict_post_hook(lambda _: self._place(loaded, held, rates), prepend=True),
        ]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
        self._plans = None

    def _checked(self, state_dict) -> dict[torch.Tensor, dict]:
        """The parameters' entries of a state dict, if its options and its state are this step's."""

        ours = [p for group in self.param_groups for p in group["params"]]
        theirs = [i for group in state_dict["param_groups"] for i in group["params"]]
        names = _STATE[self.state_bits]
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize") or (
                    group["weight_decay"] and not group.get("decoupled_weight_decay", True)):
                raise ValueError("the state dict's options (amsgrad, maximize, a coupled decay) are not this step's")
        loaded = {}
        for p, i in zip(ours, theirs):
            given = state_dict["state"].get(i)
            if not given:
                continue
            if any(name not in given for name in names) or ("exp_avg_scale" in given) != (self.state_bits == 8):
                raise ValueError(f"the state dict does not hold {self.state_bits}-bit AdamW state")
            shapes = {"step": None, "exp_avg": p.shape, "exp_avg_sq": p.shape,
                      "exp_avg_scale": (moment_blocks(p.numel()),), "exp_avg_sq_scale": (moment_blocks(p.numel()),)}
            for name in names:
                x = torch.as_tensor(given[name])
                if x.numel() != 1 if name == "step" else x.shape != shapes[name]:
                    raise ValueError(f"{name} of a parameter of shape {tuple(p.shape)} has shape {tuple(x.shape)}")
                if self.state_bits == 8 and name in ("exp_avg", "exp_avg_sq") and x.dtype != torch.uint8:
                    raise ValueError(f"{name} must hold uint8 codes")
            loaded[p] = given
        return loaded

    def _place(self, loaded: dict[torch.Tensor, dict], held: dict[torch.Tensor, dict], rates: list) -> None:
        """What was loaded, in the types of this state, into the state and the learning rates that were there."""

        for group, lr in zip(self.param_groups, rates):
            if isinstance(lr, torch.Tensor):
                lr.copy_(torch.as_tensor(group["lr"]).reshape(lr.shape))
                group["lr"] = lr
        for p, given in loaded.items():
            state = held.get(p) or self._new_state(p)
            for name in _STATE[self.state_bits]:
                state[name].copy_(torch.as_tensor(given[name]).reshape(state[name].shape))
            self.state[p] = state

    # -- the step --------------------------------------------------------------------------

    def _members(self) -> tuple:
        """The groups' parameters and how many have state, to tell a change by.  (All of them are kept alive by the
        plans or _stateless: no other takes an identity over.)"""

        return id(self.state), len(self.state), [list(map(id, group["params"])) for group in self.param_groups]

    def _build_plans(self) -> None:
        """A plan over the parameters with state, for each group and type."""

        plans, first = [], 0
        for index, group in enumerate(self.param_groups):
            by_type: dict[torch.dtype, list[torch.Tensor]] = {}
            for p in group["params"]:
                if self.state.get(p):
                    by_type.setdefault(p.dtype, []).append(p)
            for params in by_type.values():
                held = [[self.state[p][name] for p in params] for name in _STATE[self.state_bits]]
                scales = dict(zip(("exp_avg_scales", "exp_avg_sq_scales"), held[3:]))
                plans.append((index, AdamWPlan(params, held[1], held[2], held[0], **scales,
                                               seed=self._options["seed"], first=first)))
                first += len(params)
        self._plans = plans
        self._planned = self._members()
        self._stateless = [p for group in self.param_groups for p in group["params"] if not self.state.get(p)]

    def _norms(self, grads: list[list], capturing: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
        """For a step that clips: the norm of several plans' gradients, and the scalar that its norm goes to (None: a
        new one)."""

        gradient = next((g for many in grads for g in many if g is not None), None)
        tensors = (p for group in self.param_groups for p in group["params"]) if gradient is None else [gradient]
        device = next((t.device for t in tensors), None)
        if device is None:
            return None, None
        if capturing and self._norm_held is None:
            self._norm_held = torch.empty((), device=device, dtype=torch.float64)
        out = self._norm_held
        if out is not None and out.device != device:
            out = None
        if gradient is None:
            self.norm = (torch.empty((), device=device, dtype=torch.float64) if out is None else out).zero_()
        elif len(grads) > 1:
            return _grad_norm([g for many in grads for g in many], out), out
        return None, out

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter with a gradient; the closure's value, if there is one."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        stale = self._plans is None or self._planned != self._members() or any(
            list(map(_ptr, plan.params)) != plan._addresses for _, plan in self._plans)
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and any(_on_host(group["lr"]) for group in self.param_groups):
            raise RuntimeError("a learning rate on the host would stay as captured: give a device scalar, or a number")
        if stale:
            self._stateless = [p for group in self.param_groups for p in group["params"] if not self.state.get(p)]
        fresh = [p for p in self._stateless if p.grad is not None]
        if fresh:
            require_device(*fresh)
            if capturing:
                raise RuntimeError("AdamW state cannot be made inside a graph capture: take one step before it")
            for p in fresh:
                self.state[p] = self._new_state(p)
        if fresh or stale:
            self._build_plans()
        grads = [[p.grad for p in plan.params] for _, plan in self._plans]
        norm, out = (None, None) if self.max_norm is None else self._norms(grads, capturing)
        for (index, plan), many in zip(self._plans, grads):
            if all(g is None for g in many):
                continue
            group = self.param_groups[index]
            lr = float(group["lr"]) if _on_host(group["lr"]) else group["lr"]
            self.norm = plan._step(many, lr=lr, betas=group["betas"], eps=group["eps"],
                                   weight_decay=group["weight_decay"], max_norm=self.max_norm, norm=norm, out=out)
            if capturing and not any(plan is p and lr is rate for p, rate in self._captured):
                self._captured.append((plan, lr))
        return loss
