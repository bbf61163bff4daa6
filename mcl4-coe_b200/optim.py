"""AdamW over the layer's many parameter tensors in one launch, with the moments in 32 or in
8 bits (``mcl4moe_adamw_step``).

``adamw_step`` is the operator on lists of tensors; ``AdamW`` the ``torch.optim`` optimizer
on it.  Both tell torch that the parameters changed (their version counters), which is what
the NVFP4 weight caches go by.
"""

from __future__ import annotations

import ctypes
from array import array
from operator import attrgetter
from typing import Sequence

import torch
from torch import Tensor

from . import _lib
from .nvfp4 import _ptr, _require_cuda
from .routing import DTYPE_CODES, _launch

STATE_BLOCK = 256  # elements of a tensor that share a scale of its 8-bit moments


_dtype_of = attrgetter("dtype")


def _check_list(name: str, tensors: Sequence[Tensor], dtype: torch.dtype, device: int, sizes: list[int]) -> array:
    """The tensors' addresses, after the checks (C-level maps: an optimizer step has hundreds of tensors)."""
    if len(tensors) != len(sizes):
        raise ValueError(f"{name}: {len(tensors)} tensors for {len(sizes)} parameters")
    if (list(map(Tensor.numel, tensors)) == sizes and set(map(_dtype_of, tensors)) == {dtype}
            and set(map(Tensor.get_device, tensors)) == {device} and all(map(Tensor.is_contiguous, tensors))):
        return array("Q", list(map(Tensor.data_ptr, tensors)))
    for i, (t, n) in enumerate(zip(tensors, sizes)):
        if t.dtype != dtype or t.get_device() != device or not t.is_contiguous() or t.numel() != n:
            raise ValueError(f"{name}[{i}] must be {n} contiguous {dtype} elements on the first parameter's device, got "
                             f"{t.numel()} of {t.dtype} on {t.device}")
    raise AssertionError(name)


@torch.no_grad()
def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], *, step: int | Tensor, lr: float | Tensor = 1e-3,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               exp_avg_scales: Sequence[Tensor] | None = None, exp_avg_sq_scales: Sequence[Tensor] | None = None,
               masters: Sequence[Tensor] | None = None, grad_scale: Tensor | None = None, seed: int = 0,
               indices: Sequence[int] | None = None) -> None:
    """One AdamW step over lists of tensors, in place::

        g = grad * grad_scale
        m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^step) m / (sqrt(v / (1 - beta2^step)) + eps)

    ``params`` (one type: bf16, fp16 or fp32) and ``grads`` (one type) are contiguous;
    ``masters`` (fp32) take the update where they are given, and the parameters their
    rounded values.  fp32 ``exp_avgs`` / ``exp_avg_sqs`` are 32-bit moments.  With
    ``exp_avg_scales`` and ``exp_avg_sq_scales`` (fp32, one for each 256 elements) the
    moments are 8 bits, float8_e4m3fn and float8_e5m2 times their scale, a power of
    two; they are rounded stochastically with noise that ``seed``, the step and the
    tensor's place in the list (or ``indices``) alone decide.  ``step`` counts from 1;
    ``step`` (int64) and ``lr`` (fp32) may be device scalars, read when the kernel
    runs.  ``grad_scale`` (fp32 device scalar) is what clipping multiplies gradients
    with.  A moment that is not finite is NaN in 8 bits, its block's others stay.
    """
    params, grads, exp_avgs, exp_avg_sqs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    exp_avg_scales, exp_avg_sq_scales, masters = (None if t is None else list(t)
                                                  for t in (exp_avg_scales, exp_avg_sq_scales, masters))
    if len(grads) != len(params):
        raise ValueError(f"{len(grads)} gradients for {len(params)} parameters")
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None):
        raise ValueError("8-bit moments need exp_avg_scales and exp_avg_sq_scales")
    beta1, beta2 = betas
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if not isinstance(step, Tensor) and int(step) < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not params:
        return
    first = params[0]
    dev = first.device
    if first.dtype not in DTYPE_CODES or grads[0].dtype not in DTYPE_CODES:
        raise ValueError(f"parameters and gradients must be bf16, fp16 or fp32, got {first.dtype} and {grads[0].dtype}")
    index, sizes = first.get_device(), list(map(Tensor.numel, params))
    if not all(map(Tensor.is_contiguous, grads)):
        grads = [g.contiguous() for g in grads]
    moments = (torch.float8_e4m3fn, torch.float8_e5m2) if eight else (torch.float32, torch.float32)
    written = dict(params=params, exp_avgs=exp_avgs, exp_avg_sqs=exp_avg_sqs)
    at = dict(params=_check_list("params", params, first.dtype, index, sizes),
              exp_avgs=_check_list("exp_avgs", exp_avgs, moments[0], index, sizes),
              exp_avg_sqs=_check_list("exp_avg_sqs", exp_avg_sqs, moments[1], index, sizes))
    if eight:
        blocks = [-(-n // STATE_BLOCK) for n in sizes]
        for name, tensors in (("exp_avg_scales", exp_avg_scales), ("exp_avg_sq_scales", exp_avg_sq_scales)):
            at[name] = _check_list(name, tensors, torch.float32, index, blocks)
            written[name] = tensors
    if masters is not None:
        at["masters"] = _check_list("masters", masters, torch.float32, index, sizes)
        written["masters"] = masters
    places = [p for a in at.values() for p in a if p]  # an empty tensor has no address
    if len(set(places)) != len(places):
        raise ValueError("a tensor is in the lists twice")
    at["grads"] = _check_list("grads", grads, grads[0].dtype, index, sizes)
    for name, t, dtype in (("step", step, torch.int64), ("lr", lr, torch.float32), ("grad_scale", grad_scale, torch.float32)):
        if isinstance(t, Tensor) and (t.dtype != dtype or t.numel() != 1 or t.device != dev):
            raise ValueError(f"{name} as a tensor must be one {dtype} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if indices is not None and len(indices) != len(params):
        raise ValueError(f"{len(indices)} indices for {len(params)} parameters")
    _require_cuda(first, "adamw_step")
    args = _lib.AdamwArgs(n=len(params), param_dtype=DTYPE_CODES[first.dtype],
                          grad_dtype=DTYPE_CODES[grads[0].dtype], bits=8 if eight else 32, beta1=beta1, beta2=beta2,
                          eps=eps, weight_decay=weight_decay, seed=int(seed) & 0xFFFFFFFFFFFFFFFF)
    at["numels"] = array("q", sizes)
    for name, a in at.items():
        setattr(args, name, a.buffer_info()[0])
    if indices is not None:
        at["indices"] = array("i", indices)
        args.indices = at["indices"].buffer_info()[0]
    if isinstance(step, Tensor):
        args.step_dev = step.data_ptr()
    else:
        args.step = int(step)
    if isinstance(lr, Tensor):
        args.lr_dev = lr.data_ptr()
    else:
        args.lr = float(lr)
    args.grad_scale = _ptr(grad_scale)
    _launch(dev, "mcl4moe_adamw_step", _lib.load().mcl4moe_adamw_step, ctypes.byref(args))
    torch.autograd.graph.increment_version([t for tensors in written.values() for t in tensors])


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one ``adamw_step`` call per parameter group, device and pair of types.

    ``state_bits`` 8 keeps the moments in 8 bits (``adamw_step`` says how), which takes
    2.03 instead of 8 bytes a parameter; ``master_weights`` gives bf16 / fp16 parameters
    float32 masters.  ``step(grad_scale=t)`` multiplies the gradients by the device scalar
    ``t`` (clipping).  ``lr`` may be a float32 tensor on the parameters' device.

    ``capturable`` keeps one step count per group and device in device memory, so that a
    captured step goes on counting when it is replayed.  A capture needs it, and an eager step
    before, which makes the state.  A replay does not go through torch,
    so the parameters' versions stand still and an NVFP4 weight cache has to be told
    (``invalidate_cache``).
    """

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False, seed: int = 0,
                 capturable: bool = False) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not isinstance(lr, Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=master_weights, seed=int(seed),
                                      capturable=bool(capturable)))

    def _new_state(self, p: Tensor, group: dict) -> dict:
        if not p.is_contiguous():
            raise ValueError("AdamW takes contiguous parameters")
        state: dict = {"step": 0}
        if group["state_bits"] == 8:
            blocks = -(-p.numel() // STATE_BLOCK)
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float8_e5m2)
            state["exp_avg_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
            state["exp_avg_sq_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
        else:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32)
        return state

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            self._check_capture()
        place = 0  # a parameter's number in the optimizer keys its noise
        for group in self.param_groups:
            calls: dict = {}
            if "step_counts" in group and not group["capturable"]:
                self._host_counts(group)
            for p in group["params"]:
                place += 1
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW takes dense gradients")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                if not group["capturable"]:
                    state["step"] += 1
                key = (p.device, p.dtype, p.grad.dtype, state["step"], "master" in state)
                calls.setdefault(key, []).append((p, state, place - 1))
            counts = self._device_counts(group, calls)
            for (device, _, _, step, master), items in calls.items():
                states = [s for _, s, _ in items]
                eight = group["state_bits"] == 8
                adamw_step([p for p, _, _ in items], [p.grad for p, _, _ in items],
                           [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                           step=counts[device] if counts else step, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                           exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None,
                           masters=[s["master"] for s in states] if master else None, grad_scale=grad_scale,
                           seed=group["seed"], indices=[i for _, _, i in items])
        return loss

    def _check_capture(self) -> None:
        """What a replay could not repeat: a step count on the host would stay at its value, and state made
        during the capture would be made again by each replay."""
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not group["capturable"]:
                    raise RuntimeError("a captured AdamW step needs capturable=True")
                if not self.state.get(p) or str(p.device) not in group.get("step_counts", {}):
                    raise RuntimeError("an AdamW step can be captured once an eager one has made the parameters' state")

    def _device_counts(self, group: dict, calls: dict) -> dict | None:
        """capturable: the group's step count on each device, moved on by one.  A group whose ``capturable``
        was changed (a checkpoint brings its own) goes on from where its other kind of count stood."""
        if not group["capturable"]:
            return None
        counts = group.setdefault("step_counts", {})
        for device in {key[0] for key in calls}:
            if str(device) not in counts:
                before = {s["step"] for key, items in calls.items() if key[0] == device for _, s, _ in items}
                if len(before) != 1:
                    raise ValueError(f"capturable keeps one step count, these parameters have {sorted(before)}")
                counts[str(device)] = torch.full((), *before, dtype=torch.int64, device=device)
            counts[str(device)] += 1
        return {key[0]: counts[str(key[0])] for key in calls}

    def _host_counts(self, group: dict) -> None:
        """Not capturable (any more): the counts that lived on the devices, for each parameter."""
        counts = {d: int(t) for d, t in group.pop("step_counts").items()}
        for p in group["params"]:
            if self.state.get(p) and str(p.device) in counts:
                self.state[p]["step"] = counts[str(p.device)]

    def load_state_dict(self, state_dict: dict) -> None:
        """As ``torch.optim.Optimizer``'s, which would cast the moments to the parameters' type."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, Tensor):
                    self.state[p][name] = value.detach().to(p.device, copy=True)
        for group in self.param_groups:
            devices = {str(p.device): p.device for p in group["params"]}
            if "step_counts" in group:
                group["step_counts"] = _placed_counts(group["step_counts"], devices)
            if isinstance(group["lr"], Tensor) and len(devices) == 1:
                group["lr"] = group["lr"].to(*devices.values())


def _placed_counts(saved: dict, devices: dict) -> dict:
    """A group's saved step counts on the devices that its parameters have now: by name where every saved
    device is among them, else (a checkpoint of another rank) the one value that all of them hold."""
    if set(saved) <= set(devices):
        return {d: t.detach().to(devices[d], copy=True) for d, t in saved.items()}
    values = {int(t) for t in saved.values()}
    if len(values) != 1:
        raise ValueError(f"the saved step counts {saved} do not say which holds for parameters on {sorted(devices)}")
    return {d: torch.full((), *values, dtype=torch.int64, device=device) for d, device in devices.items()}
