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
    params, grads = list(params), list(grads)
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
