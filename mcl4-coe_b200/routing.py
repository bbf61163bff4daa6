"""Routing from router scores: softmax or sigmoid, a balance bias, expert groups, top-k,
renormalised and scaled weights, with the gradient (``mcl4moe_route_scores``).

``SparseMoE`` uses it for every configuration beyond the reference's plain softmax
top-k (``MoEConfig.score_function``, ``expert_groups``, ``balance_bias``, ...); the
plain path keeps the fused router of ``mcl4moe_moe_forward``.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .nvfp4 import _ptr, _raw_stream, _require_cuda

DTYPE_CODES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
SCORE_FUNCTIONS = ("softmax", "sigmoid")
GROUP_SCORES = ("top2", "max")
MAX_EXPERTS, MAX_TOP_K = 512, 32


def _launch(device: torch.device, what: str, fn, *args) -> None:
    """One library call on ``device``'s current stream (``device`` need not be the current one)."""
    index = device.index
    if index == torch.cuda.current_device():
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _raw_stream(index))
    if st != _lib.OK:
        _lib.check(st, what)


def _rows(t: Tensor) -> Tensor:
    """``t`` as rows [n, last] whose elements are next to each other and whose rows do not overlap."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _refuse_tangents(what: str, *tensors: Tensor | None) -> None:
    """Forward-mode derivatives, which the kernels would drop without a word."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of a dual level no tensor has a tangent
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _f32(t: Tensor | None) -> Tensor | None:
    """``t`` as contiguous float32 (differentiably)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def _ld(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _route_forward(logits, k, score, bias, groups, top_groups, group_score, renorm, scale, valid):
    n, E = logits.shape
    idx = logits.new_empty((n, k), dtype=torch.int32)
    w = logits.new_empty((n, k), dtype=torch.float32)
    counts = logits.new_empty((E,), dtype=torch.int32)
    _launch(logits.device, "mcl4moe_route_scores", _lib.load().mcl4moe_route_scores, logits.data_ptr(),
            DTYPE_CODES[logits.dtype], _ld(logits), _ptr(bias), _ptr(valid), n, E, k, score, groups, top_groups,
            group_score, renorm, scale, idx.data_ptr(), w.data_ptr(), counts.data_ptr())
    return w, idx, counts


class _RouteScores(torch.autograd.Function):
    """The weights as a function of the logits; the ids and counts leave through ``box`` (outputs that
    autograd need not know of)."""

    @staticmethod
    def forward(ctx, logits, args, box):
        w, idx, counts = _route_forward(logits, *args)
        ctx.save_for_backward(logits, idx)
        ctx.args = args
        ctx.set_materialize_grads(False)
        box += (idx, counts)
        return w

    @staticmethod
    def backward(ctx, d_w):
        if torch.is_grad_enabled():  # create_graph: a second differentiation has to be refused
            return _RouteScores._once(ctx, d_w)
        return _RouteScores._gradients(ctx, d_w)

    @staticmethod
    def _gradients(ctx, d_w):
        if d_w is None:
            return None, None, None
        logits, idx = ctx.saved_tensors
        k, score, _, _, _, _, renorm, scale, _ = ctx.args
        n, E = logits.shape
        d_w = _f32(d_w)
        d_logits = logits.new_empty((n, E))
        _launch(logits.device, "mcl4moe_route_scores_backward", _lib.load().mcl4moe_route_scores_backward,
                logits.data_ptr(), DTYPE_CODES[logits.dtype], _ld(logits), idx.data_ptr(), d_w.data_ptr(), n, E, k,
                score, renorm, scale, d_logits.data_ptr())
        return d_logits, None, None

    @staticmethod
    @once_differentiable
    def _once(ctx, d_w):
        return _RouteScores._gradients(ctx, d_w)


def route_experts(logits: Tensor, top_k: int, *, score: str = "softmax", bias: Tensor | None = None,
                  num_groups: int = 1, top_groups: int | None = None, group_score: str = "top2",
                  renormalize: bool = True, scale: float = 1.0,
                  valid: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """Experts of each token from its router logits ``[.., E]`` (bf16, fp16 or fp32).

    Returns ``(weights, ids, counts)``: fp32 ``[.., top_k]`` weights
    ``scale * s / (sum of the chosen s if renormalize)`` with ``s`` the softmax or
    sigmoid of the logits; int32 ``[.., top_k]`` ids, best first, ties to the lower id;
    int32 ``[E]`` slots of each expert.  ``bias`` (``[E]``) is added to the scores for
    the selection alone and gets no gradient.  With ``num_groups`` > 1 (groups of
    consecutive experts) only the ``top_groups`` groups with the best value are
    searched: the sum of a group's two best keys (``"top2"``; a group with one unmasked
    expert counts that one) or its best (``"max"``).

    An expert whose logit or bias is ``-inf`` is masked: never chosen, and a row that
    runs out of experts has id -1 and weight 0 in its last slots, as have rows whose
    ``valid`` (``[..]``) is false.  NaN ranks first and makes its row's weights NaN; so
    does +inf under a softmax.
    ids follow exact arithmetic on the given logits (near ties are decided in float64).
    The gradient reaches the logits through the weights; differentiable once, in reverse mode.
    """
    if logits.ndim < 1 or logits.dtype not in DTYPE_CODES:
        raise ValueError(f"logits must be bf16, fp16 or fp32 rows, got {logits.dtype} {tuple(logits.shape)}")
    if score not in SCORE_FUNCTIONS:
        raise ValueError(f"score must be one of {SCORE_FUNCTIONS}, got {score!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score must be one of {GROUP_SCORES}, got {group_score!r}")
    E = logits.shape[-1]
    top_k, num_groups = int(top_k), int(num_groups)
    if not 1 <= E <= MAX_EXPERTS or top_k > MAX_TOP_K:
        raise ValueError(f"route_experts takes 1 to {MAX_EXPERTS} experts and a top_k up to {MAX_TOP_K}, got {E} and {top_k}")
    top_groups = num_groups if top_groups is None else int(top_groups)
    if num_groups < 1 or E % num_groups != 0 or not 1 <= top_groups <= num_groups:
        raise ValueError(f"{E} experts do not form {num_groups} equal groups of which {top_groups} stay open")
    if not 1 <= top_k <= top_groups * (E // num_groups):
        raise ValueError(f"top_k {top_k} is outside 1 to {top_groups * (E // num_groups)}, the experts that stay open")
    if top_groups == num_groups:
        num_groups = top_groups = 1  # every group stays open
    dev = logits.device
    if bias is not None:
        if bias.shape != (E,) or bias.device != dev:
            raise ValueError(f"bias must have one entry per expert on {dev}, got {tuple(bias.shape)} on {bias.device}")
        bias = _f32(bias.detach())
    if valid is not None:
        if valid.shape != logits.shape[:-1] or valid.device != dev:
            raise ValueError("valid must have one entry per token on the logits' device")
        if valid.dtype != torch.bool:
            valid = valid != 0
        valid = valid.contiguous()
    _refuse_tangents("route_experts", logits)
    _require_cuda(logits, "route_experts")
    lead = logits.shape[:-1]
    rows = _rows(logits)
    args = (top_k, SCORE_FUNCTIONS.index(score), bias, num_groups, top_groups, GROUP_SCORES.index(group_score),
            int(bool(renormalize)), float(scale), valid)
    if torch.is_grad_enabled() and logits.requires_grad:
        box: list = []
        w = _RouteScores.apply(rows, args, box)
        idx, counts = box
    else:
        w, idx, counts = _route_forward(rows, *args)
    if len(lead) != 1:
        w, idx = w.view(*lead, top_k), idx.view(*lead, top_k)
    return w, idx, counts
