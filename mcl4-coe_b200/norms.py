"""The norms before and after a block, its gate and the residual sum, in one kernel each way
(``mcl4moe_residual_norm``): what stands around ``SparseMoE`` in a layer,
``x + moe(moe_norm(x))`` (src/mcl4_coe/backbone.py:1269, RMSNorm src/mcl4_coe/ple.py:17).
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .nvfp4 import _ptr, _require_cuda
from .routing import DTYPE_CODES, _f32, _launch, _ld, _refuse_tangents, _rows

GATE_ACTIVATIONS = ("none", "sigmoid", "tanh")
MAX_COLS = 16384
_NONE, _CHANNEL, _ROW, _FULL = range(4)
# Rows from which a gate shared by consecutive rows is summed inside the kernel (one partial
# row of column sums per group); smaller groups are written out as one gate row per row.
_MIN_GROUP_ROWS = 32
_MAX_GROUPS = 65533


def _gate_form(gate: Tensor, x: Tensor) -> tuple[Tensor, int, int, torch.Size | None]:
    """(gate, mode, rows that share a gate row, None) for a gate that broadcasts to ``x``.  A 16-bit gate's
    gradient is rounded where its rows are added up, not before: a gate of single values goes in as float32,
    one that has to be written out a row each stays as it is, with ``x``'s shape in the last place, for the
    autograd function to do that and to add up the rows of a float32 gradient."""
    if gate.ndim == 1 and gate.shape[0] == x.shape[-1]:
        return gate.contiguous().view(1, -1), _CHANNEL, max(1, x.numel() // x.shape[-1]), None
    if gate.ndim > x.ndim or any(g != 1 and g != s for g, s in zip(gate.shape[::-1], x.shape[::-1])):
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
    gate = gate.reshape((1,) * (x.ndim - gate.ndim) + tuple(gate.shape))
    lead, x_lead, d = gate.shape[:-1], x.shape[:-1], x.shape[-1]
    rows = x.numel() // max(1, d)
    if lead == x_lead and gate.shape[-1] == d and rows > 1:
        return _rows(gate), _FULL, 1, None
    summed = gate.dtype != torch.float32 and gate.requires_grad and torch.is_grad_enabled()
    if gate.shape[-1] == 1 and d > 1:
        if summed and gate.numel() != rows:
            gate = gate.float()
        return gate.expand(*x_lead, 1).reshape(rows).contiguous(), _ROW, 1, None
    cut = max((i + 1 for i, s in enumerate(lead) if s != 1), default=0)
    groups = 1
    for s in lead[:cut]:
        groups *= s
    if lead[:cut] == x_lead[:cut]:
        share = max(1, rows // max(1, groups))
        if groups == 1 or (share >= _MIN_GROUP_ROWS and groups <= _MAX_GROUPS):
            return gate.reshape(groups, d).contiguous(), _CHANNEL, share, None
    return (gate, _FULL, 1, x.shape) if summed else (_spread(gate, x.shape), _FULL, 1, None)


def _spread(gate: Tensor, shape: torch.Size) -> Tensor:
    return gate.expand(shape).reshape(-1, shape[-1]).contiguous()


def _fill(args, x, branch, post, pre, gate, mode, gate_rows, act, norm_dtype, scales):
    args.rows, args.cols = x.shape
    args.x, args.ld_x, args.x_dtype = x.data_ptr(), _ld(x), DTYPE_CODES[x.dtype]
    if branch is not None:
        args.branch, args.ld_branch, args.branch_dtype = branch.data_ptr(), _ld(branch), DTYPE_CODES[branch.dtype]
    args.post_weight, args.pre_weight = _ptr(post), _ptr(pre)
    if gate is not None:
        args.gate, args.gate_dtype, args.gate_mode = gate.data_ptr(), DTYPE_CODES[gate.dtype], mode
        args.gate_rows, args.gate_act = gate_rows, act
        args.ld_gate = _ld(gate) if mode == _FULL else 0
    args.norm_dtype = DTYPE_CODES[norm_dtype]
    args.residual_scale, args.branch_scale, args.eps = scales
    return args


def _norm_forward(x, branch, post, pre, gate, mode, gate_rows, act, norm_dtype, scales, stats=None):
    y = None if branch is None else x.new_empty(x.shape)
    h = None if pre is None else x.new_empty(x.shape, dtype=norm_dtype)
    if x.shape[0] == 0:
        return y, h
    args = _fill(_lib.NormArgs(), x, branch, post, pre, gate, mode, gate_rows, act, norm_dtype, scales)
    args.stream_out, args.norm_out, args.stats = _ptr(y), _ptr(h), _ptr(stats)
    _launch(x.device, "mcl4moe_residual_norm", _lib.load().mcl4moe_residual_norm, args)
    return y, h


class _ResidualNorm(torch.autograd.Function):
    """Saves the inputs and the rows' two reciprocal root mean squares; the backward computes the rest again."""

    @staticmethod
    def forward(ctx, x, branch, post, pre, gate, form, gate_shape):
        ctx.gate_of = None if gate_shape is None else gate.shape  # what the gradient's rows are added up to
        ctx.x_shape = gate_shape
        if gate_shape is not None:
            gate = _spread(gate, gate_shape)
        stats = x.new_empty((x.shape[0], 2), dtype=torch.float32)
        y, h = _norm_forward(x, branch, post, pre, gate, *form, stats)
        ctx.save_for_backward(x, branch, post, pre, gate, stats)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, d_y, d_h):
        if torch.is_grad_enabled():  # create_graph: a second differentiation has to be refused
            return _ResidualNorm._once(ctx, d_y, d_h)
        return _ResidualNorm._gradients(ctx, d_y, d_h)

    @staticmethod
    @once_differentiable
    def _once(ctx, d_y, d_h):
        return _ResidualNorm._gradients(ctx, d_y, d_h)

    @staticmethod
    def _gradients(ctx, d_y, d_h):
        if d_y is None and d_h is None:
            return (None,) * 7
        x, branch, post, pre, gate, stats = ctx.saved_tensors
        mode = ctx.form[0]
        need = ctx.needs_input_grad
        if x.shape[0] == 0:
            like = (x, branch, post, pre, gate if ctx.gate_of is None else gate.new_empty(ctx.gate_of))
            return tuple(torch.zeros_like(t) if n and t is not None else None for n, t in zip(need, like)) + (None, None)
        lib = _lib.load()
        dev = x.device
        args = _fill(_lib.NormArgs(), x, branch, post, pre, gate, *ctx.form)
        args.stats = stats.data_ptr()
        if d_y is not None:
            d_y = _rows(d_y)
            args.d_stream, args.ld_d_stream = d_y.data_ptr(), _ld(d_y)
        if d_h is not None:
            d_h = _rows(d_h)
            args.d_normed, args.ld_d_normed = d_h.data_ptr(), _ld(d_h)

        def out(wanted, like, attr, dtype=None):
            if like is None or not wanted:
                return None
            t = torch.empty_like(like) if dtype is None and like.is_contiguous() else \
                x.new_empty(like.shape, dtype=dtype or like.dtype)
            setattr(args, attr, t.data_ptr())
            return t

        d_x = out(need[0], x, "d_x")
        d_branch = out(need[1], branch, "d_branch")
        d_post = out(need[2], post, "d_post")
        d_pre = out(need[3], pre, "d_pre")
        args.gate_grad_f32 = int(ctx.gate_of is not None)
        d_gate = out(need[4], gate, "d_gate", None if mode == _FULL and ctx.gate_of is None else torch.float32)
        ws, nbytes = None, 0
        if d_post is not None or d_pre is not None or (d_gate is not None and mode == _CHANNEL):
            nbytes = lib.mcl4moe_residual_norm_workspace_size(args.rows, args.cols, args.gate_mode, args.gate_rows)
            ws = x.new_empty((nbytes,), dtype=torch.uint8)
        _launch(dev, "mcl4moe_residual_norm_backward", lib.mcl4moe_residual_norm_backward, args, _ptr(ws), nbytes)
        if d_gate is not None and ctx.gate_of is not None:
            d_gate = d_gate.view(ctx.x_shape).sum_to_size(ctx.gate_of)
        if d_gate is not None and d_gate.dtype != gate.dtype:
            d_gate = d_gate.to(gate.dtype)
        return d_x, d_branch, d_post, d_pre, d_gate, None, None


def residual_norm(x: Tensor, branch: Tensor | None = None, *, post_weight: Tensor | None = None,
                  gate: Tensor | None = None, gate_activation: str = "none", pre_weight: Tensor | None = None,
                  residual_scale: float = 1.0, branch_scale: float = 1.0, eps: float = 1e-6,
                  norm_dtype: torch.dtype | None = None) -> tuple[Tensor, Tensor | None]:
    """Adds a block's output to the residual stream and norms the sum for the next block.

    ``(y, h)`` with RMS norms over the last dimension::

        n = branch * rsqrt(mean(branch^2) + eps) * post_weight    (n = branch without it)
        y = residual_scale * x + branch_scale * act(gate) * n     (no gate: 1)
        h = y * rsqrt(mean(y^2) + eps) * pre_weight               (None without it)

    ``residual_norm(x, pre_weight=w)`` is the norm before the first block: ``(x, h)``.
    ``x`` and ``branch`` have one shape ``[.., d]`` (d <= 16384) and may differ in type
    (bf16, fp16, fp32): ``y`` has ``x``'s type, ``h`` ``norm_dtype`` (default: the
    branch's, else ``x``'s).  The weights are ``[d]``; ``gate`` broadcasts to ``x``
    (one value for each channel, token or element, or one row for each sequence) and
    goes through ``gate_activation`` ("none", "sigmoid", "tanh").  Arithmetic is fp32,
    each output is rounded once.  Every tensor gets its gradient; differentiable once, in reverse mode.
    """
    if gate_activation not in GATE_ACTIVATIONS:
        raise ValueError(f"gate_activation must be one of {GATE_ACTIVATIONS}, got {gate_activation!r}")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"x must have a last dimension of 1 to {MAX_COLS}, got {tuple(x.shape)}")
    if branch is None:
        if post_weight is not None or gate is not None or residual_scale != 1.0 or branch_scale != 1.0:
            raise ValueError("post_weight, gate and the scales need a branch")
        if pre_weight is None:
            raise ValueError("residual_norm without a branch needs pre_weight")
    elif branch.shape != x.shape:
        raise ValueError(f"branch {tuple(branch.shape)} and x {tuple(x.shape)} must have one shape")
    d, dev = x.shape[-1], x.device
    for name, t in (("x", x), ("branch", branch), ("gate", gate)):
        if t is not None and (t.dtype not in DTYPE_CODES or t.device != dev):
            raise ValueError(f"{name} must be bf16, fp16 or fp32 on {dev}, got {t.dtype} on {t.device}")
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and (t.shape != (d,) or t.device != dev):
            raise ValueError(f"{name} must be [{d}] on {dev}, got {tuple(t.shape)} on {t.device}")
    if norm_dtype is None:
        norm_dtype = x.dtype if branch is None else branch.dtype
    elif norm_dtype not in DTYPE_CODES:
        raise ValueError(f"norm_dtype must be bf16, fp16 or fp32, got {norm_dtype}")
    mode, gate_rows, gate_2d, gate_shape = _NONE, 0, None, None
    if gate is not None:
        gate_2d, mode, gate_rows, gate_shape = _gate_form(gate, x)
    _refuse_tangents("residual_norm", x, branch, post_weight, pre_weight, gate)
    _require_cuda(x, "residual_norm")
    tensors = (_rows(x), None if branch is None else _rows(branch), _f32(post_weight), _f32(pre_weight), gate_2d)
    form = (mode, gate_rows, GATE_ACTIVATIONS.index(gate_activation), norm_dtype,
            (float(residual_scale), float(branch_scale), float(eps)))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        y, h = _ResidualNorm.apply(*tensors, form, gate_shape)
    else:
        y, h = _norm_forward(*tensors, *form)
    if x.ndim != 2:
        y, h = (None if t is None else t.view(x.shape) for t in (y, h))
    return (x if branch is None else y), h
