"""Group norm with an activation on channels-last tensors, forward and backward (csrc/group_norm.hip).

``forward(x, groups, weight, bias, act, eps) -> (y, stats)`` and ``backward(dy, x, stats, groups, weight, bias, act) -> (dx, dweight,
dbias)`` are the two passes; ``group_norm_act(...)`` records them for autograd.  x is (N, ..., C) in float32, bfloat16 or float16 with
any row pitch (a channel slice of a wider buffer; an NCHW tensor in channels_last memory as ``x.permute(0, 2, 3, 1)``); the
statistics of a group are taken over the middle dimensions and the group's C / groups channels.  weight, bias: (C,) float32 or
None.  act: ACT_NONE, ACT_RELU, ACT_LRELU (0.1), ACT_SIGMOID, ACT_TANH, ACT_GELU (erf) or ACT_SILU of ``gimmvfi_hip.lib``.
Outputs are contiguous, in x's type; stats is (N, groups, 2) float32: mean and 1 / sqrt(var + eps).  Values and derivatives of the
activations are accurate relative to themselves, to a few steps of float for float32 and to 2**-16 before the rounding for 16 bits.

Both passes can be captured into a graph.  The autograd form refuses leaves that require gradients during a capture (rows.py says
why).
"""
import math

import torch

from . import lib as L
from . import rows

ACTS = (L.ACT_NONE, L.ACT_RELU, L.ACT_LRELU, L.ACT_SIGMOID, L.ACT_TANH, L.ACT_GELU, L.ACT_SILU)

LAUNCH = 1 << 23        # (image, group) pairs below which one launch stays, seven images rounded up; larger batches go out in several


def _batches(n, c, groups):
    """(first image, images) of every call: as many as the library takes in one."""
    step = min((LAUNCH - 1) // groups - 7, LAUNCH - 1, 128 * ((1 << 24) // ((c + 15) // 16) - 1))
    if n <= step or step < 1:
        return ((0, n),)
    return [(lo, min(step, n - lo)) for lo in range(0, n, step)]


def _sizes(x, groups, act, name):
    if x.dim() < 2:
        raise ValueError(f"{name} must be (N, ..., C), got shape {tuple(x.shape)}")
    if act not in ACTS:
        raise ValueError(f"activation {act} has no group norm form")
    n, c = x.shape[0], x.shape[-1]
    if groups < 1 or c < 1 or c % groups or c > 1 << 24:
        raise ValueError(f"{c} channels (at most 2**24) cannot be split into {groups} groups")
    return n, math.prod(x.shape[1:-1]), c


def forward(x, groups, weight=None, bias=None, act=L.ACT_NONE, eps=1e-5, out=None):
    """out: tensor of x's shape and type to write (rows of one pitch; must not overlap x); None: a new one."""
    lib = rows.library(x, "x")
    dt = rows.dtype_of(x, "x")
    n, hw, c = _sizes(x, groups, act, "x")
    if out is None:
        out = rows.new_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.get_device() != x.get_device():
        raise ValueError("out must have x's shape, type and device")
    w, b = rows.check_vector(weight, c, x, "weight"), rows.check_vector(bias, c, x, "bias")
    ldx, ldy = rows.pitch_of(x, "x"), rows.pitch_of(out, "out")
    stats = x.new_empty((n, groups, 2), dtype=torch.float32)
    if x.numel() == 0:
        return out, stats.zero_()
    es = x.element_size()
    for lo, k in _batches(n, c, groups):
        ws = rows.workspace(x, lib.group_norm_workspace, "group_norm", c, groups, k, hw)
        rows.launch(lib.group_norm, x, "group_norm", x.data_ptr() + lo * hw * ldx * es, ldx, c, groups, k, hw, w, b, float(eps), act,
                    out.data_ptr() + lo * hw * ldy * es, ldy, stats.data_ptr() + lo * groups * 8, ws.data_ptr(), dt)
    return out, stats


def backward(dy, x, stats, groups, weight=None, bias=None, act=L.ACT_NONE, param_grads=True):
    """stats: what forward() returned for x.  param_grads False: (dx, None, None)."""
    lib = rows.library(x, "x")
    dt = rows.dtype_of(x, "x")
    n, hw, c = _sizes(x, groups, act, "x")
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.get_device() != x.get_device():
        raise ValueError(f"dy must have x's shape, type and device, got {dy.dtype} {tuple(dy.shape)}")
    if stats.dtype != torch.float32 or stats.shape != (n, groups, 2) or not stats.is_contiguous() or stats.get_device() != x.get_device():
        raise ValueError("stats must be what forward() returned for x")
    w, b = rows.check_vector(weight, c, x, "weight"), rows.check_vector(bias, c, x, "bias")
    ldx, ldd = rows.pitch_of(x, "x"), rows.pitch_of(dy, "dy")
    dx = rows.new_like(x)
    dw = x.new_empty(c, dtype=torch.float32) if param_grads else None
    db = x.new_empty(c, dtype=torch.float32) if param_grads else None
    if x.numel() == 0:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    es = x.element_size()
    for lo, k in _batches(n, c, groups):
        ws = rows.workspace(x, lib.group_norm_workspace, "group_norm", c, groups, k, hw)
        gw, gb = (dw, db) if lo == 0 or not param_grads else (torch.empty_like(dw), torch.empty_like(db))
        rows.launch(lib.group_norm_backward, x, "group_norm_backward", dy.data_ptr() + lo * hw * ldd * es, ldd, x.data_ptr() + lo * hw * ldx * es, ldx, c,
                    groups, k, hw, w, b, stats.data_ptr() + lo * groups * 8, act, dx.data_ptr() + lo * hw * c * es, c,
                    None if gw is None else gw.data_ptr(), None if gb is None else gb.data_ptr(), ws.data_ptr(), dt)
        if lo and param_grads:
            dw.add_(gw)
            db.add_(gb)
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, act, eps):
        y, stats = forward(x, groups, weight, bias, act, eps)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1:3]
        dx, dw, db = backward(rows.as_rows(dy), x, stats, ctx.groups, weight, bias, ctx.act, need_w or need_b)
        return dx if ctx.needs_input_grad[0] else None, dw if need_w else None, db if need_b else None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, act=L.ACT_NONE, eps=1e-5):
    """y of forward(), recorded for autograd."""
    rows.refuse_captured_leaves("group_norm_act", x, weight, bias)
    return _GroupNormAct.apply(x, weight, bias, groups, act, eps)
