"""Row soft-max of attention scores with a learned relative position bias by buckets, and its gradient (csrc/rel_softmax.hip).

Scores x are (B, heads, Q, M): Q queries on a grid qh x qw, M keys on a grid kh x kw (1 x L: a sequence).  With offset = key minus query,

    v = scale * x + table[bucket(offset), head],    y = softmax(v) over the keys that are there,

table (num_buckets, heads) float32 is the learned parameter, a ``RelativeBuckets`` says which bucket an offset has.  A key is out
where key_mask (B, M) is False and where v is -inf; out keys get 0 and a query with no key left a row of zeros
(a NaN among the scores that are there makes the query's whole row NaN).  ``forward`` returns
(y, stats), ``backward`` (dx, dtable); the probabilities are computed again from x and stats, so dtable does not carry the rounding
of a 16-bit y.  ``softmax_rel_bias`` records the pair for autograd.  x is y's type or float32; rows may have a pitch.
"""
import math

import torch

from . import rows


def _pair(g, name):
    h, w = g
    if h < 1 or w < 1 or h * w >= 1 << 30:
        raise ValueError(f"{name} must have positive sides and fewer than 2**30 positions, got {tuple(g)}")
    return int(h), int(w)


class RelativeBuckets:
    """The buckets of every offset between a query grid and a key grid: ``buckets[dy + qh - 1, dx + qw - 1]`` for dy = jy - iy in
    [-(qh - 1), kh - 1], dx likewise; shape (qh + kh - 1, qw + kw - 1), any integer type, values in [0, num_buckets).  Made once
    (it looks at the values, and sorts them for the gradient) and kept beside the weights, on the device of ``buckets``.
    gradient False: not sorted -- for a program that makes a plan per step (a memory that grows) and never asks for dtable."""

    def __init__(self, q_grid, k_grid, buckets, num_buckets, gradient=True):
        self.qh, self.qw = _pair(q_grid, "q_grid")
        self.kh, self.kw = _pair(k_grid, "k_grid")
        self.num_buckets = int(num_buckets)
        shape = (self.qh + self.kh - 1, self.qw + self.kw - 1)
        if buckets.shape != shape or buckets.is_floating_point() or buckets.dtype == torch.bool:
            raise ValueError(f"buckets must be integers of shape {shape}, got {buckets.dtype} {tuple(buckets.shape)}")
        flat = buckets.reshape(-1).to(torch.int64)
        low, high = torch.stack(torch.aminmax(flat)).tolist()            # (the only time that the host waits for the device)
        if not 1 <= self.num_buckets < 1 << 31 or low < 0 or high >= self.num_buckets:
            raise ValueError(f"buckets must lie in [0, {self.num_buckets})")
        self.bucket_of, self.order, self.starts = flat.to(torch.int32).contiguous(), None, None
        if gradient:
            by_bucket, order = torch.sort(flat, stable=True)
            starts = torch.searchsorted(by_bucket, torch.arange(self.num_buckets + 1, device=flat.device))
            self.order, self.starts = order.to(torch.int32), starts.to(torch.int32)

    @classmethod
    def per_offset(cls, q_grid, k_grid, device=None, gradient=True):
        """A bucket of its own for every offset: windows, and attention over a feature map."""
        (qh, qw), (kh, kw) = _pair(q_grid, "q_grid"), _pair(k_grid, "k_grid")
        ny, nx = qh + kh - 1, qw + kw - 1
        return cls(q_grid, k_grid, torch.arange(ny * nx, device=device).reshape(ny, nx), ny * nx, gradient)

    @classmethod
    def logarithmic(cls, queries, keys, num_buckets=32, far=128, two_sided=True, first_query=None, device=None, gradient=True):
        """Sequences: near distances have a bucket each, far ones share logarithmic buckets up to distance ``far``, everything
        beyond is in the last.  two_sided: half of the buckets for keys behind the query; else keys behind it share bucket 0.
        first_query: position of the first query among the keys (None: the queries are the last positions)."""
        if num_buckets < (4 if two_sided else 2):
            raise ValueError(f"num_buckets {num_buckets} is too small")
        first = keys - queries if first_query is None else first_query
        rel = torch.arange(queries + keys - 1, dtype=torch.int64) - (queries - 1) - first
        half = num_buckets // 2 if two_sided else num_buckets
        near = half // 2
        if far <= near:
            raise ValueError(f"far must lie beyond the {near} near distances")
        d = rel.abs() if two_sided else (-rel).clamp(min=0)
        # in 64 bits, with the whole powers of the border kept on their own side
        steps = torch.floor(torch.log(d.clamp(min=1).double() / near) / math.log(far / near) * (half - near) + 1e-9).long()
        b = torch.where(d < near, d, (near + steps).clamp(max=half - 1))
        if two_sided:
            b = b + half * (rel > 0)
        return cls((1, queries), (1, keys), b.reshape(1, -1).to(device), num_buckets, gradient)

    def to(self, device):
        new = object.__new__(RelativeBuckets)
        new.__dict__.update(self.__dict__)
        new.bucket_of, new.order, new.starts = (None if t is None else t.to(device) for t in (self.bucket_of, self.order, self.starts))
        return new


def _check(x, table, plan, key_mask):
    q, m = plan.qh * plan.qw, plan.kh * plan.kw
    if x.dim() != 4 or x.shape[2] != q or x.shape[3] != m:
        raise ValueError(f"x must be (B, heads, {q}, {m}) for this plan, got {tuple(x.shape)}")
    b, h = x.shape[:2]
    if not 1 <= h <= 65535:
        raise ValueError(f"x must have 1 to 65535 heads, got {tuple(x.shape)}")
    if table.dtype != torch.float32 or table.shape != (plan.num_buckets, h) or not table.is_contiguous() or table.get_device() != x.get_device():
        raise ValueError(f"table must be a contiguous float32 tensor of shape ({plan.num_buckets}, {h}) on {x.device}, "
                         f"got {table.dtype} {tuple(table.shape)} on {table.device}")
    if plan.bucket_of.get_device() != x.get_device():
        raise ValueError(f"the plan is on {plan.bucket_of.device}, x on {x.device}: use plan.to(x.device)")
    if key_mask is not None and (key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (b, m) or
                                 not key_mask.is_contiguous() or key_mask.get_device() != x.get_device()):
        raise ValueError(f"key_mask must be a contiguous bool tensor of shape ({b}, {m}) on {x.device}, "
                         f"got {key_mask.dtype} {tuple(key_mask.shape)} on {key_mask.device}")
    return b, h, q, m


def forward(x, table, plan, scale=1.0, key_mask=None, dtype=None, pitch=None):
    """dtype: y's type (None: x's).  pitch: columns of the buffer behind y (the K padding of the product that follows); y is its
    first M columns, the rest is cleared."""
    lib = rows.library(x, "x")
    xt = rows.dtype_of(x, "x")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in rows.DTYPES or (x.dtype != dtype and x.dtype != torch.float32):
        raise ValueError(f"x must be {dtype} or float32, got {x.dtype}")
    b, h, q, m = _check(x, table, plan, key_mask)
    ldx = rows.pitch_of(x, "x")
    ld = m if pitch is None else int(pitch)
    if not m <= ld < 1 << 31:
        raise ValueError(f"pitch {ld} does not hold the {m} columns")
    y = x.new_empty((b, h, q, ld), dtype=dtype)
    stats = x.new_empty((b, h, q, 2), dtype=torch.float32)
    if b:
        ws = rows.workspace(x, lib.softmax_rel_bias_workspace, "softmax_rel_bias", b, h, plan.qh, plan.qw, plan.kh, plan.kw, 0)
        rows.launch(lib.softmax_rel_bias, x, "softmax_rel_bias", x.data_ptr(), xt, ldx, table.data_ptr(), plan.bucket_of.data_ptr(), plan.num_buckets,
                    None if key_mask is None else key_mask.data_ptr(), float(scale), y.data_ptr(), ld, ld,
                    stats.data_ptr(), b, h, plan.qh, plan.qw, plan.kh, plan.kw, ws.data_ptr(),
                    rows.DTYPES[dtype])
    return (y if ld == m else y[..., :m]), stats


def backward(dy, x, stats, table, plan, scale=1.0, key_mask=None, table_grad=True):
    """stats: what forward() returned for x, table, scale and key_mask.  table_grad False: (dx, None)."""
    lib = rows.library(x, "x")
    xt, dt = rows.dtype_of(x, "x"), rows.dtype_of(dy, "dy")
    if x.dtype != dy.dtype and x.dtype != torch.float32:
        raise ValueError(f"x must be {dy.dtype} or float32, got {x.dtype}")
    b, h, q, m = _check(x, table, plan, key_mask)
    if dy.shape != x.shape or dy.get_device() != x.get_device():
        raise ValueError(f"dy must have x's shape and device, got {tuple(dy.shape)} on {dy.device}")
    if stats.dtype != torch.float32 or stats.shape != (b, h, q, 2) or not stats.is_contiguous() or stats.get_device() != x.get_device():
        raise ValueError("stats must be what forward() returned for x")
    if table_grad and plan.order is None:
        raise ValueError("the plan was made with gradient=False")
    ldx, ldd = rows.pitch_of(x, "x"), rows.pitch_of(dy, "dy")
    dx = rows.new_like(x)
    dtable = torch.empty_like(table) if table_grad else None
    if b == 0:
        return dx, None if dtable is None else dtable.zero_()
    ws = rows.workspace(x, lib.softmax_rel_bias_workspace, "softmax_rel_bias", b, h, plan.qh, plan.qw, plan.kh, plan.kw, 1)
    rows.launch(lib.softmax_rel_bias_backward, x, "softmax_rel_bias_backward", dy.data_ptr(), ldd, x.data_ptr(), xt, ldx, table.data_ptr(), plan.bucket_of.data_ptr(),
                plan.num_buckets, plan.order.data_ptr() if table_grad else None, plan.starts.data_ptr() if table_grad else None,
                None if key_mask is None else key_mask.data_ptr(), float(scale), stats.data_ptr(),
                dx.data_ptr(), m, None if dtable is None else dtable.data_ptr(), b, h, plan.qh,
                plan.qw, plan.kh, plan.kw, ws.data_ptr(), dt)
    return dx, dtable


class _SoftmaxRelBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, plan, scale, key_mask, dtype):
        y, stats = forward(x, table, plan, scale, key_mask, dtype)
        ctx.save_for_backward(x, table, stats, key_mask)
        ctx.plan, ctx.scale = plan, scale
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, table, stats, key_mask = ctx.saved_tensors
        dx, dtable = backward(rows.as_rows(dy), x, stats, table, ctx.plan, ctx.scale, key_mask, ctx.needs_input_grad[1])
        return dx if ctx.needs_input_grad[0] else None, dtable, None, None, None, None


def softmax_rel_bias(x, table, plan, scale=1.0, key_mask=None, dtype=None):
    """y of forward(), recorded for autograd."""
    rows.refuse_captured_leaves("softmax_rel_bias", x, table)
    if plan.order is None and table.requires_grad and torch.is_grad_enabled():
        raise ValueError("table requires a gradient, and the plan was made with gradient=False")
    return _SoftmaxRelBias.apply(x, table, plan, scale, key_mask, dtype)
