"""Edges of group norm, dropout and the biased row soft-max: arguments that do not fit the launch, values at the ends of the types'
ranges, long sums.  As in test_trainable_ops.py the kernel sources run in the host emulator on the CPU and as the gfx950 library with
``-m gpu``."""
import math

import pytest
import torch

import train_ops_oracle as orc
from gimmvfi_hip import group_norm as gn
from gimmvfi_hip import lib as L
from gimmvfi_hip import rel_softmax as rs
from test_trainable_ops import BF16, F16, F32, _gen, _gn_case, _gn_inputs, _rs_case, _rs_inputs, _rs_plan, _runtime, _within, dev  # noqa: F401


# ------------------------------------------------------------------------------------------------ the launch list's arguments
def test_runtime_forms_refuse_what_they_would_read_or_write_wrongly():
    """The launch-list forms hand plain pointers on: types, lengths, layouts and the output's rows are looked at first."""
    from gimmvfi_hip.ops import View

    rt = _runtime(torch.device("cpu"), "fp16")
    x = torch.zeros(2, 3, 4, 16, dtype=F16)
    w, b = torch.ones(16), torch.zeros(16)
    gn = lambda x_=x, c=16, gb=(w, b), out=None: rt.group_norm(x_, c, 4, gb, out=out)
    gn()
    gn(out=torch.zeros(2, 3, 4, 24, dtype=F16))
    for kw in (dict(gb=(w.half(), b)), dict(gb=(w, b.half())), dict(gb=(w[:8], b)), dict(gb=(w, b[:15])), dict(gb=(w.repeat(2)[::2], b)),
               dict(x_=x.float()), dict(x_=x.bfloat16()), dict(x_=View(x, 8, 16)), dict(x_=x[..., ::2], c=8, gb=None),
               dict(x_=x[:, :, :, :8]), dict(x_=x[0]), dict(c=24, gb=None), dict(out=x[:1]), dict(out=x.float()),
               dict(out=View(torch.zeros(2, 3, 4, 24, dtype=F16), 16, 16)), dict(out=torch.zeros(2, 4, 4, 16, dtype=F16)[:, 1:])):
        with pytest.raises(ValueError):
            gn(**kw)
    plan = _rs_plan("grid", (3, 4), (3, 4), torch.device("cpu"))
    table = torch.zeros(plan.num_buckets, 2)
    s = torch.zeros(2 * 2 * 12, 12)
    rs = lambda table_=table, out=torch.zeros(48, 16, dtype=F16), x_=s, m=None: rt.softmax_rel_bias(x_, table_, plan, out, 2, 2, key_mask=m)
    rs()
    rs(out=torch.zeros(50, 12, dtype=F16))
    for kw in (dict(table_=table.half()), dict(table_=table.double()), dict(table_=torch.zeros(2, plan.num_buckets).t()),
               dict(table_=table[:-1]), dict(out=torch.zeros(48, 16)), dict(out=torch.zeros(47, 16, dtype=F16)),
               dict(out=torch.zeros(48, 11, dtype=F16)), dict(out=View(torch.zeros(48, 16, dtype=F16), 8, 12)),
               dict(out=torch.zeros(48, 32, dtype=F16)[:, ::2]), dict(m=torch.ones(2, 12))):
        with pytest.raises(ValueError):
            rs(**kw)


# ------------------------------------------------------------------------------------------------ NaN rows stay alone
# keys of a 1 x M row; above 128 columns fours of columns are taken together, four queries at a time up to 1024 and from 2049 to 4096
# columns, two at a time elsewhere
@pytest.mark.parametrize("whole", [False, True], ids=["one", "whole"])
@pytest.mark.parametrize("m", [145, 146, 147, 257, 1025, 1026, 1027, 2051, 4097])
def test_softmax_rel_bias_nan_row_reaches_its_own_offsets_only(dev, m, whole):
    plan = _rs_plan("grid", (1, 6), (1, m), dev)
    table = torch.randn(plan.num_buckets, 1, generator=_gen(1))
    x, dy = torch.randn(1, 1, 6, m, generator=_gen(2)), torch.randn(1, 1, 6, m, generator=_gen(3))
    x[0, 0, 4, slice(None) if whole else 7] = float("nan")
    y, stats = rs.forward(x.to(dev), table.to(dev), plan)
    dx, dt = rs.backward(dy.to(dev), x.to(dev), stats, table.to(dev), plan)
    for t in (y.cpu(), dx.cpu()):
        assert bool(t[0, 0, 4].isnan().all()) and not bool(t[0, 0, [0, 1, 2, 3, 5]].isnan().any())
    # query 4 of six meets the slots 1 .. m of m + 5: key j has slot j - 4 + 5
    bad = dt.cpu().isnan()[:, 0]
    assert bad[1:m + 1].all() and not bad[0] and not bad[m + 1:].any(), bad.nonzero().flatten().tolist()[-3:]
    # the offsets that no NaN meets have the gradient of the rows that hold none
    clean = x.clone()
    clean[0, 0, 4] = -float("inf")
    ref = orc.softmax_rel_bias(clean, table, plan.bucket_of, (1, 6), (1, m), 1.0, None, F32, dy)
    keep = torch.ones(m + 5, dtype=torch.bool)
    keep[1:m + 1] = False
    _within(dt.cpu()[keep], ref["dtable"][keep], ref["dtable_tol"][keep], "dtable")


# ------------------------------------------------------------------------------------------------ launches from several threads
@pytest.mark.parametrize("small_first", [0, 1])
def test_two_threads_leave_the_larger_limit_of_dynamic_lds(simlib, small_first):
    """Autograd's threads launch the backward pass with slabs of different sizes: the kernel's limit must not fall again."""
    assert simlib.dll.gvfi_emu_limit_selftest(small_first) == 1000


# ------------------------------------------------------------------------------------------------ launches of 2^32 lanes and more
def test_sizes_whose_sums_would_be_launches_of_too_many_lanes_are_taken(simlib):
    """Sixteen slots or buckets per 256 lanes: from 2^28 on the sums behind the slabs loop instead of asking for 2^32 lanes.  (In the
    emulator seven workgroups loop over everything, so every case of the suite goes through them.)"""
    assert simlib.softmax_rel_bias_workspace(1, 1, 1, 1, 1, (1 << 28) + 64, 1) > 0
    # rows of 9000 columns: 1024 lanes take sixteen rows, so 2^26 rows would be 2^32 lanes
    assert simlib.softmax_rel_bias_workspace(1 << 12, 1 << 11, 1, 8, 1, 9000, 0) == -2
    assert simlib.softmax_rel_bias_workspace(1 << 11, 1 << 11, 1, 8, 1, 9000, 0) > 0


@pytest.mark.parametrize("case", [((1, 40), (1, 300), "grid"), ((3, 5), (7, 20), "shared"), ((1, 3), (1, 5000), "log"), ((2, 2), (30, 41), "grid")],
                         ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}")
def test_softmax_rel_bias_sums_in_loops(dev, case):
    q, k, kind = case
    _rs_case(dev, 2, 2, q, k, kind, F32, F32, False, None, 0)


@pytest.mark.gpu
def test_gpu_softmax_rel_bias_one_query_2_28_keys():
    """A bucket of its own for every one of 2^28 + 64 keys: the table's gradient is the gradient of the scores, both in float."""
    d = torch.device("cuda", 0)
    m = (1 << 28) + 64
    plan = rs.RelativeBuckets.per_offset((1, 1), (1, m), device=d)
    x, dy, table = (torch.randn(1, 1, 1, m, device=d, generator=torch.Generator(device=d).manual_seed(k)) for k in (1, 2, 3))
    table = table.view(m, 1)
    y, stats = rs.forward(x, table, plan)
    dx, dt = rs.backward(dy, x, stats, table, plan)
    assert torch.equal(dx.view(-1), dt.view(-1))
    v = x.view(-1).double() + table.view(-1)
    p = torch.exp(v - v.max())
    p /= p.sum()
    # |v| and the largest value stay below 10: four roundings of each, and at most 88 of the exponential, the sums and the inverse
    rel = orc.U * (4 * 10 + 4 * 10 + 88)
    assert bool(((y.view(-1).double() - p).abs() <= p * (rel + 2 * orc.U) + 2.0 ** -126).all())
    g = dy.view(-1).double()
    dot = (p * g).sum()
    tol = p * (rel * (g - dot).abs() + (p * g.abs()).sum() * (rel + 96 * orc.U) + 8 * orc.U * (g.abs() + dot.abs())) + 2.0 ** -126
    assert bool(((dx.view(-1).double() - p * (g - dot)).abs() <= tol + 2 * orc.U * (p * (g - dot)).abs()).all())


# ------------------------------------------------------------------------------------------------ long sums
def _statistics(x, dy, groups, eps=1e-5):
    """64-bit mean, rstd of the groups, sum dy and sum dy xhat of the channels (no activation, no weights) of x, dy (N, P, C), with bounds as
    in train_ops_oracle.group_norm: 64 roundings of the mean, 72 of xhat, 96 of a channel's sums.  By runs of pixels: x may be large."""
    n, p, c = x.shape
    cg = c // groups
    runs = range(0, p, 1 << 15)
    tot = torch.zeros(n, groups, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(tot)
    for r in runs:
        v = x[:, r:r + (1 << 15)].double().reshape(n, -1, groups, cg)
        tot += v.sum((1, 3))
        mag += v.abs().sum((1, 3))
    mean, mag = tot / (p * cg), mag / (p * cg)
    sq = torch.zeros_like(tot)
    for r in runs:
        sq += ((x[:, r:r + (1 << 15)].double().reshape(n, -1, groups, cg) - mean.view(n, 1, groups, 1)) ** 2).sum((1, 3))
    rstd = 1 / torch.sqrt(sq / (p * cg) + eps)
    sums = [torch.zeros(c, dtype=torch.float64, device=x.device) for _ in range(4)]
    for r in runs:
        v = x[:, r:r + (1 << 15)].double().reshape(n, -1, groups, cg)
        d = dy[:, r:r + (1 << 15)].double().reshape(v.shape)
        hat = (v - mean.view(n, 1, groups, 1)) * rstd.view(n, 1, groups, 1)
        h_err = orc.U * (64 * ((mag + mean.abs()).view(n, 1, groups, 1) + v.abs()) * rstd.view(n, 1, groups, 1) + 72 * hat.abs())
        for s, t in zip(sums, (d, 96 * orc.U * d.abs(), d * hat, d.abs() * h_err + 96 * orc.U * (d * hat).abs())):
            s += t.sum((0, 1)).reshape(c)
    return (mean, 64 * orc.U * (mag + mean.abs())), (rstd, 72 * orc.U * rstd), sums[:2], sums[2:]


def test_group_norm_sums_of_many_pixels_per_lane(dev):
    """400 pixels for each of the four lanes of an octet of 512 channels, the first values so large that a chain of additions behind them
    loses every one: a lane's sums have to be folded on the way."""
    p = (16 if dev.type == "cpu" else 1280) * 4 * 400
    i = torch.arange(p, device=dev) // 4 % 400
    x = torch.where(i == 0, 0.0, torch.where(i == 1, 2.0 ** 24, 1.0)).to(BF16).view(1, p, 1).expand(1, p, 512).contiguous()
    dy = torch.where(i == 0, 2.0 ** 24, 1.0).to(BF16).view(1, p, 1).expand(1, p, 512).contiguous()
    mean, rstd, db, dw = _statistics(x, dy, 1)
    y, stats = gn.forward(x, 1)
    _within(stats[..., 0], *mean, "mean")
    _within(stats[..., 1], *rstd, "rstd")
    _, dgamma, dbeta = gn.backward(dy, x, stats, 1)
    _within(dbeta, *db, "dbias")
    _within(dgamma, *dw, "dweight")


def test_softmax_rel_bias_sums_of_many_tiles(dev):
    """A row in 200 tiles of 8192 columns.  The first tile's sum is 1, every other tile adds 0.12 steps of float to it (2^-23 each): additions
    one behind the other in float would lose them all, 24 steps together."""
    m = 200 * 8192
    x = torch.full((m,), -15.9423851 - math.log(8192.0) + math.log(0.12))
    x[0] = 0.0
    x[1:8192] = -math.inf
    e = torch.exp(x.double())
    plan = rs.RelativeBuckets((1, 1), (1, m), torch.zeros(1, m, dtype=torch.int64, device=dev), 1)
    table = torch.zeros(1, 1, device=dev)
    y, stats = rs.forward(x.view(1, 1, 1, m).to(dev), table, plan)
    # 1 / sum: at most 16 roundings in a tile, the joined sum's and the inverse's, of terms that are all positive; the exponential's own
    # error (|x| / 2 steps and one) applies to the small part of the sum only
    small = float(e.sum()) - 1.0
    tol = 2.0 * orc.U + small * 64 * orc.U
    assert abs(float(stats[0, 0, 0, 1]) * float(e.sum()) - 1.0) <= tol, (float(stats[0, 0, 0, 1]), float(e.sum()))


# a mean far above the spread: the one-launch form, streaming with octets that are not whole, streaming with aligned octets, channels one by
# one (more than a workgroup covers, groups that do not fit it)
@pytest.mark.parametrize("shape,groups", [((2, 99, 16), 2), ((2, 2000, 12), 3), ((1, 1100, 16), 1), ((1, 70, 1032), 3)],
                         ids=lambda v: str(v).replace(" ", ""))
def test_group_norm_common_mean_of_a_thousand(dev, shape, groups):
    g = _gen(7)
    x, dy = torch.randn(shape, generator=g) + 1000.0, torch.randn(shape, generator=g)
    ref = orc.group_norm(x, groups, None, None, L.ACT_NONE, 1e-5, dy)
    # the difference of the mean square and the squared mean, in float, is not good enough for these bounds
    v = x.reshape(shape[0], -1, groups, shape[-1] // groups)
    mean, sq = v.mean((1, 3), keepdim=True), (v * v).mean((1, 3), keepdim=True)
    naive = ((v - mean) / torch.sqrt(torch.clamp(sq - mean * mean, min=0) + 1e-5)).reshape(shape)
    assert bool(((naive.double() - ref["y"]).abs() > ref["y_tol"]).any())
    y, stats = gn.forward(x.to(dev), groups)
    _within(y, ref["y"], ref["y_tol"], "y")
    dx, dw, db = gn.backward(dy.to(dev), x.to(dev), stats, groups)
    for got, k in ((dx, "dx"), (dw, "dw"), (db, "db")):
        _within(got, ref[k], ref[k + "_tol"], k)


# forms that the cases of test_trainable_ops.py do not reach in the emulator: aligned octets streamed in several chunks; the parameters'
# gradients of more than 128 images behind the streaming form
@pytest.mark.parametrize("case", [((1, 1100, 16), 1, L.ACT_SILU, F32, None, 0, True), ((3, 700, 64), 4, L.ACT_GELU, BF16, 72, 8, True),
                                  ((130, 3, 256), 1, L.ACT_GELU, BF16, None, 0, True), ((131, 5, 20), 5, L.ACT_TANH, F16, 23, 1, True),
                                  ((260, 2, 136), 1, L.ACT_SIGMOID, F32, None, 0, True)],
                         ids=lambda c: f"{'x'.join(map(str, c[0]))}-{c[1]}-{str(c[3])[6:]}")
def test_group_norm_streamed(dev, case):
    _gn_case(dev, *case)


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.gpu
def test_gpu_group_norm_pitched_rows_beyond_32_bits_of_elements():
    """Two images of 40000 pixels of 24 channels at a pitch of 32768: the second lies behind 2^30 elements, its last pixels behind 2^31."""
    d = torch.device("cuda", 0)
    x, w, b, dy = _gn_inputs((2, 40000, 24), BF16, 12)
    wide = [torch.full((2, 40000, 32768), float("nan"), dtype=BF16, device=d) for _ in range(2)]
    assert wide[0].numel() > 1 << 31
    for t, v in zip(wide, (x, dy)):
        t[..., 32000:32024] = v.to(d)
    xd, dyd = (t[..., 32000:32024] for t in wide)
    ref = orc.group_norm(x, 3, w, b, L.ACT_SILU, 1e-5, dy)
    y, stats = gn.forward(xd, 3, w.to(d), b.to(d), L.ACT_SILU, out=wide[0][..., 8:32])
    _within(y, ref["y"], ref["y_tol"], "y")
    dx, dw, db = gn.backward(dyd, xd, stats, 3, w.to(d), b.to(d), L.ACT_SILU)
    for got, k in ((dx, "dx"), (dw, "dw"), (db, "db")):
        _within(got, ref[k], ref[k + "_tol"], k)
    assert bool(wide[0][..., 32:32000].isnan().all()) and bool(wide[0][..., :8].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(4, 1, (7, 7), (7, 7), "grid", 13_000_000), (2, 1, (5, 8), (13, 20), "grid", 30_000_000),
                                  (2, 1, (5, 4), (13, 11), "shared", 60_000_000), (1, 1, (1, 110), (1, 20000), "log", 20_000_000)],
                         ids=lambda c: f"{c[2]}-{c[3]}-{c[4]}")
def test_gpu_softmax_rel_bias_pitched_rows_beyond_32_bits_of_elements(case):
    """Every form of the kernels with the last rows behind 2^31 elements, scores, gradients and probabilities alike."""
    d = torch.device("cuda", 0)
    B, heads, q, k, kind, pitch = case
    plan, x, table, mask, dy = _rs_inputs(B, heads, q, k, kind, BF16, BF16, False, d)
    n, m = x.numel() // x.shape[-1], x.shape[-1]
    assert (n - 1) * pitch > 1 << 31
    ref = orc.softmax_rel_bias(x, table, plan.bucket_of, q, k, 0.7, None, BF16, dy)
    def spread(t):
        wide = torch.empty(n * pitch, dtype=BF16, device=d).as_strided(x.shape, (heads * x.shape[2] * pitch, x.shape[2] * pitch, pitch, 1))
        wide.copy_(t)
        return wide
    xd, dyd, td = spread(x), spread(dy), table.to(d)
    y, stats = rs.forward(xd, td, plan, 0.7, pitch=pitch)
    _within(y, ref["y"], ref["y_tol"], "y")
    del y
    dx, dt = rs.backward(dyd, xd, stats, td, plan, 0.7)
    _within(dx, ref["dx"], ref["dx_tol"], "dx")
    _within(dt, ref["dtable"], ref["dtable_tol"], "dtable")


# ------------------------------------------------------------------------------------------------ activations, relative to their values
@pytest.mark.parametrize("c", [128, 1024], ids=["one launch", "streamed"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("act", ["sigmoid", "silu", "tanh", "gelu"])
def test_group_norm_activation_relative_to_its_value(dev, act, dtype, c):
    """weight 0 and the bias as argument: y is act(bias) and dbias its derivative (times dy = 1, in float for every type) and nothing else.

    Bounds in roundings of the value: float tensors exp and division 2 steps each, 1 + e and products 1 each, tanh 4, erfc 16 and its
    argument's rounding, which erfc carries on z^2 times, twice.  16-bit tensors 2^-16 for all of it, and the output's own half step.  A derivative that
    crosses zero: relative to its two terms."""
    kind = getattr(L, "ACT_" + act.upper())
    g = _gen(c)
    z = torch.cat([torch.pow(10.0, torch.linspace(-9, 1, c // 4)), -torch.pow(10.0, torch.linspace(-9, 1, c // 4)), torch.linspace(-12.5, 12.5, c // 2)])
    x = torch.randn(1, 1, c, generator=g).to(dtype).to(dev)
    w, b = torch.zeros(c, device=dev), z.to(dev)
    y, stats = gn.forward(x, 1, w, b, kind)
    dx, dw, db = gn.backward(torch.ones_like(x), x, stats, 1, w, b, kind)
    zd = z.double()
    ref, slope = orc.act(zd, kind), orc.act_slope(zd, kind)
    if act == "tanh":
        slope = 1 / torch.cosh(zd) ** 2                      # (1 - tanh^2 has no digits left where tanh is 1)
    if act == "gelu":
        parts = 0.5 * torch.special.erfc(-zd / math.sqrt(2)) + (zd * torch.exp(-zd * zd / 2)).abs() / math.sqrt(2 * math.pi)
    elif act == "silu":
        parts = torch.sigmoid(zd) + (zd * torch.sigmoid(zd) * torch.sigmoid(-zd)).abs()
    else:
        parts = slope
    rel = (24 + 4 * zd * zd) * orc.U if act == "gelu" else torch.full_like(zd, 16 * orc.U)
    if dtype != F32:
        rel = torch.full_like(zd, 2.0 ** -16)
    _within(y.view(-1), ref, ref.abs() * rel + (orc.rounding(ref, dtype) if dtype != F32 else 0) + 2.0 ** -126, "y")
    _within(db, slope, parts * rel + 2.0 ** -126, "slope")
    assert float(dx.abs().max()) == 0


# ------------------------------------------------------------------------------------------------ small probabilities of float scores
# every form of the kernels: 16 lanes, four columns of four or two queries, column by column, tiles
@pytest.mark.parametrize("q,k", [((1, 2), (1, 100)), ((1, 5), (1, 400)), ((1, 3), (1, 1500)), ((1, 1), (1, 300)), ((2, 2), (9, 101)), ((1, 2), (1, 17000))],
                         ids=lambda v: str(v).replace(" ", ""))
def test_softmax_rel_bias_small_probabilities_keep_their_digits(dev, q, k):
    """Scores that are exact in float, one 0 and the others down to -85: the exponential of every difference is good to two steps (four
    roundings) relative to itself, the sum and the inverse add 16, the gradient's two products and difference three."""
    m = k[0] * k[1]
    x = -(torch.arange(m) % 680).float() / 8
    x = x.view(1, 1, 1, m).expand(1, 1, q[0] * q[1], m).contiguous()
    plan = rs.RelativeBuckets(q, k, torch.zeros(q[0] + k[0] - 1, q[1] + k[1] - 1, dtype=torch.int64, device=dev), 1)
    table = torch.zeros(1, 1, device=dev)
    y, stats = rs.forward(x.to(dev), table, plan)
    p = torch.softmax(x.double(), -1)
    _within(y, p, p * (20 * orc.U) + 2.0 ** -126, "y")
    dy = torch.where(torch.arange(m) % 680 == 0, 0.0, 1.0).expand_as(x).contiguous()       # (the gradient of the small ones is no difference)
    dot = (p * dy).sum(-1, keepdim=True)
    for t in (F32, BF16):                                   # (probabilities of 16 bits: the scores' gradient is float all the same)
        dx, _ = rs.backward(dy.to(t).to(dev), x.to(dev), stats, table, plan)
        _within(dx, p * (dy - dot), p * (24 * orc.U) * (dy - dot).abs() + p * dot * 32 * orc.U + 2.0 ** -126, "dx")


# ------------------------------------------------------------------------------------------------ SiLU outside group norm
def test_silu_is_refused_by_every_entry_point_of_the_convolutions(simlib):
    """A convolution that the LDS-DMA kernel takes, called by its own entry points: their epilogues know no SiLU (and would take its number
    for another function's)."""
    import ctypes as C

    from gimmvfi_hip.ops import ConvLayer, Runtime

    rt = Runtime(simlib, "bf16", "cpu")
    x, w = torch.randn(1, 4, 8, 64, generator=_gen(1)).to(BF16), torch.randn(32, 64, 1, 1, generator=_gen(2)) / 8
    layer, out = ConvLayer(rt, w, None), torch.zeros(1, 4, 8, 32, dtype=BF16)
    for kw in (dict(act1=L.ACT_SILU), dict(act2=L.ACT_SILU), {}):
        p = rt.conv(layer, x, out, algo=2, _defer=True, **kw)[0]
        entries = [simlib.conv2d, simlib.conv2d_glds] + [simlib.conv2d_patch, simlib.conv2d_col7, simlib.conv2d_p3x3, simlib.conv2d_p3x3s] * bool(kw)
        for f in entries:
            assert f(C.byref(p), None) == (-2 if kw else 0)
        if kw:
            assert simlib.conv2d_pair(C.byref(p), C.byref(p), None) == -2
            assert bool((out == 0).all())


# ------------------------------------------------------------------------------------------------ plans
def test_plan_without_the_gradients_tables(dev):
    """A program that never asks for the table's gradient gets its plan without a sort; asked for all the same, it is refused."""
    for make in (lambda **kw: rs.RelativeBuckets.logarithmic(2, 70, device=dev, **kw), lambda **kw: rs.RelativeBuckets.per_offset((1, 2), (1, 70), device=dev, **kw),
                 lambda **kw: rs.RelativeBuckets((1, 2), (1, 70), torch.arange(71, device=dev).view(1, 71) % 9, 9, **kw)):
        full, plan = make(), make(gradient=False).to(dev)
        assert plan.order is None and plan.starts is None and torch.equal(plan.bucket_of, full.bucket_of)
        assert full.starts.tolist() == [int((full.bucket_of < k).sum()) for k in range(full.num_buckets + 1)]
        table, x = torch.randn(plan.num_buckets, 2, generator=_gen(1)).to(dev), torch.randn(1, 2, 2, 70, generator=_gen(2)).to(dev)
        y, stats = rs.forward(x, table, plan)
        assert torch.equal(y, rs.forward(x, table, full)[0])
        assert torch.equal(rs.backward(y, x, stats, table, plan, table_grad=False)[0], rs.backward(y, x, stats, table, full)[0])
        with pytest.raises(ValueError, match="gradient=False"):
            rs.backward(y, x, stats, table, plan)
        with pytest.raises(ValueError, match="gradient=False"):
            rs.softmax_rel_bias(x, table.clone().requires_grad_(), plan)
        assert torch.equal(rs.softmax_rel_bias(x, table, plan), y)


# ------------------------------------------------------------------------------------------------ more images than one launch takes
def _many_images(dev, shape, groups, dtype, monkeypatch=None, limit=None):
    if limit:
        monkeypatch.setattr(gn, "LAUNCH", limit)
    _gn_case(dev, shape, groups, L.ACT_SILU, dtype, shape[-1] + 3, 1, True)


@pytest.mark.parametrize("shape,groups,limit", [((23, 40), 5, 64), ((9, 3, 2, 16), 2, 32), ((130, 5, 24), 3, 401)], ids=lambda v: str(v).replace(" ", ""))
def test_group_norm_in_several_calls(dev, monkeypatch, shape, groups, limit):
    """A batch whose (image, group) pairs are more than a launch takes goes out in several; here with a small limit."""
    _many_images(dev, shape, groups, F32, monkeypatch, limit)


@pytest.mark.gpu
def test_gpu_group_norm_of_many_rows():
    """Tokens as images of one pixel, 32 groups: 300000 x 32 pairs pass the 2^23 workgroups of a launch."""
    _many_images(torch.device("cuda", 0), (300000, 64), 32, BF16)
