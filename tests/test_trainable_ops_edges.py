"""Edges of group norm, dropout and the biased row soft-max: arguments that do not fit the launch, values at the ends of the types'
ranges, long sums.  As in test_trainable_ops.py the kernel sources run in the host emulator on the CPU and as the gfx950 library with
``-m gpu``."""
import pytest
import torch

import train_ops_oracle as orc
from gimmvfi_hip import lib as L
from gimmvfi_hip import rel_softmax as rs
from test_trainable_ops import BF16, F16, F32, _gen, _rs_plan, _runtime, _within, dev  # noqa: F401


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
