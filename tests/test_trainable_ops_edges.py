"""Edges of group norm, dropout and the biased row soft-max: arguments that do not fit the launch, values at the ends of the types'
ranges, long sums.  As in test_trainable_ops.py the kernel sources run in the host emulator on the CPU and as the gfx950 library with
``-m gpu``."""
import pytest
import torch

import train_ops_oracle as orc
from gimmvfi_hip import lib as L
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
