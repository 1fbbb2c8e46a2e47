"""What gated_linear takes of a new context's workspace."""
import gc

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rnd(*s, dt=torch.float32):
    return torch.randn(s, device="cuda").to(dt)


@pytest.mark.parametrize("dt", DT)
def test_bias_gradient_alone_takes_its_sums_only(dt):
    dt = DT[dt]
    m, d, f = 4096, 512, 1024
    gu, dh = rnd(m, 2 * f, dt=dt), rnd(m, f, dt=dt)
    x, w = rnd(m, d, dt=dt), rnd(2 * f, d, dt=dt)
    want = ops.gated_linear_bwd(dh, x, w, gu)[2]
    ctx = ops.Context(0)
    db = torch.zeros(2 * f, device="cuda")
    ctx.call("nott_gated_linear_bwd", ops.nott_dtype(dt), m, d, f, 0, dh.data_ptr(), None, None, gu.data_ptr(), None, None,
             db.data_ptr(), 0)
    torch.cuda.synchronize()
    assert torch.equal(db, want)
    assert ctx.workspace_bytes() <= 1 << 20      # 128 rows of partial sums of 2·f
    del ctx
    gc.collect()
