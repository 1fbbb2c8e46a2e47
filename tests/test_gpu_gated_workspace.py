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


def test_fp32_without_room_for_pieces():
    """Under capture, in an arena that the generic engine fits and the pieces do not, the
    call goes on with the generic engine (sums of fp32 products in another order)."""
    m, d, f = 1100, 700, 1300
    x, w, dh = rnd(m, d), rnd(2 * f, d) * d ** -0.5, rnd(m, f)
    want_h, want_gu = ops.gated_linear_fwd(x, w, save=True)
    want_dx = ops.gated_linear_bwd(dh, x, w, want_gu, need_dw=False, need_db=False)[0]
    ctx = ops.Context(0)
    h, gu, dx = (torch.zeros_like(t) for t in (want_h, want_gu, want_dx))
    rows = 2 * m    # a narrow layer of twice the rows: its [g | u] in fp32
    wide, narrow = torch.zeros(rows, 8, device="cuda"), torch.zeros(2 * f, 8, device="cuda")
    out = torch.zeros(rows, f, device="cuda")
    ctx.call("nott_gated_linear_fwd", 0, rows, 8, f, 0, wide.data_ptr(), narrow.data_ptr(), None, out.data_ptr(), None)
    torch.cuda.synchronize()
    held = ctx.workspace_bytes()
    assert held < 4 * m * 2 * f * 4     # less than four pieces of [dg | du] and of w
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.call("nott_gated_linear_fwd", 0, m, d, f, 0, x.data_ptr(), w.data_ptr(), None, h.data_ptr(), gu.data_ptr())
        ctx.call("nott_gated_linear_bwd", 0, m, d, f, 0, dh.data_ptr(), x.data_ptr(), w.data_ptr(), want_gu.data_ptr(),
                 dx.data_ptr(), None, None, 0)
    assert ctx.workspace_bytes() == held
    for _ in range(2):
        for t in (h, gu, dx):
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in ((h, want_h), (gu, want_gu), (dx, want_dx)):
            assert float((got - want).norm() / want.norm()) <= 2e-6
    del graph
    torch.cuda.synchronize()
    del ctx
    gc.collect()
