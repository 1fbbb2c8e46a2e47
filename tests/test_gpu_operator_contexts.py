"""The language-model operators at the C entry points: what they refuse before any
launch, and what a new context does without its workspace."""
import ctypes as C
import gc

import pytest
import torch

from thot_amd import _abi, ops
from thot_amd._abi import NottInvalidArgument, QkRopeDesc

pytestmark = pytest.mark.gpu


def desc(**kw):
    d = QkRopeDesc(2, 3, 4, 2, 8, 8, (C.c_int64 * 4)(4, 0, 0, 0))
    d.axes, d.norm, d.eps = 1, 1, 1e-6
    for k, v in kw.items():
        if k == "section":
            d.section[:] = v
        else:
            setattr(d, k, v)
    return d


@pytest.fixture(scope="module")
def buf():
    return torch.zeros(4096, device="cuda").data_ptr()


@pytest.mark.parametrize("kw", [
    dict(dh=0), dict(dh=513), dict(rot=7), dict(rot=10), dict(rot=-2), dict(axes=0), dict(axes=5), dict(b=-1),
    dict(section=(3, 0, 0, 0)), dict(section=(4, 1, 0, 0)), dict(section=(5, -1, 0, 0), axes=2), dict(norm=2),
    dict(eps=-1.0), dict(eps=float("nan")), dict(b=2 ** 31, t=1), dict(b=2 ** 20, t=2 ** 20), dict(hq=70000),
    dict(b=2 ** 15, t=2 ** 14, hq=8)])
def test_rope_descriptors(kw, buf):
    ctx, d = ops.context(), desc(**kw)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_qk_norm_rope_fwd", C.byref(d), 0, buf, buf, buf, buf, buf, buf, buf, buf)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_qk_norm_rope_bwd", C.byref(d), 0, buf, buf, buf, buf, buf, buf, buf, buf, buf, buf, buf, buf, 0)


def test_rope_buffers(buf):
    ctx, d = ops.context(), desc()
    good = [C.byref(d), 0, buf, buf, buf, buf, buf, buf, buf, buf]
    for i in (2, 3, 6, 7, 8, 9):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_qk_norm_rope_fwd", *[None if j == i else a for j, a in enumerate(good)])
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_qk_norm_rope_fwd", None, *good[1:])
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_qk_norm_rope_fwd", good[0], 5, *good[2:])
    good = [C.byref(d), 0] + [buf] * 12 + [0]
    for i in (2, 3, 4, 5, 8, 9, 10, 11):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_qk_norm_rope_bwd", *[None if j == i else a for j, a in enumerate(good)])
    plain = desc(norm=0)
    with pytest.raises(NottInvalidArgument, match="needs the norm"):
        ctx.call("nott_qk_norm_rope_fwd", C.byref(plain), 0, buf, buf, buf, None, buf, buf, buf, buf)


@pytest.mark.parametrize("dims", [(-1, 8, 4), (3, 0, 4), (3, 8, 0)])
def test_gated_sizes(dims, buf):
    with pytest.raises(NottInvalidArgument):
        ops.context().call("nott_gated_linear_fwd", 0, *dims, 0, buf, buf, None, buf, None)
    with pytest.raises(NottInvalidArgument):
        ops.context().call("nott_gated_linear_bwd", 0, *dims, 0, buf, buf, buf, buf, buf, buf, buf, 0)


def test_gated_arguments(buf):
    ctx = ops.context()
    for act in (-1, 5):
        with pytest.raises(NottInvalidArgument, match="activation"):
            ctx.call("nott_gated_linear_fwd", 0, 2, 8, 4, act, buf, buf, None, buf, None)
    for i in (5, 6, 8):
        a = [0, 2, 8, 4, 0, buf, buf, None, buf, None]
        a[i] = None
        with pytest.raises(NottInvalidArgument, match="null"):
            ctx.call("nott_gated_linear_fwd", *a)
    for i in (5, 6, 7, 8):      # dh, x (dw asked for), w (dx asked for), gu
        a = [0, 2, 8, 4, 0, buf, buf, buf, buf, buf, buf, buf, 0]
        a[i] = None
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_gated_linear_bwd", *a)
    assert ctx.call("nott_gated_linear_bwd", 0, 2, 8, 4, 0, buf, None, None, buf, None, None, None, 0) == 0


def test_logprob_arguments(buf):
    ctx = ops.context()
    good = [0, 3, 5, buf, buf, 1.0, 2, buf, buf, buf, buf, buf]
    for i, bad in ((0, 7), (1, -1), (2, 0), (3, None), (4, None), (5, 0.0), (5, -1.0), (5, float("nan")),
                   (5, float("inf")), (6, -1), (6, 6), (6, 65), (7, None), (10, None), (11, None), (1, 2 ** 31)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_token_logprob_fwd", *[bad if j == i else a for j, a in enumerate(good)])
    good = [0, 3, 5, buf, buf, 1.0, buf, buf, buf, buf, buf]
    for i, bad in ((0, 7), (1, -1), (2, 0), (3, None), (4, None), (5, 0.0), (6, None), (7, None), (8, None), (10, None)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_token_logprob_bwd", *[bad if j == i else a for j, a in enumerate(good)])


def test_new_context_under_capture():
    """A context without workspace cannot get any under capture: rows that would be
    split are taken whole, and a gated layer that needs none runs."""
    n, c, top = 2, 70000, 4
    z = torch.randn(n, c, device="cuda")
    y = torch.tensor([5, 69999], device="cuda")
    want = ops.token_logprob_fwd(z, y, top=top)
    x, w = torch.randn(200, 256, device="cuda").bfloat16(), torch.randn(256, 256, device="cuda").bfloat16()
    hw = ops.gated_linear_fwd(x, w)[0]
    out = [torch.zeros(n, device="cuda") for _ in range(3)]
    tv, ti = torch.zeros(n, top, device="cuda"), torch.zeros(n, top, device="cuda", dtype=torch.int64)
    h = torch.zeros_like(hw)
    ctx = ops.Context(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.call("nott_token_logprob_fwd", 0, n, c, z.data_ptr(), y.data_ptr(), 1.0, top, *(t.data_ptr() for t in out),
                 tv.data_ptr(), ti.data_ptr())
        ctx.call("nott_gated_linear_fwd", 1, 200, 256, 128, 0, x.data_ptr(), w.data_ptr(), None, h.data_ptr(), None)
    assert ctx.workspace_bytes() == 0
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ti, want[4]) and torch.equal(h, hw)
        for a, b in zip(out, want):     # sums in another order
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    del graph
    torch.cuda.synchronize()
    del ctx
    gc.collect()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_workspace_that_grows_inside_a_call(dt):
    """A new context whose arena grows under a product of the call keeps what the call
    holds: the same bits as a context that has the memory already."""
    m, d, f = 300, 392, 520
    x, w = torch.randn(m, d, device="cuda").to(dt), torch.randn(2 * f, d, device="cuda").to(dt)
    gu, dh = torch.randn(m, 2 * f, device="cuda").to(dt), torch.randn(m, f, device="cuda").to(dt)
    ops.gated_linear_bwd(dh, x, w, gu)
    want = ops.gated_linear_bwd(dh, x, w, gu)
    ctx = ops.Context(0)
    got = [torch.empty_like(t) for t in want]
    for _ in range(2):
        ctx.call("nott_gated_linear_bwd", ops.nott_dtype(dt), m, d, f, 0, dh.data_ptr(), x.data_ptr(), w.data_ptr(),
                 gu.data_ptr(), *(t.data_ptr() for t in got), 0)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert ctx.workspace_bytes() > 0
    del ctx
    gc.collect()
