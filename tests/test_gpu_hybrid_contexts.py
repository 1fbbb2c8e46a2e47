"""Differential attention, the gated linear recurrence and Adam over many tensors at the C
entry points: what they refuse before any launch, what a new context does without its
workspace, and calls at the same time on two streams."""
import ctypes as C
import gc
import math

import pytest
import torch

from thot_amd import ops
from thot_amd._abi import AdamTensor, DiffAttnDesc, NottInvalidArgument, ScanDesc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def buf():
    return torch.zeros(1 << 16, device="cuda").data_ptr()


def diff(**kw):
    d = DiffAttnDesc()
    d.b, d.h, d.hk, d.t, d.s, d.dh, d.dv, d.scale = 2, 4, 2, 3, 5, 8, 16, 0.5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(b=-1), dict(h=-2), dict(hk=-1), dict(t=-1), dict(s=-1), dict(dh=0), dict(dv=0), dict(dh=65), dict(dv=129), dict(hk=0),
    dict(hk=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(causal=2),
    dict(token_lam=-1), dict(t=4000001), dict(t=2000001), dict(s=4000001), dict(b=2 ** 22), dict(h=2 ** 20, hk=2 ** 20)])
def test_diff_descriptors(kw, buf):
    ctx, d = ops.context(), diff(**kw)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_diff_attention_fwd", C.addressof(d), 0, buf, buf, buf, buf, None, None, buf, buf, None)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_diff_attention_bwd", C.addressof(d), 0, buf, buf, buf, buf, buf, None, None, buf, buf, buf, buf, buf, buf,
                 buf, 0)


def test_diff_buffers(buf):
    ctx, d = ops.context(), diff()
    good = [C.addressof(d), 0, buf, buf, buf, buf, None, None, buf, buf, None]
    for i, bad in ((0, None), (1, 5), (2, None), (3, None), (4, None), (5, None), (8, None), (9, None)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_diff_attention_fwd", *[bad if j == i else a for j, a in enumerate(good)])
    good = [C.addressof(d), 0, buf, buf, buf, buf, buf, None, None, buf, buf, buf, buf, buf, buf, buf, 0]
    for i in (0, 2, 3, 4, 5, 6, 9, 10, 11, 12, 13, 14, 15):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_diff_attention_bwd", *[None if j == i else a for j, a in enumerate(good)])
    token = diff(token_lam=1)
    with pytest.raises(NottInvalidArgument, match="accumulate"):
        ctx.call("nott_diff_attention_bwd", C.addressof(token), *good[1:-1], 1)


def scan(**kw):
    d = ScanDesc()
    d.b, d.t, d.d, d.sigmoid, d.mix = 2, 3, 8, 1, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [dict(b=-1), dict(t=-1), dict(d=0), dict(d=-3), dict(d=2 ** 30), dict(t=2 ** 40), dict(b=2 ** 31),
                                dict(b=2 ** 23), dict(sigmoid=2), dict(mix=-1)])
def test_scan_descriptors(kw, buf):
    ctx, d = ops.context(), scan(**kw)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_linear_scan_fwd", C.addressof(d), 0, buf, buf, None, None, buf, None, None)
    with pytest.raises(NottInvalidArgument):
        ctx.call("nott_linear_scan_bwd", C.addressof(d), 0, buf, buf, buf, None, buf, None, buf, buf, None)


def test_scan_buffers(buf):
    ctx, d = ops.context(), scan()
    good = [C.addressof(d), 0, buf, buf, None, None, buf, None, None]
    for i, bad in ((0, None), (1, 7), (2, None), (3, None), (6, None)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_linear_scan_fwd", *[bad if j == i else a for j, a in enumerate(good)])
    good = [C.addressof(d), 0, buf, buf, buf, None, buf, None, buf, buf, None]
    for i in (0, 2, 3, 4, 6, 8, 9):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_linear_scan_bwd", *[None if j == i else a for j, a in enumerate(good)])


def tensor(buf, **kw):
    t = AdamTensor()
    t.p, t.g, t.m, t.v, t.scale, t.copy, t.n, t.bits = buf, buf + 4096, buf + 8192, buf + 16384, buf + 24576, None, 300, 8
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw", [dict(n=-1), dict(n=2 ** 42), dict(p_dtype=5), dict(g_dtype=-1), dict(bits=16), dict(p=None),
                                dict(g=None), dict(m=None), dict(v=None), dict(scale=None), dict(offset="p"), dict(offset="m"),
                                dict(offset="v"), dict(offset="scale")])
def test_adam_tensors(kw, buf):
    """The second of two tensors is refused before the first is touched."""
    kw = dict(kw)
    which = kw.pop("offset", None)
    bad = tensor(buf, **kw)
    if which:
        setattr(bad, which, getattr(bad, which) + 2)
    p = torch.ones(300, device="cuda")
    rest = [torch.zeros(512, device="cuda") for _ in range(4)]
    rest[0].fill_(1)
    good = tensor(buf, p=p.data_ptr(), g=rest[0].data_ptr(), m=rest[1].data_ptr(), v=rest[2].data_ptr(), scale=rest[3].data_ptr())
    two = (AdamTensor * 2)(good, bad)
    with pytest.raises(NottInvalidArgument):
        ops.context().call("nott_adam_multi_step", 1, C.addressof(two), 2, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0)
    torch.cuda.synchronize()
    assert bool((p == 1).all()) and not bool(rest[1].any())


def test_adam_arguments(buf):
    ctx, t = ops.context(), tensor(buf)
    good = [1, C.addressof(t), 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0]
    for i, bad in ((1, None), (2, -1), (3, -1.0), (3, float("nan")), (4, 1.0), (4, -0.1), (5, 1.0), (6, -1.0), (7, -1.0), (8, 0)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_adam_multi_step", *[bad if j == i else a for j, a in enumerate(good)])
    assert ctx.call("nott_adam_multi_step", 1, None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0) == 0
    for hyper, state in ((None, buf), (buf, None)):
        with pytest.raises(NottInvalidArgument):
            ctx.call("nott_adam_multi_step_graph", 1, C.addressof(t), 1, hyper, state, 0, None, 0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_new_context_under_capture(dt):
    """A context without workspace cannot get any under capture: keys that would be split
    are taken whole.  The backward, called once before, replays to the eager bits."""
    b, t, s, h, hk, dh, dv = 2, 1, 4000, 4, 2, 64, 128
    q, k, v = (torch.randn(b, n, c, w, device="cuda").to(dt) for n, c, w in ((t, 2 * h, dh), (s, 2 * hk, dh), (s, hk, dv)))
    lam = torch.rand(h, device="cuda")
    want, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
    do = torch.randn_like(want)
    grads = ops.diff_attention_bwd(do, q, k, v, lam, want, o2, lse)
    d = diff(b=b, h=h, hk=hk, t=t, s=s, dh=dh, dv=dv, scale=dh ** -0.5)
    o, l2, out = torch.zeros_like(want), torch.zeros_like(lse), [torch.zeros_like(x) for x in grads]
    bwd = [C.addressof(d), ops.nott_dtype(dt), *(x.data_ptr() for x in (do, q, k, v, lam)), None, None,
           *(x.data_ptr() for x in (want, o2, lse, *out)), 0]
    ctx = ops.Context(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.call("nott_diff_attention_fwd", C.addressof(d), ops.nott_dtype(dt), *(x.data_ptr() for x in (q, k, v, lam)), None,
                 None, o.data_ptr(), l2.data_ptr(), None)
    assert ctx.workspace_bytes() == 0
    for _ in range(2):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        # sums in another order, and in bf16 probabilities rounded against another maximum (2 maps, each
        # off by a half step of Σ p|v| <= max|v|, and the result's half step)
        u = torch.finfo(dt).eps / 2
        tol = 4 * u * float(v.abs().max()) if dt == torch.bfloat16 else 2.0 ** -12 * float(v.abs().max())
        assert float((o.double() - want.double()).abs().max()) <= tol
        assert torch.allclose(l2, lse, rtol=1e-5, atol=1e-5)
    ctx.call("nott_diff_attention_bwd", *bwd)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        ctx.call("nott_diff_attention_bwd", *bwd)
    for _ in range(2):
        for x in out:
            x.zero_()
        second.replay()
        torch.cuda.synchronize()
        for a, w in zip(out, grads):
            assert torch.equal(a, w)
    del graph, second
    torch.cuda.synchronize()
    del ctx
    gc.collect()


def test_two_streams_at_once():
    """The host layer, whose streams have a context each: calls on two of them leave each
    other's workspace and results alone."""
    from thot_amd import _nott_host as host
    dt = torch.bfloat16
    args = []
    for i in range(2):
        q, k, v = (torch.randn(1, n, c, w, device="cuda").to(dt) for n, c, w in ((2 + i, 8, 64), (6000, 4, 64), (6000, 2, 128)))
        x = torch.randn(2, 9000 + i, 2 * 96, device="cuda").to(dt)
        args.append((q, k, v, torch.rand(4, device="cuda"), x))

    def run(q, k, v, lam, x):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, x)]
        o = host.diff_attention(*leaves[:3], lam)
        h, last = host.linear_scan(leaves[3][..., :96], leaves[3][..., 96:])
        torch.autograd.backward((o, h), (o.detach(), h.detach()))
        return (o.detach(), h.detach(), last.detach(), *(t.grad for t in leaves))
    want = [run(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_cache_behind_the_queries(dt, t):
    """Causal against a cache of which only the first q_start + t keys were written: what
    lies behind them (NaN) reaches neither the output nor the gradients, without lengths."""
    b, s, h, hk, dh, dv = 2, 1100, 2, 1, 32, 64
    start = torch.tensor([5, 700], device="cuda", dtype=torch.int32)
    q, k, v = (torch.randn(b, n, c, w, device="cuda").to(dt) for n, c, w in ((t, 2 * h, dh), (s, 2 * hk, dh), (s, hk, dv)))
    lam = torch.rand(h, device="cuda")

    def run(k, v):
        o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, causal=True, q_start=start, save=True)
        return (o, lse, *ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse, causal=True, q_start=start))
    clean = run(k, v)
    kn, vn = k.clone(), v.clone()
    for i in range(b):
        kn[i, int(start[i]) + t:] = math.nan
        vn[i, int(start[i]) + t:] = math.nan
    for a, w in zip(run(kn, vn), clean):
        assert torch.equal(a, w)
        assert bool(torch.isfinite(a).all())
