"""The host layer's differential attention, gated linear recurrence and optimizer over many
tensors: the bits of thot_amd.ops, gradients only where asked, views, outputs left out."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def host():
    from thot_amd import _nott_host
    return _nott_host


def rnd(*s, dt=torch.float32):
    return torch.randn(s, device="cuda").to(dt)


@pytest.mark.parametrize("token_lam", [False, True])
@pytest.mark.parametrize("dt", DT)
def test_diff_attention_is_the_calls(host, dt, token_lam):
    dt = DT[dt]
    b, t, s, h, hk, dh, dv = 2, 37, 51, 4, 2, 16, 32
    q, k, v = rnd(b, t, 2 * h, dh, dt=dt), rnd(b, s, 2 * hk, dh, dt=dt), rnd(b, s, hk, dv, dt=dt)
    lam = torch.rand((b, t, h) if token_lam else (h,), device="cuda")
    lengths = torch.tensor([51, 20], device="cuda", dtype=torch.int32)
    start = torch.tensor([14, 3], device="cuda", dtype=torch.int32)
    kw = dict(causal=True, scale=0.3, lengths=lengths, q_start=start)
    do = rnd(b, t, h, dv, dt=dt)
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True, **kw)
    want = ops.diff_attention_bwd(do, q, k, v, lam, o, o2, lse, **kw)
    with torch.no_grad():
        assert torch.equal(host.diff_attention(q, k, v, lam, True, 0.3, lengths, start), o)
    # head-major inputs (transposed views) and a gradient whose columns are strided
    hm = [x.transpose(1, 2).contiguous().requires_grad_() for x in (q, k, v)]
    lg = lam.clone().requires_grad_()
    got = host.diff_attention(*(x.transpose(1, 2) for x in hm), lg, True, 0.3, lengths, start)
    assert torch.equal(got, o)
    got.backward(do.transpose(2, 3).contiguous().transpose(2, 3))
    torch.cuda.synchronize()
    for a, w in zip(hm, want):
        assert torch.equal(a.grad.transpose(1, 2), w)
    assert torch.equal(lg.grad, want[3])
    if not token_lam:       # a parameter's gradient is added to; a computed lambda hands its own on
        host.diff_attention(q, k, v, lg, True, 0.3, lengths, start).backward(do)
        torch.cuda.synchronize()
        assert torch.equal(lg.grad, 2 * want[3])
    base = (lam / 2).requires_grad_()
    host.diff_attention(q, k, v, 2 * base, True, 0.3, lengths, start).backward(do)
    torch.cuda.synchronize()
    assert torch.equal(base.grad, 2 * want[3])
    # only keys are trained; lambda is not a leaf and one number for all heads
    one = torch.full((1,), 0.5, device="cuda")
    ks = k.clone().requires_grad_()
    host.diff_attention(q, ks, v, one.expand(h), scale=0.3).backward(do)
    f = ops.diff_attention_fwd(q, k, v, one.repeat(h), scale=0.3, save=True)
    assert torch.equal(ks.grad, ops.diff_attention_bwd(do, q, k, v, one.repeat(h), f[0], f[2], f[1], scale=0.3)[1])
    # 1/sqrt(dh) unless given
    assert torch.equal(host.diff_attention(q, k, v, lam), ops.diff_attention_fwd(q, k, v, lam, scale=0.25)[0])


def test_rows_that_repeat_are_copied(host):
    """An expanded row has strides of zero, which mean contiguous at the C entry."""
    q, v = rnd(1, 1, 1, 8).expand(2, 5, 4, 8), rnd(1, 1, 1, 8).expand(2, 7, 1, 8)
    k, lam = rnd(2, 7, 2, 8), torch.rand(2, device="cuda")
    want = ops.diff_attention_fwd(q.contiguous(), k, v.contiguous(), lam)[0]
    assert torch.equal(host.diff_attention(q, k, v, lam), want)
    x, g = rnd(1, 1, 9).expand(2, 6, 9), rnd(2, 6, 9)
    assert torch.equal(host.linear_scan(x, g)[0], ops.linear_scan_fwd(x.contiguous(), g)[0])
    # and gradients of a sum are such rows too
    q2 = q.contiguous().requires_grad_()
    host.diff_attention(q2, k, v, lam).sum().backward()
    f = ops.diff_attention_fwd(q.contiguous(), k, v.contiguous(), lam, save=True)
    w = ops.diff_attention_bwd(torch.ones_like(f[0]), q.contiguous(), k, v.contiguous(), lam, f[0], f[2], f[1])
    assert torch.equal(q2.grad, w[0])
    x2 = rnd(2, 300, 9).requires_grad_()
    g2 = rnd(2, 300, 9)
    h, last = host.linear_scan(x2, g2)
    (h.sum() + last.sum()).backward()
    f = ops.linear_scan_fwd(x2.detach(), g2, save=True)
    w = ops.linear_scan_bwd(torch.ones_like(f[0]), x2.detach(), g2, f[2], dlast=torch.ones_like(f[1]))
    assert torch.equal(x2.grad, w[0])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("t", [1, 5, 600])
def test_linear_scan_is_the_calls(host, dt, t):
    dt = DT[dt]
    b, d = 3, 40
    xg = rnd(b, t, 2 * d, dt=dt)
    h0, dlast, dh = rnd(b, d), rnd(b, d), rnd(b, t, d, dt=dt)
    reset = torch.rand(b, t, device="cuda") < 0.02
    x, g = xg[..., :d], xg[..., d:]
    for sigmoid, mix in ((True, True), (True, False), (False, False)):
        if not sigmoid:
            xg[..., d:].clamp_(-0.9, 0.9)
        kw = dict(sigmoid=sigmoid, mix=mix, reset=reset)
        h, last, states = ops.linear_scan_fwd(x, g, h0, save=True, **kw)
        leaf, start = xg.clone().requires_grad_(), h0.clone().requires_grad_()
        gh, gl = host.linear_scan(leaf[..., :d], leaf[..., d:], start, reset, sigmoid, mix)
        assert torch.equal(gh, h) and torch.equal(gl, last)
        torch.autograd.backward((gh, gl), (dh, dlast), retain_graph=True)
        want = ops.linear_scan_bwd(dh, x, g, states, dlast=dlast, **kw)
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, torch.cat(want[:2], -1)) and torch.equal(start.grad, want[2])
        # one output alone: the other counts as zeros; a leaf's initial state is added to
        leaf.grad = None
        gl.backward(dlast, retain_graph=True)
        alone = ops.linear_scan_bwd(torch.zeros_like(dh), x, g, states, dlast=dlast, **kw)
        assert torch.equal(leaf.grad, torch.cat(alone[:2], -1)) and torch.equal(start.grad, want[2] + alone[2])
        leaf.grad = None
        gh.backward(dh)
        alone = ops.linear_scan_bwd(dh, x, g, states, **kw)
        assert torch.equal(leaf.grad, torch.cat(alone[:2], -1))
        # an initial state that was computed hands its gradient on
        base = (h0 / 2).requires_grad_()
        host.linear_scan(x, g, 2 * base, reset, sigmoid, mix)[1].backward(dlast)
        alone = ops.linear_scan_bwd(torch.zeros_like(dh), x, g, states, dlast=dlast, **kw)
        assert torch.equal(base.grad, 2 * alone[2])
        with torch.no_grad():
            assert torch.equal(host.linear_scan(x, g, start, reset, sigmoid, mix)[1], last)


def test_nothing_kept_without_a_backward(host):
    """Without gradients, what only the backward reads is neither allocated nor written."""
    q, lam, x = rnd(1, 64, 4, 32), torch.rand(2, device="cuda"), rnd(2, 512, 64)
    v = rnd(1, 64, 2, 64)

    def most(f):
        f()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        r = f()
        held = torch.cuda.memory_allocated() - before
        del r
        return held
    qg, xg = q.clone().requires_grad_(), x.clone().requires_grad_()
    assert most(lambda: host.diff_attention(qg, q, v, lam)) >= most(lambda: host.diff_attention(q, q, v, lam)) + 4 * v.numel()
    assert most(lambda: host.linear_scan(xg, x)) >= most(lambda: host.linear_scan(x, x)) + 4 * 2 * 2 * 64


def test_nothing_to_do(host):
    lam = torch.rand(2, device="cuda").requires_grad_()
    for b, t, s in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (rnd(b, n, c, 8).requires_grad_() for n, c in ((t, 4), (s, 4), (s, 2)))
        o = host.diff_attention(q, k, v, lam, True)
        o.sum().backward()
        assert o.shape == (b, t, 2, 8) and not bool(o.any())
        assert all(x.grad.shape == x.shape and not bool(x.grad.any()) for x in (q, k, v))
    assert not bool(lam.grad.any())
    for b, t in ((0, 3), (2, 0)):
        x, h0 = rnd(b, t, 8).requires_grad_(), rnd(b, 8).requires_grad_()
        h, last = host.linear_scan(x, x, h0)
        (h.sum() + last.sum()).backward()
        assert torch.equal(last, h0) and torch.equal(h0.grad if b else last, torch.ones_like(h0) if b else last)


# ------------------------------------------------------------------ the optimizer
SIZES = ((5,), (300, 7), (256,), (0,), (1000,))


@pytest.mark.parametrize("decoupled", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_is_the_calls(host, decoupled, bits):
    """Two groups, a parameter of bf16, gradients that come and go (so that step counts
    differ), one of them strided: the steps of thot_amd.ops taken one by one."""
    ps = [rnd(*s, dt=torch.bfloat16 if i == 1 else torch.float32).requires_grad_() for i, s in enumerate(SIZES)]
    twin = [p.detach().clone() for p in ps]
    cls = host.MultiTensorAdamW if decoupled else host.MultiTensorAdam
    lrs, wds = [1e-2, 3e-3], [0.0, 0.1]
    opt = cls([ps[:2], ps[2:]], lrs, wds, beta1=0.8, bits=bits)
    held = [ops.AdamMoments([t], bits=bits) if t.numel() else None for t in twin]
    steps = [0] * len(ps)
    for it in range(4):
        if it == 2:
            lrs[1] = 1e-3
            opt.set_lr(1, 1e-3)
        for i, p in enumerate(ps):
            p.grad = None if (it + i) % 3 == 2 else torch.randn_like(p)
            if i == 1 and p.grad is not None:
                p.grad = p.grad.t().contiguous().t()
        opt.step()
        for i, p in enumerate(ps):
            if p.grad is None:
                continue
            steps[i] += 1
            if p.numel():
                ops.adam_multi_step(held[i], [p.grad.contiguous()], lr=lrs[i > 1], weight_decay=wds[i > 1], beta1=0.8,
                                    step=steps[i], decoupled=decoupled)
        torch.cuda.synchronize()
        for i, p in enumerate(ps):
            assert torch.equal(p.detach(), twin[i]) and opt.state_step(p) == steps[i], (it, i)
            if p.numel():
                assert torch.equal(opt.exp_avg(p), held[i].exp_avg(0)) and torch.equal(opt.exp_avg_sq(p), held[i].exp_avg_sq(0))


def test_32_bits_are_the_arena_optimizer(host):
    """The same parameters through the optimizer that keeps them in an arena: the same bits."""
    ps = [rnd(*s).requires_grad_() for s in ((300, 7), (64,), (33,))]
    qs = [p.detach().clone().requires_grad_() for p in ps]
    a = host.MultiTensorAdamW([ps], [1e-2], [0.1])
    b = host.FusedOptimizer([qs], [1e-2], [0.1], True)
    for _ in range(3):
        for p, q in zip(ps, qs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("bits", [8, 32])
def test_saved_and_loaded(host, bits, tmp_path):
    """A loaded state goes on with the same bits; one of other parameters is refused."""
    ps = [rnd(*s).requires_grad_() for s in ((300, 7), (64,))]
    opt = host.MultiTensorAdamW([ps], [1e-2], [0.1], bits=bits)

    def step(o, ps, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device="cuda")
        o.step()
        torch.cuda.synchronize()
    step(opt, ps, 1)
    path = str(tmp_path / "state.pt")
    opt.save(path)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = host.MultiTensorAdamW([qs], [1e-2], [0.1], bits=bits)
    other.load(path)
    for o, x in ((opt, ps), (other, qs)):
        step(o, x, 2)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and other.state_step(qs[0]) == 2
    for wrong in (host.MultiTensorAdamW([qs[:1]], [1e-2], [0.1], bits=bits),
                  host.MultiTensorAdamW([qs], [1e-2], [0.1], bits=40 - bits)):
        with pytest.raises((ValueError, RuntimeError)):
            wrong.load(path)


def test_gradients_cleared_and_scaled(host):
    p = rnd(700).requires_grad_()
    q = p.detach().clone()
    opt = host.MultiTensorAdamW([[p]], [1e-2], [0.0])
    opt.set_fused_zero_grad(True)
    factor = torch.full((1,), 0.25, device="cuda")
    opt.set_grad_scale(factor)
    copy = opt.bf16_copy(p)
    p.grad = rnd(700)
    g = p.grad.clone()
    opt.step()
    m = ops.AdamMoments([q], bits=32)
    ops.adam_multi_step(m, [g / 4], lr=1e-2, step=1)
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), q) and not bool(p.grad.any()) and torch.equal(copy, q.bfloat16())
    opt.set_grad_scale(None)
    p.grad.copy_(g)
    opt.step()
    ops.adam_multi_step(m, [g], lr=1e-2, step=2)
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), q)


def test_optimizer_refusals(host):
    p = rnd(300).requires_grad_()
    W = host.MultiTensorAdamW
    for groups, kw in (([[p]], dict(bits=16)), ([[p, p]], {}), ([[p], [p]], {}), ([[rnd(4).cpu().requires_grad_()]], {}),
                       ([[rnd(4).double().requires_grad_()]], {}), ([[rnd(4, 6).t().requires_grad_()]], {}),
                       ([[p, p.detach()[10:20].requires_grad_()]], {})):
        with pytest.raises((ValueError, RuntimeError)):
            W(groups, [1e-3] * len(groups), [0.0] * len(groups), **kw)
    with pytest.raises(ValueError):
        W([[p]], [1e-3, 1e-3], [0.0])
    opt = W([[p]], [1e-3], [0.0])
    with pytest.raises(ValueError):
        opt.state_step(rnd(3))
    for bad in (torch.ones(1), torch.ones(2, device="cuda"), torch.ones(1, device="cuda").double()):
        with pytest.raises(ValueError):
            opt.set_grad_scale(bad)
    p.grad = rnd(300)
    p.data = rnd(301)[:300].view(300)[:200]
    with pytest.raises(RuntimeError, match="changed"):
        opt.step()
    # nothing trained: no state, no launch
    W([[rnd(3)]], [1e-3], [0.0]).step()


def test_step_is_not_captured(host):
    """The step count is an argument of the launch: a replay would repeat it."""
    p = rnd(300).requires_grad_()
    p.grad = rnd(300)
    opt = host.MultiTensorAdamW([[p]], [1e-3], [0.0])
    opt.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = p.detach() + 1
        with pytest.raises(RuntimeError, match="capture"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, p.detach() + 1) and opt.state_step(p) == 1
