"""linear_scan (a gated linear recurrence and its gradients) against the recurrence in
float64, token by token.

Tolerances.  u = 2^-24, G the largest |gate| that a sigmoid takes (0 otherwise).  A gate
is off by (G + 8)·u of itself: its exponent's argument is rounded, then exponential,
sum and reciprocal (value gates are exact).  With H the recurrence of absolute values,
H_t = |keep|·H_{t−1} + |take·x|, each step adds at most (G + 8)·u·H_t to what the error
before it becomes; a token is gone through three times (its span's map, the fold of the
maps, the span again), so E_t = |keep|·E_{t−1} + 3·(G + 8)·u·H_t.  The gradient of the
state is the same recurrence in reverse.  Products of two such values carry each other's
error.  Outputs are rounded once."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
MODES = [(True, True), (True, False), (False, False), (False, True)]
# tokens: one, a few (no tiles), around a tile, several tiles, several segments; channels:
# whole groups, less than a workgroup's, past it, odd
SHAPES = [(1, 1, 8), (3, 1, 72), (2, 16, 64), (2, 17, 64), (1, 255, 40), (2, 256, 128), (3, 257, 72), (2, 700, 65),
          (1, 1300, 520), (2, 2500, 72), (1, 5000, 33), (1, 2304, 9000)]


def make(b, t, d, dt, sigmoid, seed=0, resets=False, packed=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*s, dtype=dt):
        return torch.randn(s, generator=g, device="cuda").to(dtype)
    p = n(b, t, 2 * d)
    gate, x = (p[..., :d], p[..., d:]) if packed else (p[..., :d].contiguous(), p[..., d:].contiguous())
    if sigmoid:
        gate.mul_(2).add_(2)
    else:
        gate.copy_((torch.sigmoid(gate.float() + 3) * torch.randn_like(gate.float()).sign()).to(dt))
    reset = torch.rand((b, t), generator=g, device="cuda") < 0.02 if resets else None
    return x, gate, n(b, d, dtype=torch.float32), reset


def gates(gate, sigmoid, mix, reset):
    g = gate.double()
    a = torch.sigmoid(g) if sigmoid else g
    take = (torch.sigmoid(-g) if sigmoid else 1 - g) if mix else torch.ones_like(g)
    keep = a if reset is None else torch.where(reset[..., None], 0.0, a)
    return a, keep, take


def scan(keep, u, first):
    """All states, [first] included, along dim 1."""
    out = [first]
    for i in range(keep.shape[1]):
        out.append(keep[:, i] * out[-1] + u[:, i])
    return torch.stack(out, 1)


def reference(x, gate, h0, reset, sigmoid, mix):
    a, keep, take = gates(gate, sigmoid, mix, reset)
    c = 3 * U * ((gate.double().abs().max() if sigmoid else 0.0) + 8)
    y = scan(keep, take * x.double(), h0.double())
    hi = scan(keep.abs(), (take * x.double()).abs(), h0.double().abs())
    er = scan(keep.abs(), c * hi[:, 1:], torch.zeros_like(h0.double()))
    return a, keep, take, y, hi, er, c


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    tol = tol + (torch.finfo(got.dtype).eps / 2 * want.abs() * 1.01 if got.dtype != torch.float32 else 0) + 1e-38
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("sigmoid,mix", MODES)
@pytest.mark.parametrize("b,t,d", SHAPES)
def test_forward_and_backward(b, t, d, sigmoid, mix, dt):
    dt = DT[dt]
    resets = (t + d) % 2 == 0
    x, gate, h0, reset = make(b, t, d, dt, sigmoid, resets=resets, packed=d != 128)
    h, last, states = ops.linear_scan_fwd(x, gate, h0, sigmoid=sigmoid, mix=mix, reset=reset, save=True)
    a, keep, take, y, hi, er, c = reference(x, gate, h0, reset, sigmoid, mix)
    torch.cuda.synchronize()
    close(h, y[:, 1:], er[:, 1:], "h")
    close(last, y[:, -1], er[:, -1], "last")
    close(states, y[:, :-1:256], er[:, :-1:256], "states")
    g = torch.Generator(device="cuda").manual_seed(9)
    dh = torch.randn((b, t, d), generator=g, device="cuda").to(dt)
    dlast = torch.randn((b, d), generator=g, device="cuda")
    dx, dgate, dh0 = ops.linear_scan_bwd(dh, x, gate, states, sigmoid=sigmoid, mix=mix, reset=reset, dlast=dlast)
    torch.cuda.synchronize()
    # c_t = keep_t·(dh_t + c_{t+1}); e_t = dh_t + c_{t+1}

    cs = [dlast.double()]
    ch = [dlast.double().abs()]
    ce = [torch.zeros_like(cs[0])]
    for i in reversed(range(t)):
        k, v = keep[:, i], dh[:, i].double()
        cs.append(k * (v + cs[-1]))
        ch.append(k.abs() * (v.abs() + ch[-1]))
        ce.append(k.abs() * ce[-1] + c * ch[-1])
    cs, ch, ce = (torch.stack(v[::-1], 1) for v in (cs, ch, ce))
    e, eh, ee = dh.double() + cs[:, 1:], dh.double().abs() + ch[:, 1:], ce[:, 1:] + c * (dh.double().abs() + ch[:, 1:])
    before, bh, be = y[:, :-1], hi[:, :-1], er[:, :-1]
    if reset is not None:
        before, bh, be = (torch.where(reset[..., None], 0.0, v) for v in (before, bh, be))
    if mix:
        before, bh = before - x.double(), bh + x.double().abs()
    w = a * (1 - a) if sigmoid else torch.ones_like(a)
    close(dx, take * e, take.abs() * (ee + c * eh), "dx")
    if sigmoid and not mix:     # 1 − a is a difference there: off by u/2 of 1
        wt = a * (c * (1 - a) + c)
    else:
        wt = c * w
    close(dgate, e * before * w, w * (ee * bh + eh * be + c * eh * bh) + wt * eh * bh, "dgate")
    close(dh0, cs[:, 0], ce[:, 0] + c * ch[:, 0], "dh0")


def test_initial_state_and_final_gradient_left_out():
    x, gate, h0, _ = make(2, 300, 64, torch.bfloat16, True)
    a = ops.linear_scan_fwd(x, gate, save=True)
    b = ops.linear_scan_fwd(x, gate, torch.zeros_like(h0), save=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    dh = torch.randn_like(x)
    c = ops.linear_scan_bwd(dh, x, gate, a[2])
    e = ops.linear_scan_bwd(dh, x, gate, a[2], dlast=torch.zeros_like(h0))
    assert all(torch.equal(p, q) for p, q in zip(c, e))
    assert ops.linear_scan_fwd(x, gate)[2] is None


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("t", [16, 300, 2500])
def test_in_pieces(dt, t):
    """A sequence taken token by token, or in two parts, through its state."""
    dt = DT[dt]
    x, gate, h0, _ = make(2, t, 72, dt, True, seed=4)
    whole, last, _ = ops.linear_scan_fwd(x, gate, h0)
    _, _, _, _, _, er, _ = reference(x, gate, h0, None, True, True)
    cut = t // 2
    a, s, _ = ops.linear_scan_fwd(x[:, :cut], gate[:, :cut], h0)
    b, s, _ = ops.linear_scan_fwd(x[:, cut:], gate[:, cut:], s)
    close(torch.cat((a, b), 1), whole.double(), 2 * er[:, 1:] + torch.finfo(dt).eps * whole.double().abs(), "two parts")
    close(s, last.double(), 2 * er[:, -1], "state")
    if t == 16:
        s = h0
        for i in range(t):
            o, s, _ = ops.linear_scan_fwd(x[:, i:i + 1], gate[:, i:i + 1], s)
            close(o, whole[:, i:i + 1].double(), 2 * er[:, i + 1:i + 2] + torch.finfo(dt).eps * o.double().abs(), "step")


@pytest.mark.parametrize("t", [10, 400, 3000])
def test_sequences_do_not_reach_each_other(t):
    """Infinities and NaN before a reset stay there, forward and backward."""
    x, gate, h0, _ = make(1, t, 64, torch.float32, True, seed=2)
    cut = t // 2 + 1
    reset = torch.zeros((1, t), dtype=torch.bool, device="cuda")
    reset[0, cut] = True
    dirty = x.clone()
    dirty[0, cut - 3] = math.inf
    dirty[0, cut - 2] = -math.inf
    clean = ops.linear_scan_fwd(x, gate, h0, reset=reset, save=True)
    got = ops.linear_scan_fwd(dirty, gate, h0, reset=reset, save=True)
    assert got[0][0, cut - 1].isnan().all()
    assert torch.equal(got[0][:, cut:], clean[0][:, cut:]) and torch.equal(got[1], clean[1])
    dh = torch.randn_like(x.contiguous())
    want = ops.linear_scan_bwd(dh, x, gate, clean[2], reset=reset)
    dh[0, cut + 1] = math.nan
    dx, dg, dh0 = ops.linear_scan_bwd(dh, x, gate, clean[2], reset=reset)
    assert dx[0, cut].isnan().all()
    assert torch.equal(dx[:, :cut], want[0][:, :cut]) and torch.equal(dg[:, :cut], want[1][:, :cut])
    assert torch.equal(dh0, want[2])


@pytest.mark.parametrize("t", [7, 300])
def test_gates_of_infinity(t):
    """+inf keeps the state and, mixing, takes nothing in: padding; −inf forgets it."""
    x, gate, h0, _ = make(2, t, 64, torch.bfloat16, True, seed=3)
    gate[:, 4:] = math.inf
    h, last, _ = ops.linear_scan_fwd(x, gate, h0)
    assert torch.equal(last.bfloat16(), h[:, 3]) and torch.equal(h[:, 4:], h[:, 3:4].expand(-1, t - 4, -1))
    gate[:, 2] = -math.inf
    h, _, _ = ops.linear_scan_fwd(x, gate, h0)
    assert torch.equal(h[:, 2], x[:, 2])


def test_gradients_against_differences():
    b, t, d = 1, 40, 8
    for sigmoid, mix in MODES:
        x, gate, h0, reset = make(b, t, d, torch.float32, sigmoid, seed=5, resets=True)
        w = torch.randn(b, t, d, device="cuda")
        wl = torch.randn(b, d, device="cuda")

        def loss(x, gate, h0):
            y = scan(*(lambda a, k, tk: (k, tk * x.double()))(*gates(gate, sigmoid, mix, reset)), h0.double())
            return float((y[:, 1:] * w.double()).sum() + (y[:, -1] * wl.double()).sum())
        _, _, states = ops.linear_scan_fwd(x, gate, h0, sigmoid=sigmoid, mix=mix, reset=reset, save=True)
        grads = ops.linear_scan_bwd(w, x, gate, states, sigmoid=sigmoid, mix=mix, reset=reset, dlast=wl)
        for k, (v, gr) in enumerate(zip((x, gate, h0), grads)):
            way = torch.randn_like(v.contiguous()).double()
            args = [x.double(), gate.double(), h0.double()]
            step = 1e-5
            up, down = (loss(*[q + s * step * way if i == k else q for i, q in enumerate(args)]) for s in (1, -1))
            # differences are off by step²·(third derivative, of the size of the sums) and roundings
            assert abs((up - down) / (2 * step) - float((gr.double() * way).sum())) <= 1e-3 * (1 + float((gr.double() * way).norm()))


def test_given_outputs_and_strides():
    """Views of a packed gradient, outputs in place of inputs, a batch that is not the outer dimension."""
    b, t, d = 3, 300, 64
    x, gate, h0, _ = make(b, t, d, torch.bfloat16, True, seed=6)
    want, last, states = ops.linear_scan_fwd(x, gate, h0, save=True)
    dh = torch.randn_like(want)
    ref = ops.linear_scan_bwd(dh, x, gate, states)
    packed = torch.full((b, t, 2 * d + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.linear_scan_bwd(dh, x, gate, states, out=(packed[..., d:2 * d], packed[..., :d]))
    assert torch.equal(packed[..., d:2 * d], ref[0]) and torch.equal(packed[..., :d], ref[1])
    assert bool((packed[..., 2 * d:] == 7).all()) and torch.equal(got[2], ref[2])
    # time outermost
    xt, gt = x.transpose(0, 1).contiguous().transpose(0, 1), gate.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.linear_scan_fwd(xt, gt, h0)[0], want)
    # in place
    e1, x1, g1 = dh.clone(), x.clone(), gate.clone()
    ops.linear_scan_bwd(e1, x1, g1, states, out=(e1, g1))
    assert torch.equal(e1, ref[0]) and torch.equal(g1, ref[1])
    x2 = x.contiguous()
    ops.linear_scan_fwd(x2, gate, h0, out=x2)
    assert torch.equal(x2, want)
    # rows that are not aligned give what aligned ones give, but for the order of sums
    odd = torch.empty(b, t, 2 * d + 1, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:1 + d], odd[..., 1 + d:] = gate, x
    o = ops.linear_scan_fwd(odd[..., 1 + d:], odd[..., 1:1 + d], h0)
    assert bool(((o[0].float() - want.float()).abs() <= 2.0 ** -7 * (want.float().abs() + 1e-3)).all())


def test_in_place_over_segments():
    """Few channels and much time: the maps of all segments are read before anything is written."""
    x, gate, h0, _ = make(1, 4000, 64, torch.float32, True, seed=8)
    want, _, states = ops.linear_scan_fwd(x, gate, h0, save=True)
    y = x.contiguous()
    ops.linear_scan_fwd(y, gate, h0, out=y)
    dh = torch.randn_like(want)
    ref = ops.linear_scan_bwd(dh, x, gate, states)
    e, g = dh.clone(), gate.contiguous()
    ops.linear_scan_bwd(e, x, g, states, out=(e, g))
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(e, ref[0]) and torch.equal(g, ref[1])


def test_nothing_to_do():
    h0 = torch.randn(2, 8, device="cuda")
    x = torch.empty(2, 0, 8, device="cuda")
    h, last, states = ops.linear_scan_fwd(x, x, h0, save=True)
    assert h.numel() == 0 and torch.equal(last, h0) and states.numel() == 0
    dx, dg, dh0 = ops.linear_scan_bwd(x, x, x, states, dlast=h0)
    assert dx.numel() == 0 and torch.equal(dh0, h0)
    assert torch.equal(ops.linear_scan_fwd(x, x)[1], torch.zeros_like(h0))
    y = torch.empty(0, 5, 8, device="cuda")
    assert ops.linear_scan_fwd(y, y)[0].numel() == 0


def test_captured_and_on_another_stream():
    """Two graphs on one context (they share its workspace) replayed in turn, with eager work between."""
    shapes = [(1, 4000, 64), (2, 3000, 40)]
    runs = []
    s = torch.cuda.Stream()
    for k, (b, t, d) in enumerate(shapes):
        x, gate, h0, _ = make(b, t, d, torch.float32, True, seed=k)
        x, gate = x.contiguous(), gate.contiguous()
        dh = torch.randn_like(x)

        def work(x=x, gate=gate, h0=h0, dh=dh):
            h, last, st = ops.linear_scan_fwd(x, gate, h0, save=True)
            return (h, last) + ops.linear_scan_bwd(dh, x, gate, st, dlast=last)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = work()
        runs.append((graph, out, work, x))
    for i in range(3):
        for graph, out, work, x in runs:
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            got = [v.clone() for v in out]
            for a, b in zip(got, work()):
                assert torch.equal(a, b), i


def test_no_workspace_under_capture():
    """A context that cannot get its workspace takes time whole."""
    x, gate, h0, _ = make(1, 4000, 64, torch.float32, True)
    x, gate = x.contiguous(), gate.contiguous()
    want = ops.linear_scan_fwd(x, gate, h0)
    _, _, _, _, _, er, _ = reference(x, gate, h0, None, True, True)
    h, last = torch.empty_like(x), torch.empty_like(h0)
    ctx = ops.Context(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    desc = ops._SCAN.pack(1, 4000, 64, *[0] * 10, 1, 1)
    with torch.cuda.graph(graph):
        ctx.call("nott_linear_scan_fwd", desc, 0, x.data_ptr(), gate.data_ptr(), h0.data_ptr(), None, h.data_ptr(),
                 last.data_ptr(), None)
    assert ctx.workspace_bytes() == 0
    graph.replay()
    torch.cuda.synchronize()
    close(h, want[0].double(), 2 * er[:, 1:], "h")
    del graph
