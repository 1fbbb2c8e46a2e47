"""Gates whose product over time leaves fp32's range: only a gate of exactly 0 (a reset, a
sigmoid's gate of −infinity) forgets, however small the product of the others has become.

The recurrence token by token in float64 says where the outputs are NaN and infinite, and
what they are elsewhere.  Tolerances as for the recurrence itself: a gate is off by
(G + 8)·u of itself, u = 2^-24, G the largest |gate| of a sigmoid, and a token is gone
through three times, so E_t = |keep|·E_{t−1} + 3·(G + 8)·u·H_t with H the recurrence of
absolute values, plus fp32's least number (2^-149) of the largest state for a product
that fp32 does not hold."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rand(*s, seed=0, dt=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(s, generator=g, device="cuda").to(dt)


def along(keep, u, first):
    """first and all states of y_t = keep_t·y_{t−1} + u_t; a keep of 0 forgets."""
    out = [first]
    for i in range(keep.shape[1]):
        k = keep[:, i]
        out.append(torch.where(k == 0, 0.0, k * out[-1]) + u[:, i])
    return torch.stack(out, 1)


def same(got, want, tol, what):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN at other places"
    over = want.abs() > 3.4e38
    assert torch.equal(got[over].sign(), want[over].sign()) and bool(got[over].isinf().all()), f"{what}: infinities"
    ok = want.isfinite() & ~over
    assert bool(((got - want).abs() <= tol)[ok].all()), what


def check(x, gate, h0, dh, dlast, sigmoid, mix, reset=None):
    h, last, states = ops.linear_scan_fwd(x, gate, h0, sigmoid=sigmoid, mix=mix, reset=reset, save=True)
    dx, dgate, dh0 = ops.linear_scan_bwd(dh, x, gate, states, sigmoid=sigmoid, mix=mix, reset=reset, dlast=dlast)
    torch.cuda.synchronize()
    g, xd = gate.double(), x.double()
    a = torch.sigmoid(g) if sigmoid else g
    take = (torch.sigmoid(-g) if sigmoid else 1 - g) if mix else torch.ones_like(g)
    keep = a if reset is None else torch.where(reset[..., None], 0.0, a)
    c = 3 * U * ((g[g.isfinite()].abs().max() if sigmoid else 0.0) + 8)
    half = torch.finfo(x.dtype).eps / 2 * 1.01 if x.dtype == torch.bfloat16 else U

    def fin(v):
        return torch.where(v.isfinite(), v, 0.0).abs()
    y = along(keep, take * xd, h0.double())
    hi = along(fin(keep), fin(take * xd), fin(h0.double()))
    er = along(fin(keep), c * hi[:, 1:] + 2.0 ** -149 * hi.amax(1, keepdim=True), torch.zeros_like(hi[:, 0]))
    same(h, y[:, 1:], er[:, 1:] + half * y[:, 1:].abs() + 1e-38, "h")
    same(last, y[:, -1], er[:, -1] + 1e-38, "last")
    same(states, y[:, :-1:256], er[:, :-1:256] + 1e-38, "states")
    # the state's gradient, in reverse: e_t = dh_t + keep_{t+1}·e_{t+1}
    e = dh.double().clone()
    e[:, -1] += dlast.double()
    later = torch.cat((keep[:, 1:], torch.zeros_like(keep[:, :1])), 1)
    es = along(later.flip(1), e.flip(1), torch.zeros_like(e[:, 0]))[:, 1:].flip(1)
    eh = along(fin(later).flip(1), fin(e).flip(1), torch.zeros_like(e[:, 0]))[:, 1:].flip(1)
    ee = along(fin(later).flip(1), c * eh.flip(1) + 2.0 ** -149 * eh.amax(1, keepdim=True), torch.zeros_like(e[:, 0]))[:, 1:].flip(1)
    same(dx, take * es, take * ee + (c + half) * take * eh + 1e-38, "dx")
    first = torch.where(keep[:, 0] == 0, 0.0, keep[:, 0] * es[:, 0])
    same(dh0, first, fin(keep[:, 0]) * ee[:, 0] + c * fin(first) + 1e-38, "dh0")
    return h, last, dx, dgate, dh0


# the product of 2 gates, of a workgroup's share of a tile, of a tile, of a segment is below 2^-150
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("value,t,d", [(1e-30, 8, 64), (1e-30, 300, 64), (0.001, 300, 37), (0.02, 300, 64), (0.5, 520, 64),
                                       (0.02, 2100, 64), (0.9, 2600, 64), (0.9, 2600, 37)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_state_that_is_not_finite_stays(dt, t, d, value, bad):
    """In h0 and dlast: in every output behind them, or before."""
    dt = DT[dt]
    x, dh = rand(2, t, d, seed=1, dt=dt), rand(2, t, d, seed=2, dt=dt)
    gate = torch.full((2, t, d), value, device="cuda", dtype=dt)
    gate[:, :, 1::3] *= -1
    h0, dlast = rand(2, d, seed=3), rand(2, d, seed=4)
    h0[:, ::2] = bad
    dlast[:, ::2] = -bad
    h, last, dx, _, dh0 = check(x, gate, h0, dh, dlast, False, False)
    assert not last[:, ::2].isfinite().any() and not dh0[:, ::2].isfinite().any()
    assert bool(last[:, 1::2].isfinite().all()) and bool(dh0[:, 1::2].isfinite().all())
    # and from a token in the middle
    h0, dlast = rand(2, d, seed=3), rand(2, d, seed=4)
    x[:, t // 3, ::2], dh[:, t // 2, ::2] = bad, bad
    h, _, dx, _, _ = check(x, gate, h0, dh, dlast, False, False)
    assert not h[:, t // 3:, ::2].isfinite().any() and not dx[:, :t // 2 + 1, ::2].isfinite().any()
    assert bool(h[:, :t // 3].isfinite().all())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("value,t", [(-60.0, 8), (-95.0, 300), (-300.0, 8), (-300.0, 300), (-2.0, 2100)])
@pytest.mark.parametrize("mix", [False, True])
def test_through_a_sigmoid(dt, value, t, mix):
    """A sigmoid is 0 at −infinity alone, where the state is forgotten."""
    dt = DT[dt]
    x, dh = rand(2, t, 64, seed=1, dt=dt), rand(2, t, 64, seed=2, dt=dt)
    gate = torch.full((2, t, 64), value, device="cuda", dtype=dt)
    h0, dlast = rand(2, 64, seed=3), rand(2, 64, seed=4)
    h0[:, ::2], dlast[:, ::2] = math.nan, math.nan
    h, last, dx, dgate, dh0 = check(x, gate, h0, dh, dlast, True, mix)
    assert h[:, :, ::2].isnan().all() and dx[:, :, ::2].isnan().all() and dgate[:, :, ::2].isnan().all()
    gate[:, t // 2] = -math.inf
    h, last, dx, _, dh0 = check(x, gate, h0, dh, dlast, True, mix)
    assert bool(h[:, t // 2:].isfinite().all()) and bool(dx[:, :t // 2].isfinite().all()) and bool(dh0.isfinite().all())


@pytest.mark.parametrize("t", [300, 2100])
def test_resets_among_small_gates(t):
    x, dh = rand(2, t, 64, seed=1), rand(2, t, 64, seed=2)
    gate = torch.full((2, t, 64), 0.01, device="cuda")
    h0, dlast = rand(2, 64, seed=3), rand(2, 64, seed=4)
    h0[:, ::2], dlast[:, ::2] = math.nan, math.inf
    reset = torch.zeros(2, t, dtype=torch.bool, device="cuda")
    reset[0, t // 2] = True
    h, last, dx, _, dh0 = check(x, gate, h0, dh, dlast, False, True, reset)
    assert bool(h[0, t // 2:].isfinite().all()) and h[1, :, ::2].isnan().all()


@pytest.mark.parametrize("value,t", [(1e-30, 300), (0.02, 300), (0.5, 2100), (0.9, 2600)])
def test_large_states_decay(value, t):
    x, dh = rand(1, t, 64, seed=1), rand(1, t, 64, seed=2)
    gate = torch.full((1, t, 64), value, device="cuda")
    check(x, gate, rand(1, 64, seed=3) * 1e37, dh, rand(1, 64, seed=4) * 1e37, False, False)


def test_growth_from_a_state_of_zero():
    """Gates above 1, whose product over a segment of time overflows, before anything has come in."""
    t, d = 2100, 64
    x, dh = torch.zeros(1, t, d, device="cuda"), torch.zeros(1, t, d, device="cuda")
    x[:, -100:], dh[:, :100] = rand(1, 100, d, seed=1), rand(1, 100, d, seed=2)
    gate = torch.full((1, t, d), 1.2, device="cuda")
    zero = torch.zeros(1, d, device="cuda")
    h, *_ = check(x, gate, zero, dh, zero, False, False)
    assert not h[:, :-100].any() and bool(h[:, -1].isfinite().all())
