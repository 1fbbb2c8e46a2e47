"""The gate's gradient where the sigmoid is all but 1 (long memory): σ′ = σ(g)·σ(−g) keeps its
bits, with and without the mixing of the input, since 1 − σ(g) is formed from e^−g.

Per element of dgate = σ′·e·(h_{t−1} [− x]): with u = 2^-24 a sigmoid of either sign is off
by (|g| + 8)·u of itself, so σ′ by twice that; e and h come of a recurrence whose keep
is off by as much at each of the t tokens, three times over (tests of the recurrence), so
by 3·t·(G + 8)·u of the sums of magnitudes at most (all keeps are below 1)."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("mix", [False, True])
@pytest.mark.parametrize("b,t,d", [(1, 5, 64), (2, 40, 37), (2, 300, 64), (1, 1300, 520)])
def test_gradient_of_open_gates(dt, mix, b, t, d):
    dt = DT[dt]
    g = torch.Generator(device="cuda").manual_seed(t)
    x, dh = (torch.randn(b, t, d, generator=g, device="cuda").to(dt) for _ in range(2))
    gate = (torch.rand(b, t, d, generator=g, device="cuda") * 70 + 10).to(dt)
    gate[:, ::4] *= -0.1        # (some shut, so that the state does not grow with t)
    h0 = torch.randn(b, d, generator=g, device="cuda")
    h, _, states = ops.linear_scan_fwd(x, gate, h0, mix=mix, save=True)
    _, dgate, _ = ops.linear_scan_bwd(dh, x, gate, states, mix=mix)
    torch.cuda.synchronize()
    gd, xd = gate.double(), x.double()
    a, rest = torch.sigmoid(gd), torch.sigmoid(-gd)
    take = rest if mix else torch.ones_like(a)
    y, yh = [h0.double()], [h0.double().abs()]
    for i in range(t):
        y.append(a[:, i] * y[-1] + take[:, i] * xd[:, i])
        yh.append(a[:, i] * yh[-1] + (take[:, i] * xd[:, i]).abs())
    before, bh = torch.stack(y[:-1], 1), torch.stack(yh[:-1], 1)
    e, eh = [dh[:, -1].double()], [dh[:, -1].double().abs()]
    for i in reversed(range(t - 1)):
        e.append(dh[:, i].double() + a[:, i + 1] * e[-1])
        eh.append(dh[:, i].double().abs() + a[:, i + 1] * eh[-1])
    e, eh = torch.stack(e[::-1], 1), torch.stack(eh[::-1], 1)
    if mix:
        before, bh = before - xd, bh + xd.abs()
    want = a * rest * e * before
    c = U * (80 + 8)
    tol = a * rest * eh * bh * (2 * 3 * t * c + 2 * c + 8 * U) + 1e-38
    if dt == torch.bfloat16:
        tol = tol + 2.0 ** -8 * 1.01 * (want.abs() + tol)
    err = (dgate.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert bool(dgate[gate > 17].any())
