"""gated_linear's activations over the whole range of fp32 pre-activations, lowest
finite value and infinities among them (a gate that is masked through its bias), and
their derivatives, against the formulas in float64.  act(−inf) = 0 and act'(±inf)
are the limits.

Tolerances (u = 2^-24): with Z the argument of the exponential (|g|, g²/2, or the
cubic of the tanh form), its roundings put 8·|Z|·u into the result and the rest of
the formula 16·u, relative to the sum of its terms' magnitudes; nothing below 2^-112
is kept."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOOR = 2.0 ** -112
LOW = torch.finfo(torch.float32).min
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def formula(act, g):
    """(act, act', |Z|, magnitude of act' terms), float64, limits at the infinities."""
    g = g.double()
    c = g.clamp(-1e4, 1e4)      # every exponential has ended long before
    if act == "silu":
        e = torch.sigmoid(c)
        a, da, z, mag = c * e, e + c * e * (1 - e), c.abs(), e * (1 + c.abs() * (1 - e))
    elif act == "gelu":
        cdf, pdf = 0.5 * torch.erfc(-c / 2 ** 0.5), torch.exp(-c * c / 2) / (2 * math.pi) ** 0.5
        a, da, z, mag = c * cdf, cdf + c * pdf, c * c / 2, cdf + c.abs() * pdf
    elif act == "gelu_tanh":
        k = 2 * (2 / math.pi) ** 0.5
        z = k * (c + 0.044715 * c ** 3)
        e, slope = torch.sigmoid(z), k * (1 + 3 * 0.044715 * c * c)
        a, da, z, mag = c * e, e + c * e * (1 - e) * slope, z.abs(), e + c.abs() * e * (1 - e) * slope
    elif act == "sigmoid":
        a = torch.sigmoid(c)
        da, z, mag = a * (1 - a), c.abs(), a * (1 - a)
        return a, da, z, mag + a     # 1 − a is a difference of a rounded a
    else:
        a, da, z, mag = c.clamp_min(0), (c > 0).double(), 0 * c, (c > 0).double()
    return torch.where(g > 1e4, g, a), da, torch.where(g.abs() > 1e4, 0.0, z), mag + U * a.abs()


def values():
    far = [10.0 ** e for e in (2, 2.3, 3, 4, 5, 8, 10, 11, 12, 15, 19, 20, 25, 30, 36, 38)]
    v = [0.0, 1e-20, 1e-3, 0.5, 1, 5, 9, 9.5, 10, 13, 14, 15, 30, 40, 60, 79, 80, 80.5, 86, 87, 87.5, 88, 89, 90] + far
    v = v + [-LOW, math.inf]
    return torch.tensor(v + [-x for x in v], device="cuda")


def near(got, want, tol, what):
    inf = torch.isinf(want)
    assert torch.equal(got.double()[inf], want[inf]), what
    err = (got.double() - want).abs()[~inf]
    tol = tol[~inf]
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("act", ACTS)
def test_derivative(act, dt):
    """One row's db is [dh·u·act'(g) | dh·act(g)] itself, in fp32."""
    dt = DT[dt]
    g = values().to(dt)
    f = g.numel()
    gu = torch.cat((g, torch.ones_like(g)))[None].contiguous()
    x, w = torch.zeros((1, 8), device="cuda", dtype=dt), torch.zeros((2 * f, 8), device="cuda", dtype=dt)
    one = torch.ones((1, f), device="cuda", dtype=dt)
    db = ops.gated_linear_bwd(one, x, w, gu, act=act, need_dx=False, need_dw=False)[2]
    torch.cuda.synchronize()
    a, da, z, mag = formula(act, g)
    near(db[f:], a, (16 + 8 * z) * U * a.abs() + FLOOR, "act")
    near(db[:f], da, (16 + 8 * z) * U * mag + FLOOR, "act'")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [2, 40, 200, 2100])
def test_gate_set_by_its_bias(m, act, dt):
    """The forward of every path: few rows, tiles, and fp32 products of pieces."""
    dt = DT[dt]
    g = values()
    g = g.repeat(1024 // g.numel() + 1)[:1024]
    f, d = g.numel(), 768 if m > 2000 else 64
    x, w = torch.zeros((m, d), device="cuda", dtype=dt), torch.zeros((2 * f, d), device="cuda", dtype=dt)
    u = torch.full((f,), 0.25, device="cuda")
    h, gu = ops.gated_linear_fwd(x, w, torch.cat((g, u)), act=act, save=True)
    torch.cuda.synchronize()
    a, _, z, _ = formula(act, g)
    half = torch.finfo(dt).eps / 2
    want = 0.25 * a
    near(h, want.expand(m, f), (((16 + 8 * z) * U + half) * want.abs() + FLOOR).expand(m, f), "h")
    assert torch.equal(gu, torch.cat((g, u)).to(dt).expand(m, 2 * f))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("act", ACTS)
def test_nan_stays(act, dt):
    g = values().to(DT[dt])
    g[3] = math.nan
    f = g.numel()
    x, w = torch.zeros((1, 8), device="cuda", dtype=DT[dt]), torch.zeros((2 * f, 8), device="cuda", dtype=DT[dt])
    one = torch.ones((1, f), device="cuda", dtype=DT[dt])
    db = ops.gated_linear_bwd(one, x, w, torch.cat((g, one[0]))[None].contiguous(), act=act, need_dx=False,
                              need_dw=False)[2]
    hit = torch.zeros(2 * f, dtype=torch.bool, device="cuda")
    hit[3] = hit[f + 3] = True
    assert torch.equal(db.isnan(), hit)
    b = torch.cat((g.float(), torch.ones(f, device="cuda")))
    h, _ = ops.gated_linear_fwd(x, w, b, act=act)
    assert torch.equal(h[0].isnan(), hit[:f])
