"""Infinities and NaN in gated_linear's products: what IEEE sums of the products give,
at every size, so also where operands are split into bf16 pieces; and values next to
fp32's largest."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
# the first of each type takes the generic engine, the others tiles of whole or ragged pieces
SHAPES = [(70, 77, 61), (1100, 700, 1300), (2048, 768, 1024), (300, 520, 200)]


def kinds(t):
    """0 finite, 1 NaN, 2 infinity, 3 minus infinity."""
    return t.isnan().int() + 2 * t.isposinf().int() + 3 * t.isneginf().int()


def plant(t, places):
    for (r, c), v in places.items():
        t[r, c] = v
    return t


def make(m, d, f, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, dh = (torch.randn(s, generator=g, device="cuda").to(dt) for s in ((m, d), (m, f)))
    w = (torch.randn((2 * f, d), generator=g, device="cuda") * d ** -0.5).to(dt)
    gu = torch.randn((m, 2 * f), generator=g, device="cuda").to(dt)
    # short values too, whose later pieces are zero
    x[::3] = (x[::3] * 4).round() / 4
    w[::2] = torch.where(w[::2] < 0, -0.5, 0.25).to(dt)
    dh[::2] = dh[::2].sign()
    gu[::2, f:] = gu[::2, f:].sign() * 2
    return x, w, gu, dh


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,d,f", SHAPES)
def test_forward(m, d, f, dt):
    x, w, _, _ = make(m, d, f, DT[dt], m)
    clean = ops.gated_linear_fwd(x, w, save=True)[1]
    plant(x, {(1, 3): math.inf, (3, d - 1): -math.inf, (6, 5): math.nan, (9, 0): math.inf, (9, 8): -math.inf,
              (12, 7): math.inf})
    plant(w, {(5, 2): math.inf, (f + 4, 11): -math.inf, (7, 1): math.nan, (8, 3): math.inf, (10, 7): 0.0})
    gu = ops.gated_linear_fwd(x, w, save=True)[1]
    torch.cuda.synchronize()
    want = x.double() @ w.double().t()
    assert torch.equal(kinds(gu), kinds(want))
    rows, cols = torch.arange(m, device="cuda") > 12, torch.arange(2 * f, device="cuda") > 10
    cols[f + 4] = False
    assert torch.equal(gu[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,d,f", SHAPES)
def test_backward(m, d, f, dt):
    x, w, gu, dh = make(m, d, f, DT[dt], m + 1)
    plant(x, {(2, 3): math.inf, (5, 9): -math.inf, (8, d - 1): math.nan})
    plant(w, {(4, 6): math.inf, (f + 9, 1): -math.inf, (11, 12): math.nan})
    plant(dh, {(20, 5): math.inf, (23, 6): math.nan})
    plant(gu, {(26, f + 3): -math.inf})
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, gu)
    torch.cuda.synchronize()
    gate, up = gu.double().chunk(2, -1)
    e = torch.sigmoid(gate)
    v = torch.cat((dh.double() * up * e * (1 + gate * (1 - e)), dh.double() * gate * e), 1)
    for got, want in ((dx, v @ w.double()), (dw, v.t() @ x.double()), (db, v.sum(0))):
        assert torch.equal(kinds(got), kinds(want))


@pytest.mark.parametrize("m,d,f", SHAPES)
def test_values_next_to_the_largest(m, d, f):
    """3.395e38 to 3.4e38 is finite in fp32 (and infinity in bf16)."""
    x, w, gu, dh = make(m, d, f, torch.float32, m + 2)
    w *= 2.0 ** -20
    top = torch.finfo(torch.float32).max
    plant(x, {(1, 3): top, (4, 5): -top, (7, 6): 3.395e38, (7, 9): -3.395e38})
    got = ops.gated_linear_fwd(x, w, save=True)[1]
    torch.cuda.synchronize()
    want = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    # 22 half steps of each term and d/4 additions, as at any other size
    assert bool(((got.double() - want).abs() <= (0.26 * d + 22) * 2.0 ** -24 * mag).all())
