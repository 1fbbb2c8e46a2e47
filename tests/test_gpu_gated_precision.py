"""How many bits gated_linear's gradients keep: dx is rounded once, at its store, and
dw's products see every bit of [dg | du], whatever engine a size takes.

dx: its 2-norm error is that of rounding the float64 result once, with 10% for the
difference of two samples of roundings (at least 2000 elements).  dw: three pieces
of [dg | du] hold its 24 bits, so what is left is the sum: 3·m/16 steps (a matrix
instruction each), each of which rounds a partial sum that is half the final one in
the mean square; a rounding's mean square is u/√3 (u = 2^-24) of it: u·√(m/32), with
4·u for [dg | du] itself; twice that is allowed."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# m, d, f: direct-to-LDS tiles whole and ragged, splits, few rows, narrow layers, odd widths
SHAPES = [(1576, 760, 2024), (512, 256, 512), (300, 520, 200), (2048, 128, 1024), (64, 320, 128), (16, 256, 512),
          (100, 1000, 65), (700, 72, 136), (4000, 40, 33), (515, 257, 1001), (129, 136, 264)]


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("m,d,f", SHAPES)
def test_bf16_gradients(m, d, f):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, dh = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((m, d), (m, f)))
    w = (torch.randn((2 * f, d), generator=g, device="cuda") * d ** -0.5).bfloat16()
    gu = torch.randn((m, 2 * f), generator=g, device="cuda").bfloat16()
    dx, dw, _ = ops.gated_linear_bwd(dh, x, w, gu)
    torch.cuda.synchronize()
    gate, up = gu.double().chunk(2, -1)
    e = torch.sigmoid(gate)
    v = torch.cat((dh.double() * up * e * (1 + gate * (1 - e)), dh.double() * gate * e), 1)
    want = v @ w.double()
    assert off(dx, want) <= 1.1 * off(want.bfloat16(), want)
    want = v.t() @ x.double()
    assert off(dw, want) <= 2 * U * ((m / 32) ** 0.5 + 4)
    # adding to what is there rounds the sum once more
    start = torch.randn((2 * f, d), generator=g, device="cuda")
    acc = start.clone()
    ops.gated_linear_bwd(dh, x, w, gu, dw=acc, need_dx=False, need_db=False, accumulate=True)
    err = (acc.double() - start.double() - dw.double()).abs()
    assert bool((err <= 2 * U * (start.double().abs() + dw.double().abs())).all())
    # each gradient by itself is the same
    assert torch.equal(ops.gated_linear_bwd(dh, x, w, gu, need_dw=False, need_db=False)[0], dx)
    assert torch.equal(ops.gated_linear_bwd(dh, x, w, gu, need_dx=False, need_db=False)[1], dw)
