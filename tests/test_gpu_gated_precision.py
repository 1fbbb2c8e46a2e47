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


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid"])
def test_bf16_gradients_match_differences(act):
    """Against central differences of the formula at the forward's own [g | u], which short
    inputs leave exact in bf16: dx within its rounding (2^-8 of each element), dw and db
    within 2^-20 of their terms; h²·f'''/6 and 2^-53/h leave about 1e-9."""
    m, d, f = 150, 136, 144
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randint(0, 40, (m, d), generator=g, device="cuda") == 0).double() * 0.5
    w = torch.randint(-3, 4, (2 * f, d), generator=g, device="cuda").double() / 2
    b = torch.randint(-4, 5, (2 * f,), generator=g, device="cuda").double() / 4
    dh = torch.randn((m, f), generator=g, device="cuda").bfloat16()
    gu = ops.gated_linear_fwd(x.bfloat16(), w.bfloat16(), b.float(), act=act, save=True)[1]
    assert torch.equal(gu.double(), x @ w.t() + b)
    grads = ops.gated_linear_bwd(dh, x.bfloat16(), w.bfloat16(), gu, act=act)
    F = torch.nn.functional
    fn = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "sigmoid": torch.sigmoid}[act]

    def value(x, w, b):
        gate, up = (x @ w.t() + b).chunk(2, -1)
        return (fn(gate) * up * dh.double()).sum()
    at = [x, w, b]
    for i, grad in enumerate(grads):
        v, h = torch.randn(at[i].shape, generator=g, device="cuda").double(), 1e-5
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - h * v, at[i] + h * v
        diff = (value(*hi) - value(*lo)) / (2 * h)
        tol = 2.0 ** (-8 if i == 0 else -20) * float((grad.double() * v).abs().sum()) + 1e-6 * float(grad.norm())
        assert abs(float((grad.double() * v).sum() - diff)) <= tol
