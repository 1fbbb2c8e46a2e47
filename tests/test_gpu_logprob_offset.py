"""token_logprob of rows whose logits share a large offset, as masks of −1e9 or
−1e12 over a whole row leave them: log probabilities and entropy depend on the
differences to the row's maximum alone.

Tolerances count roundings (u = 2^-24): the difference to the maximum, its product
with the scale and the scale's own rounding put 3·|z − m|·u into an exponent, and a
sum of c exponentials is a chain of at most c/256 + 32 additions; the final
difference is (|z_y − m| + log c) rounded twice.  Only the log-sum-exp carries |m|·u."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def reference(z, y, scale):
    """logprob of every token, entropy, log-sum-exp, Σ p·|z − m| and |z − m|, float64."""
    d = (z.double() - z.double().amax(1, keepdim=True)) * scale
    s = d.exp().sum(1, keepdim=True).log()
    lp = d - s
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    spread = torch.where(p > 0, p * d.abs(), 0.0).sum(1)
    return lp, ent, z.double().amax(1) * scale + s[:, 0], spread, d.abs()


def check(z, y, scale, top=4):
    n, c = z.shape
    top = min(top, c)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    lp, ent, lse, tv, ti = ops.token_logprob_fwd(z, y, scale=scale, top=top)
    torch.cuda.synchronize()
    rlp, rent, rlse, spread, far = reference(z, y, s32)
    base = (4 * spread + c / 256 + 64) * U
    hit = rlp.gather(1, y[:, None])[:, 0]

    def near(got, want, tol, what):
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"
    near(lp, hit, base + 4 * U * (far.gather(1, y[:, None])[:, 0] + hit.abs()), "logprob")
    assert bool((lp <= 0).all() | (lp <= base).all())
    near(ent, rent, base * (1 + spread) + 2 * U * rent, "entropy")
    near(lse, rlse, base + 2 * U * (rlse.abs() + z.double().amax(1).abs() * s32), "lse")
    want = z.float().double().sort(dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti, want)
    near(tv, rlp.gather(1, want), base[:, None] + 4 * U * (far.gather(1, want) + rlp.gather(1, want).abs()), "top")


SHAPES = [(1, 1), (4, 100), (3, 1001), (700, 700), (2000, 3001), (2, 128256)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("offset", [1e3, -1e4, 1e6])
@pytest.mark.parametrize("n,c", SHAPES)
def test_common_offset(n, c, offset, dt):
    g = torch.Generator(device="cuda").manual_seed(3)
    z = (torch.randn((n, c), generator=g, device="cuda") + offset).to(DT[dt])
    y = torch.randint(0, c, (n,), generator=g, device="cuda")
    for scale in (1.0, 0.7):
        check(z, y, scale)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("value", [-1e8, -1e9, 1e9, -1e10, -1e11, -1e12, -1e28, 1e30, 3.3e38])
@pytest.mark.parametrize("n,c", SHAPES)
def test_equal_logits_of_any_size(n, c, value, dt):
    """−log c for every token, none of them masked."""
    z = torch.full((n, c), value, device="cuda").to(DT[dt])
    y = torch.arange(n, device="cuda") % c
    check(z, y, 1.0)


@pytest.mark.parametrize("dt", DT)
def test_one_live_token_in_a_masked_row(dt):
    """A row masked with −1e9 but for one or two tokens, and the same row wholly masked."""
    n, c = 6, 5003
    z = torch.full((n, c), -1e9, device="cuda")
    z[0, 7] = 2.0
    z[1, 7], z[1, 4000] = 2.0, 2.0
    z[2, 9] = -1e9 * 2
    z = z.to(DT[dt])
    y = torch.tensor([7, 4000, 9, 0, 1, c - 1], device="cuda")
    check(z, y, 1.0)
    lp, ent, _, _, _ = ops.token_logprob_fwd(z, y)
    assert float(lp[0]) == 0.0 and float(ent[0]) == 0.0
    assert abs(float(lp[1]) + math.log(2)) <= 4 * U and float(lp[2]) <= -1e8
