"""Differential attention over nothing: an empty batch has a gradient of zero for lambda, keys
and values that no head reads gradients of zero."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rnd(*s, dt=torch.float32):
    return torch.randn(s, device="cuda").to(dt)


def spoil_freed_memory():
    """What an allocation of a few bytes gets next holds no zeros."""
    for n in (1, 2, 4, 64, 128, 1024):
        rnd(n).fill_(7.0)


@pytest.mark.parametrize("dt", DT)
def test_empty_batch(dt):
    dt = DT[dt]
    q, k, v, lam = rnd(0, 3, 8, 16, dt=dt), rnd(0, 5, 4, 16, dt=dt), rnd(0, 5, 2, 32, dt=dt), torch.rand(4, device="cuda")
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
    held = torch.full_like(lam, 7.0)
    got = ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse, dlam=held)
    assert got[3] is held and not held.any() and all(x.numel() == 0 for x in got[:3])
    held.fill_(7.0)
    ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse, dlam=held, accumulate=True)
    assert bool((held == 7.0).all())
    spoil_freed_memory()
    assert not ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse)[3].any()


@pytest.mark.parametrize("dt", DT)
def test_empty_batch_under_autograd(dt):
    """A lambda that was computed from a parameter, as it usually is."""
    from thot_amd import _nott_host as host
    dt = DT[dt]
    q, k, v = (rnd(0, n, c, 16, dt=dt).requires_grad_() for n, c in ((3, 8), (5, 4), (5, 2)))
    base = torch.rand(4, device="cuda").requires_grad_()
    spoil_freed_memory()
    host.diff_attention(q, k, v, 2 * base).sum().backward()
    assert not base.grad.any()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hk", [2, 0])
def test_no_heads(dt, hk):
    from thot_amd import _nott_host as host
    dt = DT[dt]
    q, k, v, lam = rnd(2, 3, 0, 16, dt=dt), rnd(2, 5, 2 * hk, 16, dt=dt), rnd(2, 5, hk, 32, dt=dt), torch.empty(0, device="cuda")
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
    assert o.shape == (2, 3, 0, 32) and lse.numel() == 0
    out = (torch.empty_like(q), torch.full_like(k, 7.0), torch.full_like(v, 7.0))
    _, dk, dv, dlam = ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse, out=out)
    assert not dk.any() and not dv.any() and dlam.numel() == 0
    k, v = k.requires_grad_(), v.requires_grad_()
    spoil_freed_memory()
    host.diff_attention(q, k, v, lam).sum().backward()
    assert not k.grad.any() and not v.grad.any()
