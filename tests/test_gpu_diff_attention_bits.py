"""Differential attention of maps that resemble each other, which is what it is for: o_1 and
λ·o_2 nearly cancel, so what each map's rounding leaves is large beside their difference.
In bf16 the probabilities and dz enter their products with the remainder of their
rounding, by every kernel, whatever the alignment.

Tolerances, per element: a bf16 value and its remainder's bf16 value are off by 2^-8·2^-8 at
most; scores and sums as in the tests against float64 (e = 2^-24, (dh + 4)·e of the largest
score's magnitudes, 64·e for exponential and joins, n·e for sums of n terms), outputs by half
a step."""
import math

import pytest
import torch

from test_gpu_diff_attention import E, Ref, close, seen
from thot_amd import ops

pytestmark = pytest.mark.gpu

TWICE = 2.0 ** -16


def resembling(b, t, s, h, hk, dh, dv, seed, odd):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def maps(rows, heads, std):
        x = n(b, rows, heads, 1, dh) * std
        return (x + 0.03 * std * n(b, rows, heads, 2, dh)).flatten(2, 3)
    q, k, v = maps(t, h, 1.5), maps(s, hk, 1.0), n(b, s, hk, dv)
    if odd:     # rows that begin at odd addresses
        q, k, v = (torch.cat((x, x[..., :1]), -1).bfloat16()[..., :-1] for x in (q, k, v))
    else:
        q, k, v = (x.bfloat16() for x in (q, k, v))
    return q, k, v, torch.rand(h, generator=g, device="cuda") * 0.1 + 0.9


# every width of the wide kernels, keys split, whole; rows that are not aligned
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("b,t,s,h,hk,dh,dv,causal", [
    (1, 130, 130, 2, 2, 32, 64, True), (2, 200, 200, 4, 2, 64, 128, True), (1, 150, 150, 2, 1, 96, 192, True),
    (1, 140, 140, 4, 1, 128, 256, True), (1, 100, 300, 2, 2, 40, 72, False), (2, 1, 3000, 4, 2, 64, 128, False),
    (1, 9, 2000, 4, 1, 128, 256, False), (1, 700, 700, 1, 1, 96, 96, True)])
def test_maps_that_resemble_each_other(b, t, s, h, hk, dh, dv, causal, odd):
    q, k, v, lam = resembling(b, t, s, h, hk, dh, dv, t + dh, odd)
    scale, group = dh ** -0.5, h // hk
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, causal=causal, save=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    do = torch.randn((b, t, h, dv), generator=g, device="cuda").bfloat16()
    dq, dk, dvv, _ = ops.diff_attention_bwd(do, q, k, v, lam, o, o2, lse, causal=causal)
    torch.cuda.synchronize()
    r = Ref(q, k, v, lam, seen(b, t, s, causal, None, None), scale)
    w = 2 * r.s + TWICE + (s + 8) * E
    tol1, tol2 = ((w * r.p) @ r.v.abs()[:, :, None]).unbind(2)
    close(o2.transpose(1, 2), r.o2, tol2, "o2")
    close(o.transpose(1, 2), r.o, tol1 + r.lam.abs() * tol2, "o")
    # (the case is what it says it is)
    assert float(r.o.norm() / r.o1.norm()) < 0.3

    d, oo, oo2 = (x.double().transpose(1, 2) for x in (do, o, o2))
    D2, D2m = (d * oo2).sum(3, keepdim=True), (d * oo2).abs().sum(3, keepdim=True)
    D1, D1m = (d * oo).sum(3, keepdim=True) + r.lam * D2, (d * oo).abs().sum(3, keepdim=True) + r.lam * D2m
    dp, dpm = d @ r.v.transpose(2, 3), d.abs() @ r.v.abs().transpose(2, 3)
    p1, p2 = r.p.unbind(2)
    w1, w2 = (2 * r.s + TWICE + 4 * E * r.lse.abs().unflatten(1, (h, 2))[..., None]).unbind(2)
    sums, many = (dv + 8) * E, (max(s, t * group) + 8) * E
    dz = torch.stack((p1 * (dp - D1), -r.lam * p2 * (dp - D2)), 2)
    dzt = torch.stack((p1 * (w1 * (dp - D1).abs() + sums * (dpm + D1m)), r.lam * p2 * (w2 * (dp - D2).abs() + sums * (dpm + D2m))), 2)
    dzt = dzt + many * dz.abs()

    def heads(x):
        return x.unflatten(1, (hk, group)).sum(2)
    close(dq.view(b, t, h, 2, dh).permute(0, 2, 3, 1, 4), dz @ r.k * scale, dzt @ r.k.abs() * scale, "dq")
    close(dk.view(b, s, hk, 2, dh).permute(0, 2, 3, 1, 4), heads(dz.transpose(3, 4) @ r.q) * scale,
          heads(dzt.transpose(3, 4) @ r.q.abs()) * scale, "dk")
    pt = (w1 + many) * p1 + (w2 + many) * r.lam * p2
    close(dvv.permute(0, 2, 1, 3), heads((p1 - r.lam * p2).transpose(2, 3) @ d), heads(pt.transpose(2, 3) @ d.abs()), "dv")
    assert not math.isnan(float(dq.float().sum()))
