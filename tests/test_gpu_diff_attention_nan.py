"""Differential attention of rows that are NaN: NaN in the output and in the log-sum-exp, by
every kernel, and nowhere else."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
# few rows against many keys (keys split), many rows; b, t, s, h, hk, dh, dv
SHAPES = [(1, 1, 5000, 4, 2, 32, 64), (2, 3, 2000, 2, 2, 64, 128), (1, 40, 3000, 2, 1, 128, 256), (1, 300, 300, 2, 1, 32, 64),
          (1, 5, 900, 2, 1, 20, 41), (2, 16, 16, 2, 2, 16, 32)]


def rnd(*s, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(s, generator=g, device="cuda").to(dt)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_query(dt, shape, bad):
    dt = DT[dt]
    b, t, s, h, hk, dh, dv = shape
    if dt == torch.float32 and dh > 64:
        dh, dv = 64, 128
    q, k, v = rnd(b, t, 2 * h, dh, dt=dt, seed=1), rnd(b, s, 2 * hk, dh, dt=dt, seed=2), rnd(b, s, hk, dv, dt=dt, seed=3)
    lam = torch.rand(h, device="cuda") + 0.1
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
    for m in (0, 1):        # one map of one head's last row (an infinity times keys of both signs is NaN)
        q2 = q.clone()
        q2[0, t - 1, 2 + m] = bad
        p, lse2, p2 = ops.diff_attention_fwd(q2, k, v, lam, save=True)
        torch.cuda.synchronize()
        assert bool(p[0, t - 1, 1].isnan().all()) and bool(lse2[0, 2 + m, t - 1].isnan())
        assert bool(p2[0, t - 1, 1].isnan().all()) == (m == 1) and bool(lse2[0, 3 - m, t - 1].isfinite())
        for a, c in ((p, o), (p2, o2)):
            a = a.clone()
            a[0, t - 1, 1] = c[0, t - 1, 1]
            assert torch.equal(a, c)
        lse2[0, 2 + m, t - 1] = lse[0, 2 + m, t - 1]
        assert torch.equal(lse2, lse)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_key(dt, shape):
    """Every row of its key head sees it."""
    dt = DT[dt]
    b, t, s, h, hk, dh, dv = shape
    if dt == torch.float32 and dh > 64:
        dh, dv = 64, 128
    q, k, v = rnd(b, t, 2 * h, dh, dt=dt, seed=1), rnd(b, s, 2 * hk, dh, dt=dt, seed=2), rnd(b, s, hk, dv, dt=dt, seed=3)
    lam = torch.rand(h, device="cuda") + 0.1
    o, lse, _ = ops.diff_attention_fwd(q, k, v, lam)
    k[0, s // 2, 0] = math.nan
    p, lse2, _ = ops.diff_attention_fwd(q, k, v, lam)
    torch.cuda.synchronize()
    n = h // hk
    assert bool(p[0, :, :n].isnan().all()) and bool(lse2[0, 0:2 * n:2].isnan().all()) and bool(lse2[0, 1:2 * n:2].isfinite().all())
    assert torch.equal(p[0, :, n:], o[0, :, n:]) and torch.equal(p[1:], o[1:])
