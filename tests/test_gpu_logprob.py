"""token_logprob (log probabilities, entropy, top tokens and their gradient)
against the formulas in float64.

Tolerances count roundings (u = 2^-24).  With Z the largest |z| of a row's live
logits: the product with scale and the difference to the maximum put up to 3·Z·u
into every exponent; a sum of exponentials has chains of at most c/256 + 32
additions.  So a log probability is off by at most (6·Z + c/256 + 64)·u, the
entropy by that times 1 + Σ p·|z − m|.  p in the gradient carries the error of
z − lse: (8·Z + 32)·u of each term."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (3, 2), (5, 7), (4, 64), (7, 100), (3, 255), (2, 1000), (5, 1024), (33, 515), (3, 8191), (2, 32000),
          (1, 50257), (2, 128256), (1, 300001)]


def make(n, c, dt, seed=0, kind="normal"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn((n, c), generator=g, device="cuda") * 3
    y = torch.randint(0, c, (n,), generator=g, device="cuda")
    if kind == "ties":
        z = (z / 3).round()
    elif kind == "equal":
        z = torch.full_like(z, -1.5)
    elif kind == "masked":      # −inf and the type's lowest value, and rows with nothing else
        z[:, ::3] = -math.inf
        z[:, 1::7] = torch.finfo(dt).min
        z[0] = -math.inf
        z[-1] = torch.finfo(dt).min
    elif kind == "rising":      # every element a new maximum
        z = torch.arange(c, device="cuda").float().expand(n, c) * (20.0 / c)
    elif kind == "large":
        z = z * 1000
    z = z.to(dt).contiguous()
    if n > 1:
        y[n // 2] = -100
    return z, y


def live_size(z, scale):
    """Z: the largest |scale·logit| that exponentials see (masked ones aside)."""
    w = torch.where(z.double() > -1e30, z.double().abs(), 0.0) * scale
    return w.amax(1) + 1


def reference(z, y, scale):
    zd = z.double() * scale
    zd = torch.where(zd < -1e30, -math.inf, zd)
    m = zd.amax(1, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    e = (zd - m).exp()
    s = e.sum(1, keepdim=True)
    lp = torch.where(s > 0, zd - m - s.log(), -math.inf)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    spread = torch.where(p > 0, p * (zd - m).abs(), 0.0).sum(1)
    lse = (m + s.log())[:, 0]
    hit = torch.where(y >= 0, lp.gather(1, y.clamp_min(0)[:, None])[:, 0], 0.0)
    return lp, p, ent, spread, lse, hit


def close(got, want, tol, what):
    got = got.double()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    err = (got - want).abs()[~inf]
    tol = tol.expand_as(want)[~inf] + U * want[~inf].abs()
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"


def order(z, k):
    """The k largest of each row, ties lowest column first."""
    return z.float().double().sort(dim=1, descending=True, stable=True).indices[:, :k]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("kind", ["normal", "ties", "equal", "masked", "rising", "large"])
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward(n, c, kind, dt):
    dt = DT[dt]
    z, y = make(n, c, dt, kind=kind)
    scale, top = (0.8, min(c, 5)) if kind != "ties" else (1.0, min(c, 64))
    lp, ent, lse, tv, ti = ops.token_logprob_fwd(z, y, scale=scale, top=top)
    torch.cuda.synchronize()
    rlp, _, rent, spread, rlse, hit = reference(z, y, float(torch.tensor(scale, dtype=torch.float32)))
    tol = (6 * live_size(z, scale) + c / 256 + 64) * U
    close(lp, hit, tol, "logprob")
    close(lse, rlse, tol, "lse")
    close(ent, rent, tol * (1 + spread), "entropy")
    want = order(z, top)
    assert torch.equal(ti, want)
    close(tv, rlp.gather(1, want), tol[:, None], "top_logprob")
    # without top tokens: the same statistics
    again = ops.token_logprob_fwd(z, y, scale=scale)
    assert again[3] is None and all(torch.equal(a, b) for a, b in zip(again[:3], (lp, ent, lse)))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("kind", ["normal", "masked", "equal"])
@pytest.mark.parametrize("n,c", SHAPES)
def test_backward(n, c, kind, dt):
    dt = DT[dt]
    z, y = make(n, c, dt, kind=kind)
    scale = 1.3
    _, ent, lse, _, _ = ops.token_logprob_fwd(z, y, scale=scale)
    g = torch.Generator(device="cuda").manual_seed(5)
    dlp, dent = (torch.randn(n, generator=g, device="cuda") for _ in range(2))
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    lp, p, rent, _, _, _ = reference(z, y, s32)
    lp0 = torch.where(p > 0, lp, 0.0)
    dl = torch.where(y >= 0, dlp.double(), 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, y.clamp_min(0)[:, None], (y >= 0).double()[:, None])
    for de in (None, dent):
        got = ops.token_logprob_bwd(z, y, lse, dlp, entropy=ent if de is not None else None, dentropy=de, scale=scale)
        h = 0.0 if de is None else de.double()[:, None]
        want = s32 * (dl * (hot - p) - h * p * (lp0 + rent[:, None]))
        none = torch.isinf(rent * 0 + lp.amax(1))       # rows with nothing live
        want[none] = 0
        mag = s32 * (dl.abs() * (hot + p) + abs(h) * p * (lp0.abs() + rent[:, None] + 1))
        tol = torch.finfo(dt).eps / 2 * want.abs() + (8 * live_size(z, scale)[:, None] + 32) * U * mag + 1e-37
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
        # into the logits themselves
        z2 = z.clone()
        ops.token_logprob_bwd(z2, y, lse, dlp, entropy=ent, dentropy=de, scale=scale, out=z2)
        assert torch.equal(z2, got)


def test_gradient_matches_differences():
    z, y = make(6, 37, torch.float32, seed=3)
    _, ent, lse, _, _ = ops.token_logprob_fwd(z, y, scale=0.7)
    dlp, dent = torch.randn(6, device="cuda"), torch.randn(6, device="cuda")
    got = ops.token_logprob_bwd(z, y, lse, dlp, entropy=ent, dentropy=dent, scale=0.7).double()
    s32 = float(torch.tensor(0.7, dtype=torch.float32))

    def f(zz):
        _, _, e, _, _, hit = reference(zz, y, s32)
        return (hit * dlp.double() + e * dent.double()).sum()
    v, h = torch.randn_like(z).double(), 1e-5
    diff = (f(z.double() + h * v) - f(z.double() - h * v)) / (2 * h)
    assert abs(float((got * v).sum() - diff)) <= 1e-5 * float((got * v).abs().sum())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("c", [9, 1000, 40000, 128256])
def test_nan_and_infinity(dt, c):
    """A NaN makes its row NaN and is the largest token; +inf makes it NaN; other rows keep theirs."""
    z, y = make(4, c, DT[dt])
    y[:] = 1
    clean = ops.token_logprob_fwd(z, y, top=3)
    z2 = z.clone()
    z2[1, c - 2] = math.nan
    z2[2, 3] = math.inf
    lp, ent, lse, tv, ti = ops.token_logprob_fwd(z2, y, top=3)
    for a in (lp, ent, lse):
        assert bool(torch.isnan(a[1:3]).all())
    assert bool(torch.isnan(tv[1:3]).all())
    assert int(ti[1, 0]) == c - 2 and int(ti[2, 0]) == 3
    for a, b in zip((lp, ent, lse, tv, ti), clean):
        assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3])
    d = ops.token_logprob_bwd(z2, y, lse, torch.ones(4, device="cuda"))
    assert bool(torch.isnan(d[1]).all()) and bool(torch.isfinite(d[0]).all())


def test_labels_out_of_range_are_counted():
    ctx = ops.context()
    ctx.device_errors()
    z, y = make(5, 50, torch.float32)
    y[:] = torch.tensor([50, -1, -100, 0, 49], device="cuda")
    lp, _, lse, _, _ = ops.token_logprob_fwd(z, y)
    assert ctx.device_errors() == 2
    assert bool((lp[:3] == 0).all()) and bool((lp[3:] != 0).all())
    d = ops.token_logprob_bwd(z, y, lse, torch.ones(5, device="cuda"))
    assert torch.count_nonzero(d[:3]).item() == 0 and torch.count_nonzero(d[3:]).item() == 100


def test_empty_and_unaligned():
    e = torch.empty((0, 12), device="cuda", dtype=torch.bfloat16)
    y = torch.empty((0,), device="cuda", dtype=torch.int64)
    lp, ent, lse, tv, ti = ops.token_logprob_fwd(e, y, top=2)
    assert lp.shape == (0,) and ti.shape == (0, 2)
    assert ops.token_logprob_bwd(e, y, lse, lp).shape == (0, 12)
    for c in (1024, 32000):     # a whole number of groups, from an address that is none
        buf = torch.randn(3 * c + 1, device="cuda").bfloat16()
        z = buf[1:].view(3, c)
        y = torch.tensor([0, c - 1, 5], device="cuda")
        a, b = (ops.token_logprob_fwd(t, y, top=4) for t in (z, z.clone()))
        assert torch.equal(a[4], b[4])
        rl = reference(z, y, 1.0)
        tol = (6 * live_size(z, 1.0) + c / 256 + 64) * U
        close(a[0], rl[5], tol, "logprob")
        close(b[0], rl[5], tol, "logprob")


def test_captured_and_other_stream():
    z, y = make(16, 4096, torch.bfloat16)
    long, ly = make(2, 150000, torch.bfloat16)
    d = torch.randn(16, device="cuda")

    def step():
        f = ops.token_logprob_fwd(z, y, top=7)
        return (*f, *ops.token_logprob_fwd(long, ly, top=7), ops.token_logprob_bwd(z, y, f[2], d, entropy=f[1], dentropy=d))
    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        z.copy_(torch.randn_like(z))
        long.copy_(torch.randn_like(long))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n,c", [(3, 700), (2, 5000), (600, 3000), (2, 100000)])
def test_nan_in_the_first_column_leads(n, c, dt):
    """NaN counts as largest wherever it stands, among so many equal logits that the row is scanned for each."""
    z = torch.zeros((n, c), device="cuda", dtype=DT[dt])
    z[:, 0] = z[:, c // 2] = math.nan
    z[:, 5] = 1.0
    top = ops.token_logprob_fwd(z, torch.zeros(n, device="cuda", dtype=torch.int64), top=5)[4]
    torch.cuda.synchronize()
    want = torch.tensor([0, c // 2, 5, 1, 2], device="cuda").expand(n, 5)
    assert torch.equal(top, want)
