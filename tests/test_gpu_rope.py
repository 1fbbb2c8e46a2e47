"""qk_norm_rope (per-head norm, weight and rotation of queries and keys) against
its formula in float64.

Tolerances count roundings.  With u the half step of fp32 (2^-24), a rotated value
za·c − zb·s carries, relative to |za| + |zb|: the row's sum of squares (half of
dh/64 + 8 additions), rsqrt (2), three products, the angle's rounding to fp32
(2π·2^-25, about 4u), sin and cos (2), and the two fused steps: under 24u; then
the half step of the output's type.  The input's gradient adds the mean of
products: 48u of its own magnitudes.  A weight's gradient is a sum in chains of
fewer than 128 additions."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def half_step(dt):
    return torch.finfo(dt).eps / 2


def axis_of_pair(sections):
    return torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda", dtype=torch.long)


def rotate(x, cos, sin, rot, inter):
    """x [b, t, h, dh] turned by angles given as cos, sin [b, t, 1, rot/2]."""
    y = x.clone()
    if rot == 0:
        return y
    ia = torch.arange(0, rot, 2, device="cuda") if inter else torch.arange(rot // 2, device="cuda")
    ib = ia + 1 if inter else ia + rot // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    return y


def reference(x, gamma, pos, freq, sections, inter, norm, dy=None):
    """(y, |za| + |zb|) or, with dy, (dx, its magnitudes, dgamma, its magnitudes), float64."""
    x = x.double()
    rot = 0 if freq is None else 2 * freq.numel()
    cos = sin = None
    if rot:
        ang = (pos.double()[axis_of_pair(sections)].movedim(0, -1) * freq)[:, :, None]
        cos, sin = ang.cos(), ang.sin()
    g = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt() if norm else torch.ones_like(x[..., :1])
    xh = x * r

    def both(v):   # |a| + |b| of the pair, |v| past the rotated elements
        one = None if cos is None else torch.ones_like(cos)
        return v.abs() if rot == 0 else torch.maximum(rotate(v.abs(), one, one, rot, inter).abs(),
                                                      rotate(v.abs(), one, -one, rot, inter).abs())
    if dy is None:
        return rotate(xh * g, cos, sin, rot, inter), both(xh * g)
    dy = dy.double()
    dz = rotate(dy, cos, -sin if rot else None, rot, inter)
    mag = both(dy)
    if not norm:
        return dz, mag, None, None
    dx = r * (g * dz - xh * (g * dz * xh).mean(-1, keepdim=True))
    dmag = r * (g.abs() * mag + xh.abs() * (g * mag * xh).abs().mean(-1, keepdim=True))
    return dx, dmag, (dz * xh).sum((0, 1, 2)), (mag * xh.abs()).sum((0, 1, 2))


def inputs(b, t, hq, hk, dh, dt, seed=0, layout="packed"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda").to(dt)
    if layout == "packed":
        qkv = rnd(b, t, (hq + 2 * hk) * dh)
        q, k = (qkv[..., o * dh:(o + n) * dh].unflatten(-1, (n, dh)) for o, n in ((0, hq), (hq, hk)))
    elif layout == "head_major":
        q, k = (rnd(b, h, t, dh).transpose(1, 2) for h in (hq, hk))
    elif layout == "odd_start":     # a byte address that no vector load may use
        q, k = (rnd(b * t * h * dh + 1)[1:].view(b, t, h, dh) for h in (hq, hk))
    else:
        q, k = rnd(b, t, hq, dh), rnd(b, t, hk, dh)
    return q, k, rnd(b, t, hq, dh), rnd(b, t, hk, dh), 1 + 0.2 * rnd(dh), 1 + 0.2 * rnd(dh)


def positions(b, t, axes, far=0):
    tok = torch.arange(t, device="cuda")
    p = [far + tok[None] * (a + 1) // (3 * a + 1) + torch.arange(b, device="cuda")[:, None] * 7 for a in range(axes)]
    return torch.stack([x.expand(b, t) for x in p]).contiguous()


# b, t, hq, hk, dh, rot, axes, interleaved, norm, layout, far
CASES = [
    (1, 1, 1, 1, 64, 64, 1, False, True, "dense", 0),
    (2, 37, 4, 2, 64, 64, 1, False, True, "packed", 100000),
    (2, 37, 4, 2, 64, 64, 1, True, True, "packed", 100000),
    (3, 65, 3, 1, 128, 128, 1, False, True, "packed", 0),
    (1, 300, 16, 16, 64, 32, 1, False, True, "head_major", 0),
    (2, 50, 5, 5, 80, 60, 3, True, True, "packed", 30),
    (2, 50, 5, 5, 80, 48, 3, False, True, "packed", 30),
    (2, 50, 5, 5, 96, 96, 2, False, False, "packed", 5000),
    (1, 33, 2, 1, 256, 256, 1, False, True, "dense", 0),
    (1, 33, 2, 1, 512, 128, 4, False, True, "dense", 9),
    (1, 70, 3, 2, 33, 32, 1, False, True, "dense", 0),
    (1, 70, 3, 2, 33, 14, 1, True, True, "packed", 0),
    (2, 19, 3, 2, 64, 64, 1, False, True, "odd_start", 0),
    (2, 19, 3, 2, 72, 0, 1, False, True, "packed", 0),
    (1, 5, 1, 1, 1, 0, 1, False, True, "dense", 0),
    (1, 9, 2, 1, 2, 2, 1, False, True, "dense", 2 ** 40),
    (1, 40, 2, 2, 160, 40, 1, False, True, "packed", 0),
    (2, 21, 7, 3, 40, 40, 1, False, False, "packed", 77),
    (8, 260, 2, 1, 64, 64, 1, False, True, "packed", 0),
]


def call_args(case, dt):
    b, t, hq, hk, dh, rot, axes, inter, norm, layout, far = case
    q, k, dyq, dyk, gq, gk = inputs(b, t, hq, hk, dh, dt, layout=layout)
    if not norm:
        gq = gk = None
    pos, freq, sections = None, None, None
    if rot:
        pos, freq = positions(b, t, axes, far), ops.rope_frequencies(rot)
        n = rot // 2 // axes
        sections = [rot // 2 - n * (axes - 1)] + [n] * (axes - 1)
    return q, k, dyq, dyk, gq, gk, pos, freq, dict(norm=norm, eps=EPS, sections=sections, interleaved=inter)


def near(got, want, mag, dt, roundings, what):
    tol = half_step(dt) * want.abs() + roundings * U * mag + 1e-30
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("case", CASES)
def test_forward(case, dt):
    dt = DT[dt]
    q, k, _, _, gq, gk, pos, freq, kw = call_args(case, dt)
    before = (q.clone(), k.clone())
    yq, yk = ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk, **kw)
    torch.cuda.synchronize()
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    for x, y, g, what in ((q, yq, gq, "yq"), (k, yk, gk, "yk")):
        want, mag = reference(x, g, pos, freq, kw["sections"], kw["interleaved"], kw["norm"])
        near(y, want, mag, dt, 24, what)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("case", CASES)
def test_backward(case, dt):
    dt = DT[dt]
    q, k, dyq, dyk, gq, gk, pos, freq, kw = call_args(case, dt)
    dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk, **kw)
    torch.cuda.synchronize()
    for x, dy, dx, g, dg, what in ((q, dyq, dq, gq, dgq, "q"), (k, dyk, dk, gk, dgk, "k")):
        want, mag, wg, mg = reference(x, g, pos, freq, kw["sections"], kw["interleaved"], kw["norm"], dy)
        near(dx, want, mag, dt, 48, "d" + what)
        assert (dg is None) == (g is None)
        if g is not None:
            near(dg, wg, mg, torch.float32, 128 + 48, "dgamma_" + what)


def test_gradient_matches_differences():
    """<grad, v> against central differences of the forward formula in float64."""
    case = (2, 11, 3, 2, 24, 16, 2, False, True, "dense", 5)
    q, k, dyq, dyk, gq, gk, pos, freq, kw = call_args(case, torch.float32)
    dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk, **kw)
    for x, dy, g, dx, dg in ((q, dyq, gq, dq, dgq), (k, dyk, gk, dk, dgk)):
        def f(x_, g_):
            return (reference(x_, g_, pos, freq, kw["sections"], False, True)[0] * dy.double()).sum()
        x, g = x.double(), g.double()
        v, w, h = torch.randn_like(x), torch.randn_like(g), 1e-5
        # central differences of a smooth function: h²·f'''/6 and 2^-53/h leave about 1e-9
        for got, diff in ((dx, (f(x + h * v, g) - f(x - h * v, g)) / (2 * h)),
                          (dg, (f(x, g + h * w) - f(x, g - h * w)) / (2 * h))):
            dot = (got.double() * (v if got is dx else w)).sum()
            size = (got.double() * (v if got is dx else w)).abs().sum()
            assert abs(float(dot - diff)) <= 1e-5 * float(size)


@pytest.mark.parametrize("dt", DT)
def test_in_place_and_packed_gradients(dt):
    """Outputs that are the inputs, and gradients written into a packed buffer."""
    dt = DT[dt]
    b, t, hq, hk, dh = 2, 45, 4, 2, 64
    q, k, dyq, dyk, gq, gk = inputs(b, t, hq, hk, dh, dt)
    pos, freq = positions(b, t, 1), ops.rope_frequencies(dh)
    want = ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk)
    grads = ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk)
    packed = torch.full((b, t, (hq + 2 * hk) * dh), 7.0, device="cuda", dtype=dt)
    out = [packed[..., o * dh:(o + n) * dh].unflatten(-1, (n, dh)) for o, n in ((0, hq), (hq, hk))]
    got = ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk, out=out)
    assert torch.equal(out[0], grads[0]) and torch.equal(out[1], grads[1])
    assert torch.equal(got[2], grads[2]) and torch.equal(got[3], grads[3])
    assert bool((packed[..., (hq + hk) * dh:] == 7).all())     # v's gradient is not touched
    ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk, out=(dyq, dyk))
    assert torch.equal(dyq, grads[0]) and torch.equal(dyk, grads[1])
    ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_head_major_outputs_feed_attention():
    b, t, h, dh = 2, 40, 3, 32
    q, k, _, _, gq, gk = inputs(b, t, h, h, dh, torch.bfloat16)
    pos, freq = positions(b, t, 1), ops.rope_frequencies(dh)
    want = ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk)
    out = [torch.empty((b, h, t, dh), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk, out=[o.transpose(1, 2) for o in out])
    for o, w in zip(out, want):
        assert torch.equal(o.transpose(1, 2), w)


def test_accumulate_queries_alone_and_empty():
    b, t, hq, dh = 2, 9, 3, 64
    q, _, dyq, _, gq, gk = inputs(b, t, hq, 1, dh, torch.float32)
    pos, freq = positions(b, t, 1), ops.rope_frequencies(dh)
    yq, yk = ops.qk_norm_rope_fwd(q, None, pos, freq, gq)
    assert yk is None and torch.equal(yq, ops.qk_norm_rope_fwd(q, q, pos, freq, gq, gq)[1])
    dq, dk, dg, _ = ops.qk_norm_rope_bwd(dyq, None, q, None, pos, freq, gq)
    assert dk is None
    acc = torch.full((dh,), 3.0, device="cuda")
    ops.qk_norm_rope_bwd(dyq, None, q, None, pos, freq, gq, dgamma_q=acc, accumulate=True)
    assert torch.allclose(acc, dg + 3, rtol=2 * U, atol=0)
    e = torch.empty((0, 4, 2, dh), device="cuda")
    none = torch.empty((1, 0, 4), device="cuda", dtype=torch.int64)
    acc.fill_(3.0)
    assert ops.qk_norm_rope_fwd(e, e, none, freq, gq, gk)[0].shape == e.shape
    ops.qk_norm_rope_bwd(e, e, e, e, none, freq, gq, gk, dgamma_q=acc, dgamma_k=acc.clone(), accumulate=True)
    assert bool((acc == 3).all())
    with pytest.raises(ValueError, match="accumulate needs"):
        ops.qk_norm_rope_bwd(e, e, e, e, none, freq, gq, gk, dgamma_q=acc, accumulate=True)
    ops.qk_norm_rope_bwd(e, e, e, e, none, freq, gq, gk, dgamma_q=acc)
    assert bool((acc == 0).all())


def test_zero_head_and_nan_stay_in_their_head():
    """A head of zeros has 1/sqrt(eps) and a zero result; NaN and infinity reach no other head."""
    b, t, h, dh = 1, 6, 4, 64
    q, k, dyq, dyk, gq, gk = inputs(b, t, h, h, dh, torch.float32, layout="dense")
    pos, freq = positions(b, t, 1), ops.rope_frequencies(dh)
    clean = ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk)[0]
    q2 = q.clone()
    q2[0, 1, 2] = 0
    q2[0, 3, 1, 5] = math.nan
    q2[0, 4, 0, 7] = math.inf
    y = ops.qk_norm_rope_fwd(q2, k, pos, freq, gq, gk)[0]
    dq = ops.qk_norm_rope_bwd(dyq, dyk, q2, k, pos, freq, gq, gk)[0]
    assert bool((y[0, 1, 2] == 0).all()) and bool(torch.isfinite(dq[0, 1, 2]).all())
    assert bool(torch.isnan(y[0, 3, 1]).all())
    keep = torch.ones((b, t, h), dtype=torch.bool, device="cuda")
    keep[0, 1, 2] = keep[0, 3, 1] = keep[0, 4, 0] = False
    assert torch.equal(y[keep], clean[keep])


def test_captured_and_other_stream():
    b, t, hq, hk, dh = 2, 64, 4, 2, 128
    q, k, dyq, dyk, gq, gk = inputs(b, t, hq, hk, dh, torch.bfloat16)
    pos, freq = positions(b, t, 1), ops.rope_frequencies(dh)

    def step():
        return (*ops.qk_norm_rope_fwd(q, k, pos, freq, gq, gk), *ops.qk_norm_rope_bwd(dyq, dyk, q, k, pos, freq, gq, gk))
    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    for a, w in zip(other, want):
        assert torch.equal(a, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, step()):
            assert torch.equal(a, w), i
