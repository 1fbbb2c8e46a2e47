"""gated_linear (both projections, activation, product; backward) against its
formula in float64.

Tolerances count roundings (u = 2^-24, h the half step of the type).  A dot
product of length k is summed in chains of at most k/4 + 16 additions.  The
activation and its derivative carry (16 + 2·g²)·u of their terms (the exponent or
the error function's argument, a few steps of each function).  bf16: dx sees
[dg|du] rounded once (h of each term); dw sees it in two pieces (h² of each)."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def act64(name, g):
    """The activation and its derivative by autograd, float64."""
    F = torch.nn.functional
    g = g.detach().requires_grad_()
    a = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "relu": F.relu,
         "sigmoid": torch.sigmoid}[name](g)
    return a.detach(), torch.autograd.grad(a.sum(), g)[0]


def make(m, d, f, dt, bias, seed=0, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, std=1.0):
        n = 1
        for v in s:
            n *= v
        return (torch.randn(n + shift, generator=g, device="cuda") * std).to(dt)[shift:].view(s)
    return (rnd(m, d), rnd(2 * f, d, std=d ** -0.5), (torch.randn(2 * f, generator=g, device="cuda") if bias else None),
            rnd(m, f, std=0.1))


def near(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), f"{what}: {float((err / (tol + 1e-30)).max())} of the tolerance"


def norm_error(got, want):
    n = want.norm()
    return float((got.double() - want).norm() / n) if n > 0 else 0.0


# m, d, f, bias: single tokens, widths inside and across tiles, odd ones
SHAPES = [(1, 1, 1, True), (1, 64, 40, False), (1, 1024, 512, False), (2, 512, 1000, True), (5, 100, 33, True),
          (8, 1024, 1408, False), (16, 256, 64, True), (17, 264, 72, False), (31, 96, 300, True), (33, 128, 130, False),
          (64, 320, 128, True), (70, 77, 61, True), (128, 128, 128, False), (129, 136, 264, True), (200, 1000, 136, False),
          (256, 64, 512, True), (300, 520, 200, False), (515, 256, 1001, True), (1030, 192, 96, False)]


def forward_reference(x, w, b, act):
    xd, wd = x.double(), w.double()
    gu = xd @ wd.t() + (0 if b is None else b.double())
    mag = xd.abs() @ wd.abs().t() + (0 if b is None else b.double().abs())
    f = w.shape[0] // 2
    a, da = act64(act, gu[:, :f])
    err = (x.shape[1] / 4 + 16) * U * mag        # of the pre-activations
    return gu, err, a, da


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
def test_forward(i, shape, dt):
    m, d, f, bias = shape
    dt = DT[dt]
    act = ACTS[i % 5]
    x, w, b, _ = make(m, d, f, dt, bias)
    gu, err, a, da = forward_reference(x, w, b, act)
    g, u = gu[:, :f], gu[:, f:]
    half = torch.finfo(dt).eps / 2
    for save in (False, True):
        h, got = ops.gated_linear_fwd(x, w, b, act=act, save=save)
        torch.cuda.synchronize()
        # |act'| <= 1.13, and act'' <= 1 covers the second order
        tol = half * (a * u).abs() + (1.13 + err[:, :f]) * err[:, :f] * u.abs() + a.abs() * err[:, f:] + \
            1.13 * err[:, :f] * err[:, f:] + (16 + 2 * g * g) * U * ((a * u).abs() + 1e-6 * u.abs())
        near(h, a * u, tol * 1.01, "h")
        assert (got is None) == (not save)
        if save:
            near(got, gu, (half * gu.abs() + err) * 1.01, "gu")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
def test_backward(i, shape, dt):
    m, d, f, bias = shape
    dt = DT[dt]
    act = ACTS[(i + 2) % 5]
    x, w, b, dh = make(m, d, f, dt, bias, seed=i)
    gu = forward_reference(x, w, b, act)[0].to(dt)
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, gu, act=act)
    torch.cuda.synchronize()
    g, u = gu.double().chunk(2, -1)
    a, da = act64(act, g)
    v = torch.cat((dh.double() * u * da, dh.double() * a), 1)
    xd, wd = x.double(), w.double()
    step = torch.finfo(dt).eps / 2
    rel = (16 + 2 * g * g) * U
    ev = torch.cat((rel * (dh.double() * u).abs() * (da.abs() + 0.3), rel * (dh.double() * (a.abs() + 1e-6)).abs()), 1)
    once = ev + (step * v.abs() if dt == torch.bfloat16 else 0)
    twice = ev + (step * step * v.abs() if dt == torch.bfloat16 else 0)
    want = v @ wd
    near(dx, want, step * want.abs() + once @ wd.abs() + (2 * f / 4 + 16) * U * (v.abs() @ wd.abs()), "dx")
    # roundings that fall either way: the 2-norm is no further off than one half step
    assert norm_error(dx, want) <= (step if dt == torch.bfloat16 else 64 * U)
    want = v.t() @ xd
    near(dw, want, twice.t() @ xd.abs() + (m / 4 + 32) * U * (v.abs().t() @ xd.abs()), "dw")
    assert norm_error(dw, want) <= 2.0 ** -16
    near(db, v.sum(0), ev.sum(0) + (m / 64 + 96) * U * v.abs().sum(0), "db")
    # accumulation, and each gradient by itself
    dw2, db2 = torch.full_like(dw, 2.0), torch.full_like(db, -1.0)
    ops.gated_linear_bwd(dh, x, w, gu, act=act, dw=dw2, db=db2, need_dx=False, accumulate=True)
    # each of the two pieces' products is added to what is there: two roundings of the sum
    near(dw2, dw.double() + 2, 3 * U * (dw.double().abs() + 2), "dw accumulated")
    near(db2, db.double() - 1, 2 * U * (db.double().abs() + 1), "db accumulated")
    assert torch.equal(ops.gated_linear_bwd(dh, x, w, gu, act=act, need_dw=False, need_db=False)[0], dx)


@pytest.mark.parametrize("act", ACTS)
def test_activation_range(act):
    """Pre-activations from −100 to 100, zeros and NaN, through an identity gate projection."""
    n = 403
    x = torch.cat((torch.linspace(-100, 100, n - 3, device="cuda"), torch.tensor([0.0, -0.0, 1e-20], device="cuda")))
    x = x[:, None]
    w = torch.tensor([[1.0], [0.5]], device="cuda")
    h, gu = ops.gated_linear_fwd(x, w, act=act, save=True)
    a, da = act64(act, x.double())
    u = 0.5 * x.double()
    tail = (16 + 2 * x.double().square()) * U
    # past −40 a sigmoid is taken at e^-80: nothing to a value of any size
    near(h, a * u, 2 * U * (a * u).abs() + tail * (a * u).abs() + 1e-14, "h")
    one = torch.ones_like(x)
    dx, dw, db = ops.gated_linear_bwd(one, x, w, gu, act=act, need_dw=False, need_db=False)
    want = (u * da + 0.5 * a)
    near(dx, want, tail * (u * da).abs() + tail * a.abs() + 8 * U * (want.abs() + u.abs() + a.abs()) + 1e-12, "dx")
    x[5] = float("nan")
    h, _ = ops.gated_linear_fwd(x, w, act=act)
    assert bool(torch.isnan(h[5]).all()) and bool(torch.isfinite(h[:5]).all()) and bool(torch.isfinite(h[6:]).all())


@pytest.mark.parametrize("dt", DT)
def test_gradient_matches_differences(dt):
    m, d, f = 9, 12, 7
    x, w, b, dh = make(m, d, f, torch.float32, True)
    gu = ops.gated_linear_fwd(x, w, b, save=True)[1]
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, gu)

    def fn(x, w, b):
        gu = x @ w.t() + b
        return (act64("silu", gu[:, :f])[0] * gu[:, f:] * dh.double()).sum()
    at = [t.double() for t in (x, w, b)]
    for i, grad in enumerate((dx, dw, db)):
        v, h = torch.randn_like(at[i]), 1e-5
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - h * v, at[i] + h * v
        diff = (fn(*hi) - fn(*lo)) / (2 * h)
        assert abs(float((grad.double() * v).sum() - diff)) <= 2e-5 * float((grad.double() * v).abs().sum())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,d,f", [(4, 64, 32), (150, 128, 160)])
def test_unaligned_and_leading_dimensions(m, d, f, dt):
    """Tensors that start off a 16-byte address, and x of three dimensions."""
    dt = DT[dt]
    a = make(m, d, f, dt, True)
    x, w, b, dh = make(m, d, f, dt, True, shift=1)
    assert x.data_ptr() % 16
    gu, err, act, _ = forward_reference(x, w, b, "silu")
    h, got = ops.gated_linear_fwd(x.view(2, m // 2, d), w, b, save=True)
    assert h.shape == (2, m // 2, f) and got.shape == (2, m // 2, 2 * f)
    assert norm_error(h.reshape(m, f), act * gu[:, f:]) <= torch.finfo(dt).eps / 2 + 64 * U
    dx, dw, db = ops.gated_linear_bwd(dh.view(h.shape), x.view(2, m // 2, d), w, got)
    dx2, dw2, db2 = ops.gated_linear_bwd(dh.clone(), x.clone(), w.clone(), got.reshape(m, 2 * f).clone())
    assert norm_error(dx.reshape(m, d), dx2.double()) <= 2 * torch.finfo(dt).eps
    assert norm_error(dw, dw2.double()) <= 2.0 ** -16 and torch.allclose(db, db2, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dt", DT)
def test_empty(dt):
    dt = DT[dt]
    x, w = torch.empty((0, 16), device="cuda", dtype=dt), torch.ones((10, 16), device="cuda", dtype=dt)
    h, gu = ops.gated_linear_fwd(x, w, save=True)
    assert h.shape == (0, 5) and gu.shape == (0, 10)
    dw, db = torch.full((10, 16), 3.0, device="cuda"), torch.full((10,), 3.0, device="cuda")
    ops.gated_linear_bwd(h, x, w, gu, dw=dw, db=db, accumulate=True)
    assert bool((dw == 3).all()) and bool((db == 3).all())
    ops.gated_linear_bwd(h, x, w, gu, dw=dw, db=db)
    assert bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("m", [3, 400])
def test_captured_and_other_stream(m):
    d, f = 256, 320
    x, w, b, dh = make(m, d, f, torch.bfloat16, True)

    def step():
        h, gu = ops.gated_linear_fwd(x, w, b, save=True)
        return (h, gu, *ops.gated_linear_bwd(dh, x, w, gu))
    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, step()):
            assert torch.equal(p, q), i


# fp32 products that are taken from bf16 pieces of their operands: each term keeps all
# but 4.01 u (the two parts that are left out, 2^-16·2^-8 each, and what three pieces
# leave of each operand, 2^-24), and only hi·hi sums at full size: k/4 additions and 5
# times as many of less than 2^-7.
@pytest.mark.parametrize("m,d,f,spread", [(2150, 605, 1237, 0), (1600, 768, 1024, 20), (700, 1500, 2500, 0),
                                          (130, 2048, 4096, 20), (6001, 640, 200, 20)])
def test_large_in_fp32(m, d, f, spread):
    x, w, b, dh = make(m, d, f, torch.float32, True, seed=m)
    g = torch.Generator(device="cuda").manual_seed(m + 1)
    if spread:   # rows of very different magnitudes
        for t in (x, dh):
            t.mul_(torch.exp2(torch.randint(-spread, 2, (m, 1), generator=g, device="cuda").float()))

    def err(k, mag):
        return (0.26 * k + 22) * U * mag
    gu64 = x.double() @ w.double().t() + b.double()
    tol = err(d, x.double().abs() @ w.double().abs().t() + b.double().abs())
    h, gu = ops.gated_linear_fwd(x, w, b, save=True)
    torch.cuda.synchronize()
    near(gu, gu64, tol, "gu")
    a, da = act64("silu", gu64[:, :f])
    u, eg, eu = gu64[:, f:], tol[:, :f], tol[:, f:]
    near(h, a * u, (18 + 2 * gu64[:, :f].square()) * U * (a * u).abs() + (1.13 + eg) * eg * u.abs() + a.abs() * eu +
         1.13 * eg * eu + 2e-5 * U * u.abs(), "h")
    gate, up = gu.double().chunk(2, -1)
    a, da = act64("silu", gate)
    v = torch.cat((dh.double() * up * da, dh.double() * a), 1)
    rel = (16 + 2 * gate * gate) * U
    ev = torch.cat((rel * (dh.double() * up).abs() * (da.abs() + 0.3), rel * (dh.double() * (a.abs() + 1e-6)).abs()), 1)
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, gu)
    torch.cuda.synchronize()
    near(dx, v @ w.double(), ev @ w.double().abs() + err(2 * f, v.abs() @ w.double().abs()), "dx")
    near(dw, v.t() @ x.double(), ev.t() @ x.double().abs() + err(m, v.abs().t() @ x.double().abs()), "dw")
    near(db, v.sum(0), ev.sum(0) + (m / 64 + 96) * U * v.abs().sum(0), "db")
    dw2 = torch.full_like(dw, 2.0)
    ops.gated_linear_bwd(dh, x, w, gu, dw=dw2, need_dx=False, need_db=False, accumulate=True)
    near(dw2, dw.double() + 2, 2 * U * (dw.double().abs() + 2), "dw accumulated")


def test_large_in_fp32_captured():
    """Split operands live in the workspace: replays between eager calls of other sizes, and another stream."""
    m, d, f = 1100, 700, 1300
    x, w, b, dh = make(m, d, f, torch.float32, True)
    small = make(200, d, f, torch.float32, True)

    def step(x, dh):
        h, gu = ops.gated_linear_fwd(x, w, b, save=True)
        return (h, gu, *ops.gated_linear_bwd(dh, x, w, gu))
    want = step(x, dh)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step(x, dh)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, dh)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        step(small[0], small[3])
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, step(x, dh)):
            assert torch.equal(p, q), i


def test_large_in_fp32_keeps_nan():
    """NaN and infinity spread to what they reach and to nothing else."""
    m, d, f = 1100, 700, 1300
    x, w, b, dh = make(m, d, f, torch.float32, False)
    clean = ops.gated_linear_fwd(x, w)[0]
    x[7, 3], x[900, 699] = float("nan"), float("inf")
    h, gu = ops.gated_linear_fwd(x, w, save=True)
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[7] = rows[900] = False
    assert torch.equal(h[rows], clean[rows])
    assert bool(gu[7].isnan().all()) and not bool(gu[900].isfinite().any())
    dh[5, 9] = float("nan")
    x.nan_to_num_(0, 0, 0)
    gu = ops.gated_linear_fwd(x, w, save=True)[1]
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, gu)
    assert bool(dx[5].isnan().all()) and bool(dx[torch.arange(m, device="cuda") != 5].isfinite().all())
    hit = torch.zeros(2 * f, dtype=torch.bool, device="cuda")
    hit[9] = hit[f + 9] = True
    assert bool(dw[hit].isnan().all()) and bool(dw[~hit].isfinite().all())
    assert torch.equal(db.isnan(), hit)


@pytest.mark.parametrize("e", [-105, 100])
def test_large_in_fp32_far_from_one(e):
    """x of 2^e: a power of two changes no rounding down to 2^-105, where the pieces of every value above 2^-110 are
    whole; a smaller one (1 of 40) is off by 2^-134 at most."""
    m, d, f = 1100, 700, 1300
    x, w, _, _ = make(m, d, f, torch.float32, False)
    xs = torch.ldexp(x, torch.tensor(e, device="cuda"))
    got = ops.gated_linear_fwd(xs, w, save=True)[1]
    mag = xs.double().abs() @ w.double().abs().t()
    tol = (0.26 * d + 22) * U * mag + 2.0 ** -134 * w.double().abs().sum(1)
    near(got, xs.double() @ w.double().t(), tol, "gu")
