"""adam_multi_step (Adam / AdamW over many tensors, moments in 32 or 8 bits).

32 bits: the bits of nott_adam_step, which other tests hold to the reference.  8 bits
against the formulas in float64: with u = 2^-24, a new moment before its rounding is two
products and a sum away (4·u); root, reciprocal and their products add at most 8·u to the
update; a code is off by at most half a step, 2^-4 of the value or half the least step
(2^-10) of the scale, and what it stands for is a product with the scale away (2·u)."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")]
SIZES = [1, 3, 255, 256, 257, 1000, 4096, 4097, 12288, 70001, 0, 5, 8192 + 24]


def make(sizes, pt, gt, seed=0, offset=0):
    """Parameters and gradients; offset: elements by which they miss their alignment."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(n, std, dt):
        return (torch.randn(n + offset, generator=g, device="cuda") * std).to(dt)[offset:]
    return [one(n, 0.05, DT[pt]) for n in sizes], [one(n, 0.01 * 10 ** (i % 3 - 1), DT[gt]) for i, n in enumerate(sizes)]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("pt,gt", TYPES)
@pytest.mark.parametrize("decoupled,wd", [(True, 0.01), (False, 0.02), (True, 0.0)])
def test_32_bits_are_the_flat_step(pt, gt, decoupled, wd, offset):
    p, g = make(SIZES, pt, gt, offset=offset)
    copies = [torch.empty(t.shape, dtype=torch.bfloat16, device="cuda") for t in p]
    mo = ops.AdamMoments(p, bits=32, copies=copies)
    want = [t.clone() for t in p]
    m, v = ([torch.zeros(t.numel(), device="cuda") for t in p] for _ in range(2))
    kw = dict(lr=1e-2, beta1=0.8, beta2=0.99, eps=1e-6, weight_decay=wd)
    for step in (1, 2, 3):
        zero = step == 3
        grads = [t.clone() for t in g]
        for t in zip(want, (x.clone() for x in g), m, v):
            if t[0].numel():
                ops.adam_step(*t, step=step, decoupled=decoupled, **kw)
        ops.adam_multi_step(mo, grads, step=step, decoupled=decoupled, zero_grad=zero, **kw)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(p, want)):
            assert torch.equal(a, b) and torch.equal(copies[i], b.bfloat16()), (i, step)
            assert torch.equal(mo.exp_avg(i), m[i]) and torch.equal(mo.exp_avg_sq(i), v[i]), (i, step)
        for a, b in zip(grads, g):
            assert torch.equal(a, torch.zeros_like(b) if zero else b)


def blocks(t, rows):
    out = torch.zeros(rows * 256, dtype=torch.float64, device="cuda")
    out[:t.numel()] = t.double()
    return out.view(rows, 256)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("pt,gt", TYPES)
@pytest.mark.parametrize("decoupled,wd", [(True, 0.01), (False, 0.02)])
def test_8_bits_against_the_formulas(pt, gt, decoupled, wd, offset):
    p, g = make(SIZES, pt, gt, seed=1, offset=offset)
    mo = ops.AdamMoments(p, bits=8)
    gs = torch.tensor(0.5, device="cuda")
    lr, b1, b2, eps = 1e-2, 0.9, 0.99, 1e-8
    for step in range(1, 5):
        before = [(t.clone(), mo.exp_avg(i).double(), mo.exp_avg_sq(i).double()) for i, t in enumerate(p)]
        ops.adam_multi_step(mo, g, lr=lr, beta1=b1, beta2=b2, eps=eps, weight_decay=wd, step=step, decoupled=decoupled,
                            grad_scale=gs)
        torch.cuda.synchronize()
        for i, (p0, m0, v0) in enumerate(before):
            if not p0.numel():
                continue
            pd, ge = p0.double(), g[i].double() * 0.5
            gsize = ge.abs()
            if decoupled:
                pd = pd * (1 - lr * wd)
            else:
                # wd is rounded to fp32, so p·wd is off by U·|p·wd|, which is not small beside the sum
                # where the two cancel: a step's gradient is off by U·gsize, and with it m by (1 − β1)
                # times and r by sqrt(1 − β2) times as much (|d sqrt(a + c·g²)/dg| ≤ sqrt(c))
                gsize = gsize + (pd * wd).abs()
                ge = ge + pd * wd
            rsize = 2 * math.sqrt(1 - b2) * gsize
            m, v = m0 * b1 + ge * (1 - b1), v0 * b2 + ge * ge * (1 - b2)
            r = v.sqrt()
            denom = r / math.sqrt(1 - b2 ** step) + eps
            upd = lr / (1 - b1 ** step) * m / denom
            # m's own rounding is absolute where its two terms cancel
            msize = (m0 * b1).abs() + gsize * (1 - b1) * 2
            half = torch.finfo(p0.dtype).eps / 2
            tol = half * (pd - upd).abs() * 1.01 + 4 * U * pd.abs() + 16 * U * upd.abs() + \
                8 * U * lr / (1 - b1 ** step) * msize / denom + U * rsize / math.sqrt(1 - b2 ** step) * upd.abs() / denom
            assert bool(((p[i].double() - (pd - upd)).abs() <= tol).all()), (i, step)
            rows = -(-p0.numel() // 256)
            for got, want, size, nm in ((mo.exp_avg(i), m, msize, "m"), (mo.exp_avg_sq(i).double().sqrt(), r, r + rsize, "r")):
                scale = blocks(want, rows).abs().amax(1, keepdim=True).expand(rows, 256).reshape(-1)[:want.numel()] / 448
                # a nonzero root is at least the least code (2^-9), half a step more than rounding gives
                least = (2.0 ** -9 if nm == "r" else 2.0 ** -10) * scale
                tol = torch.maximum(want.abs() * 2.0 ** -4, least) * (1 + 2.0 ** -18) + 16 * U * size
                assert bool(((got.double() - want).abs() <= tol).all()), (nm, i, step)
            assert bool(((mo.exp_avg_sq(i) > 0) | (r == 0)).all())
    # the padding of a last block stays zero
    for i, t in enumerate(p):
        rest = mo.m[mo.first[i]:mo.first[i] - (-t.numel() // 256)].float().reshape(-1)[t.numel():]
        assert not rest.any()


def test_fading_gradients_decay_through_the_scale():
    """After gradients stop, both moments keep falling by β although no code changes."""
    p = [torch.zeros(512, device="cuda")]
    mo = ops.AdamMoments(p, bits=8)
    g = [torch.linspace(-1, 1, 512, device="cuda")]
    ops.adam_multi_step(mo, g, lr=0.0, step=1)
    v0, m0 = mo.exp_avg_sq(0).clone(), mo.exp_avg(0).clone()
    zero = [torch.zeros_like(g[0])]
    for step in range(2, 102):
        ops.adam_multi_step(mo, zero, lr=0.0, beta1=0.99, step=step)
    torch.cuda.synchronize()
    # 100 products and roots in fp32 (3 roundings each, twice in v) and one code at the most
    live = v0 > v0.max() * 2.0 ** -16
    assert bool(((mo.exp_avg_sq(0) / v0)[live] / 0.999 ** 100 - 1).abs().max() <= 600 * U)
    big = m0.abs() > m0.abs().max() * 2.0 ** -8
    assert bool(((mo.exp_avg(0) / m0)[big] / 0.99 ** 100 - 1).abs().max() <= 600 * U)


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_and_missing_gradients(bits):
    """More tensors than a launch holds, of all types in turn, some without a gradient."""
    sizes = [(37 * i) % 700 + 1 for i in range(150)]
    p, g = [], []
    for i, n in enumerate(sizes):
        a, b = make([n], *TYPES[i % 4], seed=i)
        p, g = p + a, g + b
    g = [None if i % 7 == 3 else t for i, t in enumerate(g)]
    before = [t.clone() for t in p]
    mo = ops.AdamMoments(p, bits=bits)
    ops.adam_multi_step(mo, g, lr=0.1, step=1)
    torch.cuda.synchronize()
    for i, (a, b, x) in enumerate(zip(p, before, g)):
        if x is None:
            assert torch.equal(a, b) and not mo.exp_avg(i).any()
        else:       # the first step is lr towards −sign(g)
            want = b.double() - 0.1 * x.double() / (x.double().abs() + 1e-8)
            assert bool(((a.double() - want).abs() <= torch.finfo(a.dtype).eps / 2 * want.abs() + 1e-5).all()), i


def test_gradients_that_are_not_finite():
    """The parameter shows it; other blocks are untouched."""
    p, g = make([1024], "f32", "f32")
    g[0][300] = math.nan
    g[0][600] = math.inf
    mo = ops.AdamMoments(p, bits=8)
    ops.adam_multi_step(mo, g, lr=0.1, step=1)
    torch.cuda.synchronize()
    assert p[0][300].isnan() and mo.exp_avg(0)[300].isnan() and mo.exp_avg_sq(0)[300].isnan()
    assert not mo.exp_avg(0)[600].isfinite()
    fine = torch.cat((torch.arange(256), torch.arange(768, 1024))).cuda()
    for t in (p[0], mo.exp_avg(0), mo.exp_avg_sq(0)):
        assert bool(t[fine].isfinite().all()) and bool(t[fine].abs().max() > 0)


def test_tiny_moments_count_as_zero():
    p = [torch.ones(256, device="cuda")]
    mo = ops.AdamMoments(p, bits=8)
    ops.adam_multi_step(mo, [torch.full((256,), 1e-37, device="cuda")], lr=0.0, step=1)
    torch.cuda.synchronize()
    assert not mo.exp_avg(0).any() and bool(p[0].isfinite().all())


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps(bits):
    """A captured step replayed with another learning rate and gradients, between eager work,
    is the eager step."""
    sizes = [1000, 4096, 77]
    p, g = make(sizes, "f32", "f32", seed=3)
    q = [t.clone() for t in p]
    a, b = ops.AdamMoments(p, bits=bits), ops.AdamMoments(q, bits=bits)
    hp = torch.tensor([1e-2, 0.9, 0.999, 1e-8, 0.01], dtype=torch.float64).pin_memory()
    state = torch.zeros(8, dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.adam_multi_step_graph(a, g, hp, state)
    for step in range(1, 5):
        hp[0] = 1e-2 / step
        for t in g:
            t.copy_(torch.randn_like(t) * 0.01)
        graph.replay()
        torch.cuda.synchronize()
        ops.adam_multi_step(b, g, lr=1e-2 / step, weight_decay=0.01, step=step)
        torch.cuda.synchronize()
        assert int(state[0]) == step
        for i, (x, y) in enumerate(zip(p, q)):
            assert torch.equal(x, y) and torch.equal(a.exp_avg(i), b.exp_avg(i)) and torch.equal(a.exp_avg_sq(i), b.exp_avg_sq(i))


def test_another_stream():
    p, g = make([5000], "f32", "f32")
    want = [p[0].clone()]
    ops.adam_multi_step(ops.AdamMoments(want), g, lr=0.1, step=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adam_multi_step(ops.AdamMoments(p), g, lr=0.1, step=1)
    torch.cuda.synchronize()
    assert torch.equal(p[0], want[0])
