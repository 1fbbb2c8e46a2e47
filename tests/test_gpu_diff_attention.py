"""Differential attention and its gradients against the formulas in float64.

Tolerances, per element, with u the half step of what is rounded (bf16 2^-8 of the
value at most, half of finfo.eps = 2^-7; fp32 2^-24) and e = 2^-24: a score is a sum of dh products in fp32, off by
at most (dh + 4)·e·Σ|q·k|·scale =: s; a probability is off by 2·s + 64·e of itself, and
where it enters a product in bf16 by 2^-8 more: call that w.  So o is off by
w·(Σ p₁|v| + λ Σ p₂|v|) + its own rounding; dv by w·Σ (p₁ + λ p₂)|dO|; dz, which takes
the forward's o and o₂ as they were stored (those are what the reference takes too), by
w·p·(|dp| + |D|) + the sums' (dv + 8)·e of Σ|dO·v|, and dq, dk by the sums of those.
Sums of n terms add at most n·e of the sum of magnitudes (n below 2^12: 2^-12)."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(b, t, s, h, hk, dh, dv, dt, seed=0, token_lam=False, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)
    if packed and t == s:
        w = n(b, t, 2 * (h + hk) * dh + hk * dv)
        q = w[..., :2 * h * dh].unflatten(-1, (2 * h, dh))
        k = w[..., 2 * h * dh:2 * (h + hk) * dh].unflatten(-1, (2 * hk, dh))
        v = w[..., 2 * (h + hk) * dh:].unflatten(-1, (hk, dv))
    else:
        q, k, v = n(b, t, 2 * h, dh, std=1.5), n(b, s, 2 * hk, dh), n(b, s, hk, dv)
    lam = torch.rand((b, t, h) if token_lam else (h,), generator=g, device="cuda") * 1.2 - 0.2
    return q, k, v, lam


def seen(b, t, s, causal, lengths, start):
    """[b, t, s]: whether a query sees a key."""
    j = torch.arange(s, device="cuda")[None, None]
    i = torch.arange(t, device="cuda")[None, :, None]
    m = torch.ones((b, t, s), dtype=torch.bool, device="cuda")
    if causal:
        m &= j <= i + (0 if start is None else start.long()[:, None, None])
    if lengths is not None:
        m &= j < lengths.long().clamp(0, s)[:, None, None]
    return m


class Ref:
    """Forward in float64, with the sums of magnitudes that the tolerances need."""

    def __init__(self, q, k, v, lam, mask, scale):
        self.args = q, k, v, lam
        b, t, h2, dh = q.shape
        hk = v.shape[2]
        self.h, self.g = h2 // 2, h2 // 2 // hk
        self.q = q.double().view(b, t, self.h, 2, dh).permute(0, 2, 3, 1, 4)
        kk = k.double().view(b, -1, hk, 2, dh).permute(0, 2, 3, 1, 4)
        self.k = kk.repeat_interleave(self.g, 1)
        self.v = v.double().permute(0, 2, 1, 3).repeat_interleave(self.g, 1)
        self.lam = (lam.double().permute(0, 2, 1) if lam.dim() == 3 else lam.double()[None, :, None].expand(b, -1, t))[..., None]
        m = mask[:, None, None]
        self.scale = scale
        z = (self.q @ self.k.transpose(3, 4) * scale).masked_fill(~m, -math.inf)
        top = z.amax(4, keepdim=True) if z.shape[4] else z.new_zeros(z.shape[:4] + (1,))
        top = torch.where(top > -math.inf, top, 0.0)
        e = (z - top).exp()
        self.l = e.sum(4, keepdim=True)
        self.p = torch.where(self.l > 0, e / self.l, 0.0)
        self.lse = (top + self.l.log())[..., 0].flatten(1, 2)
        self.o1, self.o2 = (self.p @ self.v[:, :, None]).unbind(2)
        self.o = self.o1 - self.lam * self.o2
        size = (self.q.abs() @ self.k.abs().transpose(3, 4) * scale).masked_fill(~m, 0.0)
        # an error of the largest score shifts the whole row: the row's largest s
        self.s = (dh + 4) * E * (size.amax(4, keepdim=True) if size.shape[4] else 0.0) + 64 * E


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    inf = want.isinf()
    assert torch.equal(got.double()[inf], want[inf]), what
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else E
    tol = tol + half * 1.01 * (want.abs() + tol) + 1e-30
    err = (got.double() - want).abs()[~inf]
    tol = tol.expand_as(want)[~inf]
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max())} of the tolerance"


def check(q, k, v, lam, *, causal=False, scale=None, lengths=None, start=None, backward=True, seed=1, out=False):
    b, t, h2, dh = q.shape
    s, hk, dv = v.shape[1:]
    h, dt = h2 // 2, q.dtype
    kw = dict(causal=causal, scale=scale, lengths=lengths, q_start=start)
    scale = dh ** -0.5 if scale is None else scale
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True, **kw)
    torch.cuda.synchronize()
    mask = seen(b, t, s, causal, lengths, start)
    r = Ref(q, k, v, lam, mask, scale)
    w = 2 * r.s + (2.0 ** -8 if dt == torch.bfloat16 else 0.0) + 2.0 ** -12 * (2.0 ** -12 if dt == torch.float32 else 1.0)
    mag = (w * r.p) @ r.v.abs()[:, :, None]
    tol2 = mag[:, :, 1]
    tol1 = mag[:, :, 0]
    close(o2.transpose(1, 2), r.o2, tol2, "o2")
    close(o.transpose(1, 2), r.o, tol1 + r.lam.abs() * tol2, "o")
    close(lse, r.lse, r.s[..., 0].flatten(1, 2) * 2 + 4 * E * torch.where(r.lse.isinf(), 0.0, r.lse.abs()), "lse")
    again = ops.diff_attention_fwd(q, k, v, lam, **kw)
    assert again[2] is None and torch.equal(again[0], o) and torch.equal(again[1], lse)
    if not backward:
        return o, lse, o2
    g = torch.Generator(device="cuda").manual_seed(seed)
    do = torch.randn((b, t, h, dv), generator=g, device="cuda").to(dt)
    dq, dk, dvv, dlam = ops.diff_attention_bwd(do, q, k, v, lam, o, o2, lse, **kw)
    torch.cuda.synchronize()
    d = do.double().transpose(1, 2)
    oo, oo2 = o.double().transpose(1, 2), o2.double().transpose(1, 2)
    D2 = (d * oo2).sum(3, keepdim=True)
    D1 = (d * oo).sum(3, keepdim=True) + r.lam * D2
    dp = d @ r.v.transpose(2, 3)
    dpm = d.abs() @ r.v.abs().transpose(2, 3)
    D2m = (d * oo2).abs().sum(3, keepdim=True)
    D1m = (d * oo).abs().sum(3, keepdim=True) + r.lam.abs() * D2m
    p1, p2 = r.p.unbind(2)
    # the probabilities take the fp32 lse as it is
    ww = w + 4 * E * torch.where(r.lse.isinf(), 0.0, r.lse.abs()).unflatten(1, (h, 2))[..., None]
    w1, w2 = ww.unbind(2)
    sums = (dv + 8) * E
    dz = torch.stack((p1 * (dp - D1), -r.lam * p2 * (dp - D2)), 2)
    dzt = torch.stack((p1 * (w1 * (dp - D1).abs() + sums * (dpm + D1m)),
                       r.lam.abs() * p2 * (w2 * (dp - D2).abs() + sums * (dpm + D2m))), 2)
    # sums over keys or rows in fp32
    many = (max(s, t * r.g) + 8) * E
    dzt = dzt + many * dz.abs()

    def heads(x):       # sum over the heads that share a key head
        return x.unflatten(1, (hk, r.g)).sum(2)
    close(dq.view(b, t, h, 2, dh).permute(0, 2, 3, 1, 4), dz @ r.k * scale, dzt @ r.k.abs() * scale, "dq")
    close(dk.view(b, s, hk, 2, dh).permute(0, 2, 3, 1, 4), heads(dz.transpose(3, 4) @ r.q) * scale,
          heads(dzt.transpose(3, 4) @ r.q.abs()) * scale, "dk")
    pw, pt = p1 - r.lam * p2, (w1 + many) * p1 + (w2 + many) * r.lam.abs() * p2
    close(dvv.permute(0, 2, 1, 3), heads(pw.transpose(2, 3) @ d), heads(pt.transpose(2, 3) @ d.abs()), "dv")
    dl, dlt = -D2[..., 0].transpose(1, 2), sums * D2m[..., 0].transpose(1, 2)
    if lam.dim() == 3:
        close(dlam, dl, dlt, "dlam")
    else:
        close(dlam, dl.sum((0, 1)), dlt.sum((0, 1)), "dlam")
    return o, lse, o2, do, dq, dk, dvv, dlam


SHAPES = {   # b, t, s, h, hk, dh, dv
    "f32": [(1, 1, 1, 1, 1, 4, 8), (2, 3, 5, 2, 1, 16, 32), (2, 64, 64, 2, 2, 16, 32), (1, 65, 130, 4, 2, 20, 41),
            (1, 200, 200, 3, 3, 40, 80), (1, 129, 129, 4, 1, 64, 128), (2, 70, 70, 2, 2, 64, 64)],
    "bf16": [(1, 1, 1, 1, 1, 8, 16), (2, 3, 5, 2, 1, 16, 32), (2, 64, 64, 2, 2, 32, 64), (1, 129, 257, 4, 2, 64, 128),
             (1, 300, 300, 6, 3, 40, 80), (1, 200, 200, 2, 1, 72, 144), (1, 150, 150, 4, 1, 128, 256), (2, 260, 260, 2, 2, 96, 96),
             (1, 130, 130, 2, 2, 64, 72), (1, 65, 100, 2, 1, 20, 41), (1, 90, 90, 2, 2, 100, 199)],
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt,shape", [(d, x) for d in SHAPES for x in SHAPES[d]])
def test_against_float64(dt, shape, causal):
    b, t, s, h, hk, dh, dv = shape
    q, k, v, lam = make(*shape, DT[dt], token_lam=(t + dh) % 2 == 1, packed=True)
    check(q, k, v, lam, causal=causal)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("t,s", [(1, 300), (5, 700), (40, 1000)])
def test_lengths_and_offsets(dt, t, s):
    """Padded sequences, empty ones, rows that see nothing, queries at the end of a cache."""
    b, h, hk, dh, dv = 5, 4, 2, 32, 64
    q, k, v, lam = make(b, t, s, h, hk, dh, dv, DT[dt], seed=3)
    lengths = torch.tensor([s, s - 7, 0, t + 64, 1], dtype=torch.int32, device="cuda")
    check(q, k, v, lam, lengths=lengths)
    check(q, k, v, lam, lengths=lengths, start=lengths - t, causal=True)     # (row 4 begins before its keys)
    start = torch.tensor([0, s - 3, 5, -2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    check(q, k, v, lam, start=start, causal=True)
    check(q, k, v, lam, start=start, causal=True, lengths=torch.tensor([-5, s + 9, 70, 64, 65], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dt,dh,dv", [("bf16", 16, 32), ("bf16", 64, 128), ("bf16", 96, 192), ("bf16", 128, 256), ("f32", 64, 128),
                                      ("bf16", 20, 40)])
@pytest.mark.parametrize("b,t,s,h,hk", [(1, 1, 5000, 4, 4), (2, 1, 2049, 8, 2), (1, 7, 3000, 8, 1), (1, 33, 1500, 3, 1)])
def test_keys_split_over_workgroups(b, t, s, h, hk, dt, dh, dv):
    q, k, v, lam = make(b, t, s, h, hk, dh, dv, DT[dt], seed=4)
    lengths = torch.tensor([s - 1, 130][:b], dtype=torch.int32, device="cuda")
    check(q, k, v, lam, lengths=lengths, start=lengths - t, causal=True, backward=False)
    check(q, k, v, lam, backward=False)


@pytest.mark.parametrize("dt", DT)
def test_values_behind_the_last_key_are_not_read(dt):
    """NaN in unused slots of a cache, forward and backward, few rows and many."""
    for t, s in ((1, 1000), (200, 300)):
        q, k, v, lam = make(2, t, s, 2, 1, 32, 64, DT[dt], seed=5)
        lengths = torch.tensor([t + 37, t + 1], dtype=torch.int32, device="cuda")
        kw = dict(causal=True, lengths=lengths, q_start=lengths - t)
        k2, v2 = k.clone(), v.clone()
        for i, n in enumerate(lengths.tolist()):
            k2[i, n:], v2[i, n:] = math.nan, math.nan
        a = ops.diff_attention_fwd(q, k, v, lam, save=True, **kw)
        c = ops.diff_attention_fwd(q, k2, v2, lam, save=True, **kw)
        assert all(torch.equal(x, y) for x, y in zip(a, c))
        do = torch.randn_like(a[0])
        x = ops.diff_attention_bwd(do, q, k, v, lam, a[0], a[2], a[1], **kw)
        y = ops.diff_attention_bwd(do, q, k2, v2, lam, a[0], a[2], a[1], **kw)
        assert all(torch.equal(p, r) for p, r in zip(x, y))
        for i, n in enumerate(lengths.tolist()):
            assert not x[1][i, n:].any() and not x[2][i, n:].any()


@pytest.mark.parametrize("dt", DT)
def test_large_scores(dt):
    """One key takes nearly all of a row: probabilities of 1 and of 0."""
    q, k, v, lam = make(1, 100, 100, 2, 2, 32, 64, DT[dt], seed=6)
    check(q * 8, k * 4, v, lam, causal=True)


def test_head_major_and_given_outputs():
    b, t, h, hk, dh, dv = 2, 150, 4, 2, 64, 128
    q, k, v, lam = make(b, t, t, h, hk, dh, dv, torch.bfloat16, seed=7)
    want = ops.diff_attention_fwd(q, k, v, lam, causal=True, save=True)
    hm = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    out = torch.empty(b, h, t, dv, dtype=q.dtype, device="cuda").transpose(1, 2)
    got = ops.diff_attention_fwd(*hm, lam, causal=True, save=True, out=out)
    assert got[0] is out and all(torch.equal(x, y) for x, y in zip(got, want))
    do = torch.randn_like(want[0])
    ref = ops.diff_attention_bwd(do, q, k, v, lam, want[0], want[2], want[1], causal=True)
    n = 2 * (h + hk) * dh + hk * dv
    packed = torch.full((b, t, n + 8), 3.0, dtype=q.dtype, device="cuda")
    views = (packed[..., :2 * h * dh].unflatten(-1, (2 * h, dh)), packed[..., 2 * h * dh:2 * (h + hk) * dh].unflatten(-1, (2 * hk, dh)),
             packed[..., 2 * (h + hk) * dh:n].unflatten(-1, (hk, dv)))
    dlam = torch.ones_like(lam)
    got = ops.diff_attention_bwd(do.transpose(1, 2).contiguous().transpose(1, 2), *hm, lam, out, want[2], want[1], causal=True,
                                 out=views, dlam=dlam, accumulate=True)
    assert all(torch.equal(x, y) for x, y in zip(got[:3], ref[:3])) and bool((packed[..., n:] == 3).all())
    assert torch.equal(dlam, 1 + ref[3])
    # rows that are not aligned: another kernel, the same up to roundings
    odd = torch.empty(b, t, n + 1, dtype=q.dtype, device="cuda")
    oq = odd[..., 1:1 + 2 * h * dh].unflatten(-1, (2 * h, dh))
    oq.copy_(q)
    check(oq, k, v, lam, causal=True)


def test_nothing_to_do():
    for dt in DT.values():
        q, k, v, lam = make(2, 3, 0, 2, 1, 16, 32, dt)
        o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
        assert not o.any() and not o2.any() and bool((lse == -math.inf).all())
        dq, dk, dv, dlam = ops.diff_attention_bwd(torch.ones_like(o), q, k, v, lam, o, o2, lse)
        assert not dq.any() and dk.numel() == 0 and not dlam.any()
        q, k, v, lam = make(2, 0, 5, 2, 1, 16, 32, dt)
        o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
        dq, dk, dv, dlam = ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse)
        assert o.numel() == 0 and not dk.any() and not dv.any() and not dlam.any()


def test_gradients_against_differences():
    """fp32 gradients against central differences of the formula in float64."""
    q, k, v, lam = make(1, 20, 20, 2, 1, 16, 32, torch.float32, seed=8)
    mask = seen(1, 20, 20, True, None, None)
    o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, causal=True, save=True)
    w = torch.randn_like(o)
    grads = ops.diff_attention_bwd(w, q, k, v, lam, o, o2, lse, causal=True)

    def loss(*a):
        return float((Ref(*a, mask, 0.25).o.transpose(1, 2) * w.double()).sum())
    for i, gr in enumerate(grads):
        args = [x.double() for x in (q, k, v, lam)]
        way = torch.randn_like(args[i])
        step = 1e-5
        up, down = (loss(*[x + sg * step * way if j == i else x for j, x in enumerate(args)]) for sg in (1, -1))
        want = float((gr.double() * way).sum())
        assert abs((up - down) / (2 * step) - want) <= 1e-4 * (1 + float((gr.double() * way).norm())), i


def test_captured_and_on_another_stream():
    """Two graphs on one context replayed in turn, with eager work between, one with split keys."""
    runs, s = [], torch.cuda.Stream()
    for i, (t, n) in enumerate(((1, 3000), (200, 200))):
        q, k, v, lam = make(2, t, n, 4, 2, 64, 128, torch.bfloat16, seed=i)

        def work(q=q, k=k, v=v, lam=lam):
            o, lse, o2 = ops.diff_attention_fwd(q, k, v, lam, save=True)
            return (o, lse, o2) + ops.diff_attention_bwd(o, q, k, v, lam, o, o2, lse)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = work()
        runs.append((graph, out, work, q))
    for i in range(3):
        for graph, out, work, q in runs:
            q.copy_(torch.randn_like(q))
            graph.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in out]
            for a, b in zip(got, work()):
                assert torch.equal(a, b), i
