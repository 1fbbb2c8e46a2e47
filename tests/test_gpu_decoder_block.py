"""The language-model operators as they are used together: a decoder block and
its scored logits, through the host layer's differentiable functions and through
thot_amd.ops, against the same block in float64.

Tolerances: forward and backward pass through about 36 operations.  fp32: each
leaves at most 64 half steps (2^-24) of its result's size (dot products of up to
4096 terms), and what follows enlarges an error at most fourfold: 36·64·4·2^-24 =
5.5e-4 of the 2-norm.  bf16: one half step (2^-8) each: 36·2^-8 = 0.14."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
TOL = {torch.float32: 36 * 64 * 4 * 2.0 ** -24, torch.bfloat16: 36 * 2.0 ** -8}
B, T, H, DH, F, V = 2, 48, 4, 32, 200, 500
E = H * DH


@pytest.fixture(scope="module")
def host():
    from thot_amd import _nott_host
    return _nott_host


def parameters(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*s, std):
        return torch.randn(s, generator=g, device="cuda") * std
    p = {"ln1": 1 + n(E, std=0.1), "ln1b": n(E, std=0.1), "wqkv": n(3 * E, E, std=E ** -0.5), "gq": 1 + n(DH, std=0.1),
         "gk": 1 + n(DH, std=0.1), "wo": n(E, E, std=E ** -0.5), "ln2": 1 + n(E, std=0.1), "ln2b": n(E, std=0.1),
         "wgu": n(2 * F, E, std=E ** -0.5), "bgu": n(2 * F, std=0.1), "wd": n(E, F, std=F ** -0.5),
         "wv": n(V, E, std=E ** -0.5)}
    x = n(B, T, E, std=1.0)
    y = torch.randint(0, V, (B * T,), generator=g, device="cuda")
    y[3] = -100
    weight = torch.randn(B * T, generator=g, device="cuda")
    pos = (torch.arange(T, device="cuda")[None] + torch.tensor([[5], [70000]], device="cuda"))[None].contiguous()
    return p, x, y, weight, pos


def reference(p, x, y, weight, pos, dt):
    """Loss and gradients in float64, parameters and input as the type holds them."""
    keep32 = ("bgu",)
    leaf = {k: (v if k in keep32 else v.to(dt)).double().requires_grad_() for k, v in p.items()}
    h = x.to(dt).double()
    q = leaf
    F_ = torch.nn.functional
    freq = ops.rope_frequencies(DH)
    ang = pos[0].double()[..., None] * freq
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]

    def rope(v, g):
        v = v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * g
        a, b = v.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).transpose(1, 2)
    qkv = F_.layer_norm(h, (E,), q["ln1"], q["ln1b"], 1e-5) @ q["wqkv"].t()
    qh, kh, vh = (t.reshape(B, T, H, DH) for t in qkv.chunk(3, -1))
    s = rope(qh, q["gq"]) @ rope(kh, q["gk"]).transpose(2, 3) * DH ** -0.5
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    o = (s.softmax(-1) @ vh.transpose(1, 2)).transpose(1, 2).reshape(B, T, E)
    h = h + o @ q["wo"].t()
    g, u = (F_.layer_norm(h, (E,), q["ln2"], q["ln2b"], 1e-5) @ q["wgu"].t() + q["bgu"]).chunk(2, -1)
    h = h + (F_.silu(g) * u) @ q["wd"].t()
    lp = (h.reshape(B * T, E) @ q["wv"].t()).log_softmax(-1)
    hit = torch.where(y >= 0, lp.gather(1, y.clamp_min(0)[:, None])[:, 0], 0.0)
    ent = -(lp.exp() * lp).sum(-1)
    loss = (hit * weight.double()).sum() + 0.1 * ent.sum()
    loss.backward()
    return loss.detach(), hit.detach(), ent.detach(), {k: v.grad for k, v in leaf.items()}


class Block:
    """The block through the host layer; fp32 masters, working copies in dt."""

    def __init__(self, host, p, dt):
        self.h, self.dt = host, dt
        self.p = {k: v.clone().requires_grad_() for k, v in p.items()}
        self.c = {k: v.detach().to(dt) if k != "bgu" else None for k, v in self.p.items()}
        self.freq = ops.rope_frequencies(DH)

    def lin(self, x, w, b=None):
        return self.h.linear(x, self.p[w], b, self.c[w])

    def __call__(self, x, y, weight, pos):
        h, p, c = self.h, self.p, self.c
        x = x.to(self.dt)
        qkv = self.lin(h.layer_norm(x, p["ln1"], p["ln1b"], c["ln1"], c["ln1b"]), "wqkv")
        q, k, v = (qkv[..., i * E:(i + 1) * E].unflatten(-1, (H, DH)) for i in range(3))
        q, k = h.qk_norm_rope(q, k, pos, self.freq, p["gq"], p["gk"], c["gq"], c["gk"])
        o = h.attention(q, k, v.transpose(1, 2))
        x = x + self.lin(o.transpose(1, 2).reshape(B, T, E), "wo")
        n = h.layer_norm(x, p["ln2"], p["ln2b"], c["ln2"], c["ln2b"])
        x = x + self.lin(h.gated_linear(n, p["wgu"], p["bgu"], c["wgu"]), "wd")
        lp, ent = h.token_logprob(self.lin(x.reshape(B * T, E), "wv"), y)
        return (lp * weight).sum() + 0.1 * ent.sum(), lp, ent


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dt", DT)
def test_block_against_float64(host, dt):
    dt = DT[dt]
    p, x, y, weight, pos = parameters()
    want, hit, ent, grads = reference(p, x, y, weight, pos, dt)
    blk = Block(host, p, dt)
    loss, lp, e = blk(x, y, weight, pos)
    loss.backward()
    torch.cuda.synchronize()
    assert off(lp.detach(), hit) <= TOL[dt] and off(e.detach(), ent) <= TOL[dt]
    for k, g in grads.items():
        assert off(blk.p[k].grad, g) <= TOL[dt], k
    # a second pass adds into the same gradients
    before = {k: v.grad.clone() for k, v in blk.p.items()}
    blk(x, y, weight, pos)[0].backward()
    torch.cuda.synchronize()
    for k, v in blk.p.items():
        assert off(v.grad, 2 * before[k].double()) <= 2.0 ** -20, k


def test_host_functions_are_the_calls(host):
    """Each differentiable function gives the bits of thot_amd.ops, and gradients only where asked."""
    p, x, y, _, pos = parameters(1)
    xb = x.bfloat16()
    w, wc = p["wgu"].requires_grad_(), p["wgu"].detach().bfloat16()
    xg = xb.clone().requires_grad_()
    h = host.gated_linear(xg, w, p["bgu"], wc, 2)
    h2, gu = ops.gated_linear_fwd(xb, wc, p["bgu"], act="gelu_tanh", save=True)
    assert torch.equal(h, h2)
    dh = torch.randn_like(h)
    h.backward(dh)
    dx, dw, _ = ops.gated_linear_bwd(dh, xb, wc, gu, act="gelu_tanh", need_db=False)
    assert torch.equal(xg.grad, dx) and torch.equal(w.grad, dw) and p["bgu"].grad is None
    with torch.no_grad():
        assert torch.equal(host.gated_linear(xg, w, p["bgu"], wc, 2), h2)
    q = xb.reshape(B, T, H, DH).clone().requires_grad_()
    freq = ops.rope_frequencies(DH)
    yq, yk = host.qk_norm_rope(q, q, pos, freq)     # one tensor as both, no weights
    a, b = ops.qk_norm_rope_fwd(q.detach(), q.detach(), pos, freq)
    assert torch.equal(yq, a.transpose(1, 2)) and torch.equal(yk, b.transpose(1, 2))
    g = torch.randn_like(yq)
    yq.backward(g)                                  # yk unused: its gradient is absent
    want = ops.qk_norm_rope_bwd(g.transpose(1, 2), torch.zeros_like(a), q.detach(), q.detach(), pos, freq)[0]
    assert torch.equal(q.grad, want)
    z = torch.randn(6, 40, device="cuda", requires_grad=True)
    lab = torch.tensor([0, 39, 7, -100, 3, 3], device="cuda")
    lp, ent = host.token_logprob(z, lab, 0.5)
    ent.sum().backward()                            # the entropy alone
    f = ops.token_logprob_fwd(z.detach(), lab, scale=0.5)
    one = torch.ones(6, device="cuda")
    assert torch.equal(lp, f[0]) and torch.equal(ent, f[1])
    assert torch.equal(z.grad, ops.token_logprob_bwd(z.detach(), lab, f[2], 0 * one, entropy=f[1], dentropy=one, scale=0.5))


def test_host_refusals(host):
    q = torch.zeros(2, 3, 4, 8, device="cuda")
    pos = torch.zeros(1, 2, 3, device="cuda", dtype=torch.int64)
    freq = torch.ones(4, device="cuda", dtype=torch.float64)
    for kw in (dict(k=q[:, :2]), dict(positions=pos[:, :1]), dict(positions=pos.int()), dict(inv_freq=freq.float()),
               dict(inv_freq=torch.ones(5, device="cuda", dtype=torch.float64)), dict(sections=[3]), dict(eps=-1.0),
               dict(gamma_q=torch.ones(7, device="cuda")), dict(norm=False, gamma_q=torch.ones(8, device="cuda")),
               dict(k=q.bfloat16())):
        a = dict(q=q, k=q, positions=pos, inv_freq=freq)
        a.update(kw)
        with pytest.raises((ValueError, RuntimeError)):
            host.qk_norm_rope(**a)
    x = torch.zeros(3, 8, device="cuda")
    for w in (torch.zeros(9, 8, device="cuda"), torch.zeros(4, 7, device="cuda"), torch.zeros(4, 8, device="cuda").bfloat16()):
        with pytest.raises((ValueError, RuntimeError)):
            host.gated_linear(x, w)
    with pytest.raises((ValueError, RuntimeError)):
        host.gated_linear(x, torch.zeros(4, 8, device="cuda"), act=9)
    with pytest.raises((ValueError, RuntimeError)):
        host.token_logprob(x, torch.zeros(2, device="cuda", dtype=torch.int64))
    with pytest.raises((ValueError, RuntimeError)):
        host.token_logprob(x, torch.zeros(3, device="cuda", dtype=torch.int64), 0.0)


def test_captured_while_an_eager_graph_lives(host):
    """The block's forward and backward captured once and replayed, while the graph
    of an eager pass over the same parameters is kept."""
    p, x, y, weight, pos = parameters(2)
    blk = Block(host, p, torch.bfloat16)

    def step():
        loss, lp, ent = blk(x, y, weight, pos)
        loss.backward()
        return lp.detach(), ent.detach()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    kept = blk(x, y, weight, pos)       # an eager graph that is not run backward yet
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    torch.cuda.synchronize()
    for i in range(3):
        x.copy_(torch.randn_like(x))
        for v in blk.p.values():
            v.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.grad.clone() for k, v in blk.p.items()}
        for v in blk.p.values():
            v.grad.zero_()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        for k, v in blk.p.items():
            assert torch.equal(v.grad, got[k]), (i, k)
    kept[0].backward()
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(v.grad).all()) for v in blk.p.values())


@pytest.mark.parametrize("dt", DT)
def test_serving_step_matches_the_prompt(dt):
    """A prompt taken token by token (single-token calls at their positions) gives
    what the whole prompt gives: rotated heads, gated outputs, log probabilities."""
    dt = DT[dt]
    p, x, y, _, pos = parameters(3)
    x = x.to(dt)
    wqkv, wgu, wv = (p[k].to(dt) for k in ("wqkv", "wgu", "wv"))
    freq = ops.rope_frequencies(DH)

    def run(x, pos, y):
        b, t = x.shape[:2]
        qkv = ops.linear_fwd(x, wqkv).view(b, t, 3, H, DH)
        q, k = ops.qk_norm_rope_fwd(qkv[:, :, 0], qkv[:, :, 1], pos, freq)
        h, _ = ops.gated_linear_fwd(x, wgu, p["bgu"])
        lp, _, _, tv, ti = ops.token_logprob_fwd(ops.linear_fwd(x, wv).view(b * t, V), y, top=3)
        return q, k, h, lp.view(b, t), tv.view(b, t, 3)
    whole = run(x, pos, y)
    for t in (0, 17, T - 1):
        one = run(x[:, t:t + 1].contiguous(), pos[:, :, t:t + 1].contiguous(),
                  y.view(B, T)[:, t].contiguous())
        for a, b in zip(one, whole):
            # both are within one half step of their sums' results, and of sums in another order
            tol = torch.finfo(dt).eps * (b[:, t:t + 1].double().abs() + 4)
            assert bool(((a.double() - b[:, t:t + 1].double()).abs() <= 2 * tol).all())
