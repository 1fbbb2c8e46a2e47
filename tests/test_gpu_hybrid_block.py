"""Differential attention, the gated linear recurrence and Adam over many tensors as they
are used together: a block of both layers with scored logits, trained with moments of 8
bits and served token by token, through the host layer's differentiable functions and
through thot_amd.ops, against the same block in float64.

Tolerances: forward and backward pass through about 40 operations.  fp32: each leaves at
most 64 half steps (2^-24) of its result's size (sums of up to 4096 terms), and what
follows enlarges an error at most fourfold: 40·64·4·2^-24 = 6.1e-4 of the 2-norm.
bf16: one half step (2^-8) each: 40·2^-8 = 0.16."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
TOL = {torch.float32: 40 * 64 * 4 * 2.0 ** -24, torch.bfloat16: 40 * 2.0 ** -8}
B, T, H, HK, DH, V = 2, 300, 4, 2, 32, 500
E = 2 * H * DH
NQ, NK = 2 * H * DH, 2 * HK * DH            # columns of the maps' queries and keys; values: as many as keys
MASTER32 = ("lam",)


@pytest.fixture(scope="module")
def host():
    from thot_amd import _nott_host
    return _nott_host


def parameters(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*s, std):
        return torch.randn(s, generator=g, device="cuda") * std
    p = {"ln1": 1 + n(E, std=0.1), "ln1b": n(E, std=0.1), "wqkv": n(NQ + 2 * NK, E, std=E ** -0.5),
         "gq": 1 + n(DH, std=0.1), "gk": 1 + n(DH, std=0.1), "lam": 0.5 + n(H, std=0.2), "wo": n(E, E, std=E ** -0.5),
         "ln2": 1 + n(E, std=0.1), "ln2b": n(E, std=0.1), "wxg": n(2 * E, E, std=E ** -0.5),
         "ws": n(E, E, std=E ** -0.5), "wv": n(V, E, std=E ** -0.5)}
    x = n(B, T, E, std=1.0)
    y = torch.randint(0, V, (B * T,), generator=g, device="cuda")
    y[3] = -100
    weight = torch.randn(B * T, generator=g, device="cuda")
    pos = torch.arange(T, device="cuda").repeat(B, 1)[None].contiguous()
    reset = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    reset[0, 77] = reset[1, 256] = True
    return p, x, y, weight, pos, reset


def reference(p, x, y, weight, pos, reset, dt):
    """Loss and gradients in float64, parameters and input as the type holds them."""
    q = leaf = {k: (v if k in MASTER32 else v.to(dt)).double().requires_grad_() for k, v in p.items()}
    h = x.to(dt).double()
    F_ = torch.nn.functional
    ang = pos[0].double()[..., None] * ops.rope_frequencies(DH)
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]

    def rope(v, g):
        v = v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * g
        a, b = v.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).transpose(1, 2)
    qkv = F_.layer_norm(h, (E,), q["ln1"], q["ln1b"], 1e-5) @ q["wqkv"].t()
    qh = rope(qkv[..., :NQ].reshape(B, T, 2 * H, DH), q["gq"])
    kh = rope(qkv[..., NQ:NQ + NK].reshape(B, T, 2 * HK, DH), q["gk"])
    vh = qkv[..., NQ + NK:].reshape(B, T, HK, 2 * DH).transpose(1, 2)
    kh = kh.reshape(B, HK, 2, T, DH).repeat_interleave(H // HK, 1).reshape(B, 2 * H, T, DH)
    s = qh @ kh.transpose(2, 3) * DH ** -0.5
    m = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), -math.inf).softmax(-1)
    m = m.reshape(B, H, 2, T, T)
    o = (m[:, :, 0] - q["lam"][:, None, None] * m[:, :, 1]) @ vh.repeat_interleave(H // HK, 1)
    h = h + o.transpose(1, 2).reshape(B, T, E) @ q["wo"].t()
    u, g = (F_.layer_norm(h, (E,), q["ln2"], q["ln2b"], 1e-5) @ q["wxg"].t()).chunk(2, -1)
    a = g.sigmoid()
    st, states = torch.zeros(B, E, dtype=torch.float64, device="cuda"), []
    for i in range(T):
        st = torch.where(reset[:, i, None], 0.0, st) * a[:, i] + (1 - a[:, i]) * u[:, i]
        states.append(st)
    h = h + torch.stack(states, 1) @ q["ws"].t()
    lp = (h.reshape(B * T, E) @ q["wv"].t()).log_softmax(-1)
    hit = torch.where(y >= 0, lp.gather(1, y.clamp_min(0)[:, None])[:, 0], 0.0)
    ent = -(lp.exp() * lp).sum(-1)
    loss = (hit * weight.double()).sum() + 0.1 * ent.sum()
    loss.backward()
    return hit.detach(), ent.detach(), {k: v.grad for k, v in leaf.items()}


class Block:
    """The block through the host layer; fp32 masters, working copies in dt."""

    def __init__(self, host, p, dt):
        self.h, self.dt = host, dt
        self.p = {k: v.clone().requires_grad_() for k, v in p.items()}
        self.c = {k: None if k in MASTER32 else v.detach().to(dt) for k, v in self.p.items()}
        self.freq = ops.rope_frequencies(DH)

    def lin(self, x, w):
        return self.h.linear(x, self.p[w], None, self.c[w])

    def __call__(self, x, y, weight, pos, reset):
        h, p, c = self.h, self.p, self.c
        x = x.to(self.dt)
        qkv = self.lin(h.layer_norm(x, p["ln1"], p["ln1b"], c["ln1"], c["ln1b"]), "wqkv")
        q, k = qkv[..., :NQ].unflatten(-1, (2 * H, DH)), qkv[..., NQ:NQ + NK].unflatten(-1, (2 * HK, DH))
        v = qkv[..., NQ + NK:].unflatten(-1, (HK, 2 * DH))
        q, k = h.qk_norm_rope(q, k, pos, self.freq, p["gq"], p["gk"], c["gq"], c["gk"])
        o = h.diff_attention(q.transpose(1, 2), k.transpose(1, 2), v, p["lam"], True)
        x = x + self.lin(o.flatten(2), "wo")
        ug = self.lin(h.layer_norm(x, p["ln2"], p["ln2b"], c["ln2"], c["ln2b"]), "wxg")
        s, _ = h.linear_scan(ug[..., :E], ug[..., E:], None, reset)
        x = x + self.lin(s, "ws")
        lp, ent = h.token_logprob(self.lin(x.reshape(B * T, E), "wv"), y)
        return (lp * weight).sum() + 0.1 * ent.sum(), lp, ent


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dt", DT)
def test_block_against_float64(host, dt):
    dt = DT[dt]
    p, *args = parameters()
    hit, ent, grads = reference(p, *args, dt)
    blk = Block(host, p, dt)
    loss, lp, e = blk(*args)
    loss.backward()
    torch.cuda.synchronize()
    assert off(lp.detach(), hit) <= TOL[dt] and off(e.detach(), ent) <= TOL[dt]
    for k, g in grads.items():
        assert off(blk.p[k].grad, g) <= TOL[dt], k
    # a second pass adds into the same gradients
    before = {k: v.grad.clone() for k, v in blk.p.items()}
    blk(*args)[0].backward()
    torch.cuda.synchronize()
    for k, v in blk.p.items():
        assert off(v.grad, 2 * before[k].double()) <= 2.0 ** -20, k


@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps(host, bits):
    """Steps of the block with the optimizer over its parameters, gradients clipped by a
    factor on the device: the bits of the same steps by hand through thot_amd.ops."""
    p, *args = parameters(4)
    blk, twin = Block(host, p, torch.bfloat16), Block(host, p, torch.bfloat16)
    names = list(p)
    decay, plain = [k for k in names if p[k].dim() == 2], [k for k in names if p[k].dim() == 1]
    opt = host.MultiTensorAdamW([[blk.p[k] for k in decay], [blk.p[k] for k in plain]], [2e-3, 1e-3], [0.1, 0.0], bits=bits)
    for k in names:
        if k not in MASTER32:
            blk.c[k] = opt.bf16_copy(blk.p[k])
    held = [ops.AdamMoments([twin.p[k].detach() for k in ks], bits=bits, copies=[twin.c[k] for k in ks])
            for ks in (decay, plain)]
    factor = torch.ones((), device="cuda")
    opt.set_grad_scale(factor)
    for step in range(1, 4):
        for b in (blk, twin):
            for v in b.p.values():
                v.grad = None
            b(*args)[0].backward()
        square = torch.stack([v.grad.square().sum() for v in blk.p.values()]).sum()
        factor.copy_(torch.clamp(1.0 / square.sqrt(), max=1.0))
        opt.step()
        for ks, h, lr, wd in zip((decay, plain), held, (2e-3, 1e-3), (0.1, 0.0)):
            ops.adam_multi_step(h, [twin.p[k].grad for k in ks], lr=lr, weight_decay=wd, step=step, grad_scale=factor)
        torch.cuda.synchronize()
        for k in names:
            assert torch.equal(blk.p[k], twin.p[k]), (step, k)
            assert k in MASTER32 or torch.equal(blk.c[k], twin.c[k]), (step, k)
            assert not torch.equal(blk.p[k].detach(), p[k]), (step, k)
    for ks, h in zip((decay, plain), held):
        for i, k in enumerate(ks):
            assert torch.equal(opt.exp_avg(blk.p[k]), h.exp_avg(i)) and torch.equal(opt.exp_avg_sq(blk.p[k]), h.exp_avg_sq(i))


def test_captured_while_an_eager_graph_lives(host):
    """Forward, backward and step captured once and replayed, while the graph of an eager
    pass over the same parameters is kept."""
    p, *args = parameters(2)
    x = args[0]
    blk = Block(host, p, torch.bfloat16)
    names = [k for k in p if k not in MASTER32]
    for v in blk.p.values():
        v.grad = torch.zeros_like(v)
    moments = ops.AdamMoments([v.detach() for v in blk.p.values()], bits=8, copies=[blk.c[k] for k in blk.p])
    hyper = torch.tensor([1e-3, 0.9, 0.999, 1e-8, 0.0], dtype=torch.float64, device="cuda")
    state = torch.zeros(8, dtype=torch.int64, device="cuda")

    def train():
        loss, lp, ent = blk(*args)
        loss.backward()
        ops.adam_multi_step_graph(moments, [v.grad for v in blk.p.values()], hyper, state, weight_decay_nonzero=False,
                                  zero_grad=True)
        return lp.detach(), ent.detach()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            train()
    torch.cuda.current_stream().wait_stream(s)
    kept = blk(*args)       # an eager graph that is not run backward yet
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = train()
    torch.cuda.synchronize()

    def snapshot():
        torch.cuda.synchronize()
        return [t.clone() for t in (*(v.detach() for v in blk.p.values()), *(blk.c[k] for k in names), moments.m.view(torch.uint8),
                                    moments.v.view(torch.uint8), moments.scale, state)]

    def restore(saved):
        # (.data: the kept graph is run backward over the values as they are then)
        for t, v in zip((*(v.data for v in blk.p.values()), *(blk.c[k].data for k in names), moments.m.view(torch.uint8),
                         moments.v.view(torch.uint8), moments.scale, state), saved):
            t.copy_(v)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        start = snapshot()
        graph.replay()
        got = snapshot()
        restore(start)
        want = train()
        after = snapshot()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert all(torch.equal(a, b) for a, b in zip(got, after)), i
        assert int(state[0]) == 3 + i
        assert all(not bool(v.grad.any()) for v in blk.p.values()), i
    kept[0].backward()
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(v.grad).all()) for v in blk.p.values())


@pytest.mark.parametrize("dt", DT)
def test_serving_step_matches_the_prompt(dt):
    """A prompt whose tokens follow one by one (keys and values in a cache, the
    recurrence's state carried) gives what the whole prompt gives."""
    dt = DT[dt]
    p, x, *_ = parameters(3)
    x = x.to(dt)
    wqkv, wxg, lam = p["wqkv"].to(dt), p["wxg"].to(dt), p["lam"]
    kc = torch.full((B, T, 2 * HK, DH), math.nan, device="cuda", dtype=dt)
    vc = torch.full((B, T, HK, 2 * DH), math.nan, device="cuda", dtype=dt)

    def run(x, at, state):
        n = x.shape[1]
        qkv = ops.linear_fwd(x, wqkv)
        kc[:, at:at + n] = qkv[..., NQ:NQ + NK].unflatten(-1, (2 * HK, DH))
        vc[:, at:at + n] = qkv[..., NQ + NK:].unflatten(-1, (HK, 2 * DH))
        start = torch.full((B,), at, dtype=torch.int32, device="cuda")
        o, _, _ = ops.diff_attention_fwd(qkv[..., :NQ].unflatten(-1, (2 * H, DH)), kc, vc, lam, causal=True,
                                         lengths=start + n, q_start=start)
        ug = ops.linear_fwd(x, wxg)
        s, last, _ = ops.linear_scan_fwd(ug[..., :E], ug[..., E:], state)
        return o, s, last
    whole = run(x, 0, None)
    kc.fill_(math.nan)
    vc.fill_(math.nan)
    o, s, last = run(x[:, :T - 9].contiguous(), 0, None)
    parts = [(o, s)]
    for t in range(T - 9, T):
        o, s, last = run(x[:, t:t + 1].contiguous(), t, last)
        parts.append((o, s))
    torch.cuda.synchronize()
    for i in range(2):
        got = torch.cat([q[i] for q in parts], 1)
        # the projections may sum in another order (half a step of their results, of size 1 to 4), and
        # softmax, states and outputs pass that on: a few half steps of values of that size
        tol = torch.finfo(dt).eps * 16 * (whole[i].double().abs() + 4)
        assert bool(((got.double() - whole[i].double()).abs() <= tol).all())
    assert bool(((last - whole[2]).abs() <= torch.finfo(dt).eps * 16 * (whole[2].abs() + 4)).all())
