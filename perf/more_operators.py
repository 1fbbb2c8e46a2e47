"""Three more language-model operators whose speed is followed, with their plain forms.

``diff``  differential attention, forward and backward: every head has two maps, and
          its output is the first map's minus lambda times the second's, with a learned
          lambda; shared key heads, padded sequences, a cache for single tokens.
``scan``  a gated linear recurrence over time, forward and backward: the state is
          multiplied by a gate and takes the input in, channel by channel.
``adam``  one step of Adam with decoupled weight decay over many tensors at once, its
          two moments held in 32 bits or in 8 (blocks of 256 with a scale each).

``run`` computes them with elementary torch operations, or, where ``own`` is
true, with this library's calls.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_CHUNK = 256     # the backward scan is given the state before every 256th token
_BLOCK = 256     # elements of a moment that share a scale
_E4M3 = 448.0    # the largest value of the 8-bit type


def listed():
    return [
        # One new token of each of 8 sequences against a cache: 4 query heads to a key
        # head, lengths of half the cache to all of it.
        {"name": "diff_step_bf16", "kind": "diff", "dir": "fwd", "dtype": "bf16", "b": 8, "t": 1, "s": 16384, "h": 16,
         "hk": 4, "dh": 64, "dv": 128, "mask": "cache", "token_lam": False, "save": False},
        # The benchmark's attention (8 x 1024 tokens, width 1024) as 8 differential heads.
        {"name": "diff_bf16", "kind": "diff", "dir": "fwd", "dtype": "bf16", "b": 8, "t": 1024, "s": 1024, "h": 8, "hk": 8,
         "dh": 64, "dv": 128, "mask": "causal", "token_lam": False, "save": True},
        # Its backward pass.
        {"name": "diff_bwd_bf16", "kind": "diff", "dir": "bwd", "dtype": "bf16", "b": 8, "t": 1024, "s": 1024, "h": 8,
         "hk": 8, "dh": 64, "dv": 128, "mask": "causal", "token_lam": False},
        # The backward pass of a long sequence with wide heads, shared key heads and a
        # lambda of every token's own.
        {"name": "diff_long_bwd_bf16", "kind": "diff", "dir": "bwd", "dtype": "bf16", "b": 1, "t": 4096, "s": 4096, "h": 16,
         "hk": 4, "dh": 128, "dv": 256, "mask": "causal", "token_lam": True},
        # A padded batch in the framework's default type, widths that end inside tiles.
        {"name": "diff_ragged_f32", "kind": "diff", "dir": "fwd", "dtype": "f32", "b": 3, "t": 777, "s": 777, "h": 6,
         "hk": 3, "dh": 40, "dv": 80, "mask": "padded", "token_lam": False, "save": True},
        # One token of each of 64 sequences: the state's update.
        {"name": "scan_step_bf16", "kind": "scan", "dir": "fwd", "dtype": "bf16", "b": 64, "t": 1, "d": 2048,
         "sigmoid": True, "mix": True, "resets": False, "save": False},
        # A training batch, gate and input as one projection leaves them.
        {"name": "scan_bf16", "kind": "scan", "dir": "fwd", "dtype": "bf16", "b": 4, "t": 4096, "d": 2048,
         "sigmoid": True, "mix": True, "resets": False, "save": True},
        # Its backward pass.
        {"name": "scan_bwd_bf16", "kind": "scan", "dir": "bwd", "dtype": "bf16", "b": 4, "t": 4096, "d": 2048,
         "sigmoid": True, "mix": True, "resets": False},
        # One long row of packed documents, decays given as they are, few channels.
        {"name": "scan_packed_bwd_f32", "kind": "scan", "dir": "bwd", "dtype": "f32", "b": 1, "t": 50001, "d": 520,
         "sigmoid": False, "mix": False, "resets": True},
        # The tensors of a small model: launches are all there is.
        {"name": "adam_small_f32", "kind": "adam", "dir": "step", "dtype": "f32", "tensors": 24, "n": 60000, "bits": 32,
         "copies": False, "odd": True},
        # A decoder's tensors: fp32 masters and gradients, bf16 working copies, 8-bit moments.
        {"name": "adam8_f32", "kind": "adam", "dir": "step", "dtype": "f32", "tensors": 24, "n": 60000000, "bits": 8,
         "copies": True, "odd": False},
        # Parameters and gradients in bf16, in odd sizes.
        {"name": "adam8_bf16", "kind": "adam", "dir": "step", "dtype": "bf16", "tensors": 28, "n": 8000000, "bits": 8,
         "copies": False, "odd": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["diff", "diff", "scan", "adam"])
    c = {"kind": kind, "dir": rng.choice(["fwd", "bwd"]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "diff":
        dh = rng.choice([16, 32, 64, 64, 72, 96, 128, 128] if c["dtype"] == "bf16" else [16, 20, 32, 40, 64])
        dv = rng.choice([2 * dh, 2 * dh, 2 * dh, dh, dh + 8])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 1, 2, 4])
        mask = rng.choice(["causal", "causal", "padded", "cache", "none"])
        pairs = 16 * 4096 * 4096 * 128 // (2 * h * dh) // (4 if c["dtype"] == "f32" else 1)
        b = rng.choice([1, 2, 3, 8])
        if mask == "cache":
            c["dir"] = "fwd"
            t = rng.choice([1, 1, 1, 2, 5, 16])
            s = _log(rng, t, max(t, min(65536, pairs // (b * t), 100 * 1000 * 1000 // (b * hk * (2 * dh + dv)))))
        else:
            # (a lone key's gradients are zero but for roundings: nothing to compare)
            s = t = _log(rng, 1 if c["dir"] == "fwd" else 24, min(4096, math.isqrt(pairs // b)))
        c.update(b=b, t=t, s=s, h=h, hk=hk, dh=dh, dv=dv, mask=mask, token_lam=rng.random() < 0.4)
        if c["dir"] == "fwd":
            c["save"] = mask != "cache" and rng.random() < 0.7
    elif kind == "scan":
        d = _log(rng, 64, 8192) // 8 * 8 + rng.choice([0, 0, 0, 0, 4, 1])
        tokens = _log(rng, 1, max(1, min(200000, 33 * 1000 * 1000 // d)))
        b = rng.choice([1, 1, 2, 4, 16])
        sigmoid = rng.random() < 0.7
        c.update(b=b, t=max(1, tokens // b), d=d, sigmoid=sigmoid, mix=rng.random() < (0.7 if sigmoid else 0.3),
                 resets=rng.random() < 0.3)
        if c["dir"] == "fwd":
            c["save"] = rng.random() < 0.5
    else:
        tensors = rng.randint(1, 28)
        c.update(dir="step", tensors=tensors, n=_log(rng, 10 * tensors, 60000000), bits=rng.choice([8, 8, 32]),
                 copies=c["dtype"] == "f32" and rng.random() < 0.5, odd=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case)
    if case["kind"] == "diff":
        b, t, n, h, hk, dh, dv = (case[k] for k in ("b", "t", "s", "h", "hk", "dh", "dv"))
        s["causal"], s["lengths"], s["start"], s["scale"] = case["mask"] in ("causal", "cache"), None, None, dh ** -0.5
        if case["mask"] == "cache":
            # a cache of keys and values; sequences of different lengths, the new tokens at their ends
            s["q"], s["k"], s["v"] = normal(b, t, 2 * h, dh, std=1.5), normal(b, n, 2 * hk, dh), normal(b, n, hk, dv)
            s["lengths"] = torch.randint(max(t, n // 2), n + 1, (b,), generator=g, device="cuda").int()
            s["start"] = s["lengths"] - t
        else:
            # the packed projection and its views
            qkv = normal(b, t, 2 * (h + hk) * dh + hk * dv)
            s["q"] = qkv[..., :2 * h * dh].unflatten(-1, (2 * h, dh))
            s["k"] = qkv[..., 2 * h * dh:2 * (h + hk) * dh].unflatten(-1, (2 * hk, dh))
            s["v"] = qkv[..., 2 * (h + hk) * dh:].unflatten(-1, (hk, dv))
            if case["mask"] == "padded":    # padding at the end of some sequences
                s["lengths"] = torch.randint((n + 3) // 4, n + 1, (b,), generator=g, device="cuda").int()
        shape = (b, t, h) if case["token_lam"] else (h,)
        s["lam"] = torch.rand(shape, generator=g, device="cuda") * 0.6 + 0.2
        if case["dir"] == "bwd":
            s["o"], s["lse"], s["o2"] = _diff_forward(s)   # what the forward kept
            s["do"] = normal(b, t, h, dv)
    elif case["kind"] == "scan":
        b, t, d = (case[k] for k in ("b", "t", "d"))
        # gate and input as the halves of one projection
        p = normal(b, t, 2 * d)
        s["gate"], s["x"] = p[..., :d], p[..., d:]
        if case["sigmoid"]:
            s["gate"].mul_(1.5).add_(3.0)
        else:
            s["gate"].copy_(torch.sigmoid(s["gate"].float() * 1.5 + 3.0))
        s["h0"] = normal(b, d, dtype=torch.float32)
        s["reset"] = torch.rand((b, t), generator=g, device="cuda") < 1 / 500 if case["resets"] else None
        if case["dir"] == "bwd":
            s["states"] = _scan_forward(s)[2]              # what the forward kept
            s["dh"], s["dlast"] = normal(b, t, d), normal(b, d, dtype=torch.float32)
    else:
        k = case["tensors"]
        share = [math.exp(3 * (0.618 * i % 1)) for i in range(k)]    # the largest 20 times the smallest
        sizes = [max(1, int(case["n"] * w / sum(share))) for w in share]
        if not case["odd"]:     # matrices of whole rows
            sizes = [max(1, n // 4096) * 4096 for n in sizes]
        s["p"] = [normal(n, std=0.02) for n in sizes]
        s["g"] = [normal(n, std=0.01) for n in sizes]
        s["copy"] = [p.to(torch.bfloat16) for p in s["p"]] if case["copies"] else None
        s["first"], blocks = [], 0      # the first block of each tensor's moments
        for n in sizes:
            s["first"].append(blocks)
            blocks += -(-n // _BLOCK)
        m = normal(blocks, _BLOCK, std=0.003, dtype=torch.float32)
        v = normal(blocks, _BLOCK, std=0.01, dtype=torch.float32).square_() * 0.5 + 1e-6
        if case["bits"] == 8:
            s["m"], ms = _to8(m)
            s["v"], vs = _to8(v.sqrt())
            s["scale"] = torch.stack((ms, vs), 1)
        else:
            s["m"], s["v"] = m, v
        s["step"], s["lr"], s["wd"] = 12, 1e-3, 0.01
    return s


# ---------------------------------------------------------------- plain forms
def _visible(s):
    """[b, 1, 1, t, s]: whether a query sees a key; None where all do."""
    i = torch.arange(s["t"], device="cuda")[None, :, None]
    j = torch.arange(s["s"], device="cuda")[None, None]
    seen = None
    if s["causal"]:
        seen = j <= (i if s["start"] is None else i + s["start"][:, None, None])
    if s["lengths"] is not None:
        inside = j < s["lengths"][:, None, None]
        seen = inside if seen is None else seen & inside
    return None if seen is None else seen[:, None, None]


def _operands(s):
    """q [b, h, 2, t, dh], k [b, h, 2, s, dh], v [b, h, 1, s, dv], lambda [., h, t, 1] in 32 bits."""
    b, h, hk, t, n = (s[x] for x in ("b", "h", "hk", "t", "s"))
    q = s["q"].float().reshape(b, t, h, 2, s["dh"]).permute(0, 2, 3, 1, 4)
    k = s["k"].float().reshape(b, n, hk, 2, s["dh"]).permute(0, 2, 3, 1, 4).repeat_interleave(h // hk, 1)
    v = s["v"].float().permute(0, 2, 1, 3).repeat_interleave(h // hk, 1)[:, :, None]
    lam = s["lam"].permute(0, 2, 1)[..., None] if s["lam"].dim() == 3 else s["lam"][None, :, None, None]
    return q, k, v, lam


def _diff_forward(s):
    q, k, v, lam = _operands(s)
    z = q @ k.transpose(3, 4) * s["scale"]
    seen = _visible(s)
    if seen is not None:
        z = z.masked_fill_(~seen, -math.inf)
    m = z.amax(4, keepdim=True).clamp_min(-3e38)
    e = torch.exp(z - m)
    total = e.sum(4, keepdim=True)
    lse = (m + torch.log(total))[..., 0].flatten(1, 2)               # [b, 2·h, t]
    o1, o2 = (e / total.clamp_min(1e-38) @ v).unbind(2)             # [b, h, t, dv]
    o = o1 - lam * o2
    dt = s["q"].dtype
    return o.transpose(1, 2).to(dt).contiguous(), lse, o2.transpose(1, 2).to(dt).contiguous()


def _diff_plain(s):
    if s["dir"] == "fwd":
        o, lse, o2 = _diff_forward(s)
        return {"o": o, "lse": lse, "o2": o2} if s["save"] else {"o": o, "lse": lse}
    q, k, v, lam = _operands(s)
    b, h, hk, t, n, dt = (*(s[x] for x in ("b", "h", "hk", "t", "s")), s["q"].dtype)
    do, o, o2 = (s[x].float().transpose(1, 2) for x in ("do", "o", "o2"))
    z = q @ k.transpose(3, 4) * s["scale"]
    seen = _visible(s)
    if seen is not None:
        z = z.masked_fill_(~seen, -math.inf)
    p = torch.exp(z - s["lse"].unflatten(1, (h, 2))[..., None].clamp_min(-3e38))
    p1, p2 = p.unbind(2)
    dp = do @ v[:, :, 0].transpose(2, 3)
    d2 = (do * o2).sum(3, keepdim=True)
    d1 = (do * o).sum(3, keepdim=True) + lam * d2
    dz = torch.stack((p1 * (dp - d1), -lam * p2 * (dp - d2)), 2)
    dq = dz @ k * s["scale"]
    dk = dz.transpose(3, 4) @ q * s["scale"]
    dv = (p1 - lam * p2).transpose(2, 3) @ do
    dlam = -d2[..., 0].transpose(1, 2)
    return {"dq": dq.permute(0, 3, 1, 2, 4).flatten(2, 3).to(dt),
            "dk": dk.unflatten(1, (hk, h // hk)).sum(2).permute(0, 3, 1, 2, 4).flatten(2, 3).to(dt),
            "dv": dv.unflatten(1, (hk, h // hk)).sum(2).transpose(1, 2).to(dt),
            "dlam": dlam.contiguous() if s["lam"].dim() == 3 else dlam.sum((0, 1))}


def _scanned(a, u):
    """y_t = a_t·y_{t−1} + u_t along dim 1 from y_{−1} = 0, by doubling."""
    step = 1
    while step < a.shape[1]:
        u = torch.cat((u[:, :step], u[:, step:] + a[:, step:] * u[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return u


def _gates(s):
    """The gate, what multiplies the state, and what multiplies the input."""
    a = s["gate"].float()
    if s["sigmoid"]:
        a = torch.sigmoid(a)
    keep = a if s["reset"] is None else torch.where(s["reset"][..., None], 0.0, a)
    return a, keep, (torch.sigmoid(-s["gate"].float()) if s["sigmoid"] else 1 - a) if s["mix"] else None


def _scan_states(s):
    """All states [b, t + 1, d], the initial one first."""
    _, keep, take = _gates(s)
    u = s["x"].float() if take is None else take * s["x"].float()
    u = torch.cat((s["h0"][:, None], u), 1)
    return _scanned(torch.cat((torch.zeros_like(keep[:, :1]), keep), 1), u)


def _scan_forward(s):
    y = _scan_states(s)
    return y[:, 1:].to(s["x"].dtype), y[:, -1], y[:, :-1:_CHUNK].contiguous()


def _scan_plain(s):
    if s["dir"] == "fwd":
        h, last, states = _scan_forward(s)
        return {"h": h, "last": last, "states": states} if s["save"] else {"h": h, "last": last}
    a, keep, take = _gates(s)
    before, x = _scan_states(s)[:, :-1], s["x"].float()
    dh = torch.cat((s["dh"].float()[:, :-1], (s["dh"][:, -1].float() + s["dlast"])[:, None]), 1)
    later = torch.cat((keep[:, 1:], torch.zeros_like(keep[:, :1])), 1)
    e = _scanned(later.flip(1), dh.flip(1)).flip(1)          # the gradient of every state
    da = e * before if s["reset"] is None else torch.where(s["reset"][..., None], 0.0, e * before)
    if s["mix"]:
        da = da - e * x
    if s["sigmoid"]:
        da = da * a * torch.sigmoid(-s["gate"].float())
    dx = e if take is None else e * take
    return {"dx": dx.to(s["x"].dtype), "dgate": da.to(s["x"].dtype), "dh0": e[:, 0] * keep[:, 0]}


def _to8(y):
    """Blocks [., 256] as e4m3 values and their scales."""
    scale = y.abs().amax(1) / _E4M3
    inverse = torch.where(scale > 0, 1 / scale, 0.0)[:, None]
    return (y * inverse).clamp(-_E4M3, _E4M3).to(torch.float8_e4m3fn), scale


def _blocks(tensors):
    """The tensors as rows of 256, each beginning a row of its own, zeros behind its end."""
    return torch.cat([torch.nn.functional.pad(t.float(), (0, -t.numel() % _BLOCK)) for t in tensors]).view(-1, _BLOCK)


def _adam_plain(s):
    p, g = _blocks(s["p"]), _blocks(s["g"])
    if s["bits"] == 8:
        m = s["m"].float() * s["scale"][:, :1]
        r = s["v"].float() * s["scale"][:, 1:]
        v = r * r
    else:
        m, v = s["m"], s["v"]
    c1, c2 = 1 - 0.9 ** s["step"], 1 - 0.999 ** s["step"]
    p = p * (1 - s["lr"] * s["wd"])
    m = m * 0.9 + g * (1 - 0.9)
    v = v * 0.999 + g * g * (1 - 0.999)
    r = torch.sqrt(v)
    p = p + m * (-s["lr"] / c1) / (r / math.sqrt(c2) + 1e-8)
    if s["bits"] == 8:
        q, ms = _to8(m)
        w, vs = _to8(r)
        w = torch.where(r > 0, w.float().clamp_min(2.0 ** -9), 0.0).to(w.dtype)   # a root above zero stays above zero
        s["m"].copy_(q)
        s["v"].copy_(w)
        s["scale"].copy_(torch.stack((ms, vs), 1))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    flat, dt = p.view(-1), _DT[s["dtype"]]
    new = [flat[f * _BLOCK:f * _BLOCK + t.numel()].to(dt) for f, t in zip(s["first"], s["p"])]
    torch._foreach_copy_(s["p"], new)
    if s["copy"] is not None:
        torch._foreach_copy_(s["copy"], new)


def _adam_outputs(s):
    """The step's results, which lie in the state's own buffers."""
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["bits"] == 8:
        out["scale"] = s["scale"]
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    return out


# ----------------------------------------------------------------------- run
def _own(s):
    from thot_amd import ops
    if s["kind"] == "diff":
        kw = dict(causal=s["causal"], scale=s["scale"], lengths=s["lengths"], q_start=s["start"])
        if s["dir"] == "fwd":
            o, lse, o2 = ops.diff_attention_fwd(s["q"], s["k"], s["v"], s["lam"], save=s["save"], **kw)
            return {"o": o, "lse": lse, "o2": o2} if s["save"] else {"o": o, "lse": lse}
        dq, dk, dv, dlam = ops.diff_attention_bwd(s["do"], s["q"], s["k"], s["v"], s["lam"], s["o"], s["o2"], s["lse"], **kw)
        return {"dq": dq, "dk": dk, "dv": dv, "dlam": dlam}
    if s["kind"] == "scan":
        kw = dict(sigmoid=s["sigmoid"], mix=s["mix"], reset=s["reset"])
        if s["dir"] == "fwd":
            h, last, states = ops.linear_scan_fwd(s["x"], s["gate"], s["h0"], save=s["save"], **kw)
            return {"h": h, "last": last, "states": states} if s["save"] else {"h": h, "last": last}
        dx, dgate, dh0 = ops.linear_scan_bwd(s["dh"], s["x"], s["gate"], s["states"], dlast=s["dlast"], **kw)
        return {"dx": dx, "dgate": dgate, "dh0": dh0}
    if "moments" not in s:      # the optimizer that a program keeps beside its parameters
        s["moments"] = ops.AdamMoments(s["p"], bits=s["bits"], copies=s["copy"], m=s["m"], v=s["v"], scale=s.get("scale"))
    ops.adam_multi_step(s["moments"], s["g"], lr=s["lr"], weight_decay=s["wd"], step=s["step"])
    return _adam_outputs(s)


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "adam":
        _adam_plain(state)
        return _adam_outputs(state)
    return (_diff_plain if state["kind"] == "diff" else _scan_plain)(state)


# ---------------------------------------------------------------------- work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    fwd = case["dir"] == "fwd"
    if case["kind"] == "diff":
        b, t, n, h, hk, dh, dv = (case[k] for k in ("b", "t", "s", "h", "hk", "dh", "dv"))
        keys = n * 3 // 4 if case["mask"] == "cache" else (5 * n + 7) // 8 if case["mask"] == "padded" else n
        pairs = b * h * (t * (t + 1) // 2 if case["mask"] == "causal" else t * keys)
        q, k, v, o = b * t * 2 * h * dh * e, b * keys * 2 * hk * dh * e, b * keys * hk * dv * e, b * t * h * dv * e
        lam = 4 * (b * t * h if case["token_lam"] else h)
        if fwd:
            return {"bytes": q + k + v + o * (2 if case["save"] else 1) + 8 * b * h * t + lam, "flops": pairs * (4 * dh + 4 * dv)}
        return {"bytes": 2 * (q + k + v) + 3 * o + 8 * b * h * t + 2 * lam, "flops": pairs * (12 * dh + 4 * dv)}
    if case["kind"] == "scan":
        n, rows = case["b"] * case["t"] * case["d"], case["b"] * case["d"]
        kept = 4 * rows * -(-case["t"] // _CHUNK)
        mask = case["b"] * case["t"] if case["resets"] else 0
        if fwd:
            return {"bytes": 3 * n * e + 8 * rows + mask + (kept if case["save"] else 0), "flops": 8 * n}
        return {"bytes": 5 * n * e + 8 * rows + mask + kept, "flops": 20 * n}
    n = case["n"]
    state = 2 + 8 / _BLOCK if case["bits"] == 8 else 8
    return {"bytes": n * (3 * e + 2 * state + (2 if case["copies"] else 0)), "flops": 16 * n}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    dbl = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() and "8" not in str(v.dtype) else v
           for k, v in s.items()}
    if case["kind"] == "diff":
        return _exact_diff(case, dbl)
    if case["kind"] == "scan":
        return _exact_scan(case, dbl)
    # the moments before they are rounded to 8 bits stand for what is held
    out = {"p": [], "copy": []}
    first = s["first"] + [s["m"].shape[0]]
    ms, vs, scales = [], [], []
    for i, (p, g) in enumerate(zip(s["p"], s["g"])):
        n, rows = p.numel(), slice(first[i], first[i + 1])
        m, v = s["m"][rows].double(), s["v"][rows].double()
        if case["bits"] == 8:
            m, v = m * s["scale"][rows, :1].double(), (v * s["scale"][rows, 1:].double()) ** 2
        whole = torch.zeros(m.numel(), dtype=torch.float64, device="cuda")
        whole[:n] = g.double()
        whole = whole.view_as(m)
        m.lerp_(whole, 0.1)
        v.lerp_(whole * whole, 0.001)
        denom = (v / (1 - 0.999 ** 12)).sqrt() + 1e-8
        new = p.double() * (1 - 1e-5) - 1e-3 * (m / (1 - 0.9 ** 12) / denom).flatten()[:n]
        out["p"].append(new)
        out["copy"].append(new)
        if case["bits"] == 8:
            v = v.sqrt()
            sc = torch.stack((m.abs().amax(1), v.amax(1)), 1) / 448
            scales.append(sc)
            m, v = m / sc[:, :1], v / sc[:, 1:]
        ms.append(m)
        vs.append(v)
    out["m"], out["v"] = torch.cat(ms), torch.cat(vs)
    if case["bits"] == 8:
        out["scale"] = torch.cat(scales)
    if not case["copies"]:
        del out["copy"]
    return out


def _exact_diff(case, s):
    b, t, n, h, hk, dh = (case[x] for x in ("b", "t", "s", "h", "hk", "dh"))
    parts, back = [], case["dir"] == "bwd"
    length = s["lengths"].tolist() if s["lengths"] is not None else [n] * b
    start = s["start"].tolist() if s["start"] is not None else [0] * b
    sums = {"dk": torch.zeros_like(s["k"]), "dv": torch.zeros_like(s["v"])}
    for i in range(b):
        for c in range(h):      # one head of one sequence at a time
            j, end = c // (h // hk), length[i]
            lam = s["lam"][i, :, c] if case["token_lam"] else s["lam"][c].expand(t)
            val, maps = s["v"][i, :end, j], []
            for r in (0, 1):
                z = s["q"][i, :, 2 * c + r] @ s["k"][i, :end, 2 * j + r].t() * s["scale"]
                if s["causal"]:
                    z += torch.full_like(z, -math.inf).triu(start[i] + 1)
                maps.append(z)
            if not back:
                lse = torch.stack([z.logsumexp(1) for z in maps])
                o1, o2 = ((z - l[:, None]).exp() @ val for z, l in zip(maps, lse))
                parts.append((o1 - lam[:, None] * o2, lse, o2))
                continue
            do, d = s["do"][i, :, c], []
            p1, p2 = ((z - s["lse"][i, 2 * c + r][:, None]).exp() for r, z in enumerate(maps))
            second = torch.einsum("td,td->t", do, s["o2"][i, :, c])
            first = torch.einsum("td,td->t", do, s["o"][i, :, c]) + lam * second
            w = do @ val.t()
            for r, (p, y) in enumerate(((p1, w - first[:, None]), (p2, (second[:, None] - w) * lam[:, None]))):
                ds = p * y * s["scale"]
                d.append(ds @ s["k"][i, :end, 2 * j + r])
                sums["dk"][i, :end, 2 * j + r] += ds.t() @ s["q"][i, :, 2 * c + r]
            sums["dv"][i, :end, j] += (p1 - p2 * lam[:, None]).t() @ do
            parts.append((torch.stack(d), -second))
    if not back:
        out = {"o": torch.stack([p[0] for p in parts]).unflatten(0, (b, h)).transpose(1, 2),
               "lse": torch.cat([p[1] for p in parts]).unflatten(0, (b, 2 * h))}
        return dict(out, o2=torch.stack([p[2] for p in parts]).unflatten(0, (b, h)).transpose(1, 2)) if case["save"] else out
    dq = torch.cat([p[0] for p in parts]).unflatten(0, (b, 2 * h)).transpose(1, 2)
    dlam = torch.stack([p[1] for p in parts]).unflatten(0, (b, h)).transpose(1, 2)
    return {"dq": dq, "dk": sums["dk"], "dv": sums["dv"], "dlam": dlam if case["token_lam"] else dlam.sum((0, 1))}


def _exact_scan(case, s):
    if case["t"] > 100000 or case["t"] * case["b"] * case["d"] > 40000000:
        return None
    back = case["dir"] == "bwd"
    gate, x = s["gate"], s["x"]
    a = 1 / (1 + torch.exp(-gate)) if case["sigmoid"] else gate
    took = (1 / (1 + torch.exp(gate)) if case["sigmoid"] else 1 - gate) if case["mix"] else torch.ones_like(gate)
    keep = a * ~s["reset"][..., None] if case["resets"] else a
    h, before, after = s["h0"], [], []
    for i in range(case["t"]):
        before.append(h)
        h = keep[:, i] * h + took[:, i] * x[:, i]
        after.append(h)
    if not back:
        out = {"h": torch.stack(after, 1), "last": h}
        return dict(out, states=torch.stack(before[::_CHUNK], 1)) if case["save"] else out
    e, dx, dg = s["dlast"], [], []
    for i in reversed(range(case["t"])):
        e = e + s["dh"][:, i]
        dx.append(e * took[:, i])
        d = e * before[i] * (1.0 if not case["resets"] else ~s["reset"][:, i, None])
        d = d - e * x[:, i] if case["mix"] else d
        dg.append(d * a[:, i] * (1 - a[:, i]) if case["sigmoid"] else d)
        e = e * keep[:, i]
    return {"dx": torch.stack(dx[::-1], 1), "dgate": torch.stack(dg[::-1], 1), "dh0": e}
