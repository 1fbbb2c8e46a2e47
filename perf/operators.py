"""The language-model operators whose speed is followed, with their plain forms.

Three operators, each forward and backward:

``rope``     queries and keys between the packed projection and attention: the
             root-mean-square norm of every head, its weight, and the rotation
             by the token's position (one position, or several axes).
``gated``    a gated feed-forward layer: gate and up projection of one packed
             weight, the activation and the product.
``logprob``  the log probability of each row's given token, the entropy of the
             row and its most likely tokens.

``run`` computes them with elementary torch operations, or, where ``own`` is
true, with this library's calls.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One new token of each of 8 sequences, far into a long text: launches
        # and latency are all there is.
        {"name": "rope_step_bf16", "kind": "rope", "dir": "fwd", "dtype": "bf16", "b": 8, "t": 1, "hq": 32, "hk": 8,
         "dh": 128, "rot": 128, "axes": 1, "interleaved": False, "start": 100000},
        # The benchmark's attention (8 x 1024 tokens, 16 heads of 64), queries and
        # keys as the packed projection leaves them.
        {"name": "rope_bf16", "kind": "rope", "dir": "fwd", "dtype": "bf16", "b": 8, "t": 1024, "hq": 16, "hk": 16,
         "dh": 64, "rot": 64, "axes": 1, "interleaved": False, "start": 0},
        # The backward pass of long sequences with shared key heads.
        {"name": "rope_bwd_bf16", "kind": "rope", "dir": "bwd", "dtype": "bf16", "b": 4, "t": 4096, "hq": 32, "hk": 8,
         "dh": 128, "rot": 128, "axes": 1, "interleaved": False, "start": 0},
        # Frames of a video: positions in time, height and width, an odd number
        # of tokens, neighbouring elements as pairs, only part of the head rotated.
        {"name": "rope_video_bwd_f32", "kind": "rope", "dir": "bwd", "dtype": "f32", "b": 3, "t": 1577, "hq": 12,
         "hk": 12, "dh": 80, "rot": 60, "axes": 3, "interleaved": True, "start": 0},
        # One token of each of 8 sequences: the weights are read once for 8 rows.
        {"name": "gated_step_bf16", "kind": "gated", "dir": "fwd", "dtype": "bf16", "m": 8, "d": 1024, "f": 4096,
         "act": "silu", "bias": False, "save": False},
        # A training batch of 8 x 1024 tokens, pre-activations kept for the backward.
        {"name": "gated_bf16", "kind": "gated", "dir": "fwd", "dtype": "bf16", "m": 8192, "d": 1024, "f": 4096,
         "act": "silu", "bias": False, "save": True},
        # The same batch's backward pass.
        {"name": "gated_bwd_bf16", "kind": "gated", "dir": "bwd", "dtype": "bf16", "m": 8192, "d": 1024, "f": 4096,
         "act": "silu", "bias": False},
        # 8 sequences of 197 tokens, widths that end inside tiles, biases.
        {"name": "gated_ragged_bwd_bf16", "kind": "gated", "dir": "bwd", "dtype": "bf16", "m": 1576, "d": 760,
         "f": 2024, "act": "gelu_tanh", "bias": True},
        # The same layer's forward in fp32, the framework's default type.
        {"name": "gated_ragged_f32", "kind": "gated", "dir": "fwd", "dtype": "f32", "m": 1576, "d": 768, "f": 2048,
         "act": "gelu", "bias": True, "save": True},
        # The answers of one decoding step of 8 sequences: a few long rows.
        {"name": "logprob_step_bf16", "kind": "logprob", "dir": "fwd", "dtype": "bf16", "n": 8, "c": 128256, "top": 8,
         "scale": 1.25, "masked": 256},
        # A scored training batch, the benchmark's logits.
        {"name": "logprob_bf16", "kind": "logprob", "dir": "fwd", "dtype": "bf16", "n": 16384, "c": 32000, "top": 5,
         "scale": 1.0, "masked": 0},
        # Its gradient in fp32, rows that are not 16-byte aligned, with an
        # entropy term.
        {"name": "logprob_bwd_f32", "kind": "logprob", "dir": "bwd", "dtype": "f32", "n": 4096, "c": 50257,
         "scale": 1.0, "masked": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "gated", "logprob"])
    c = {"kind": kind, "dir": rng.choice(["fwd", "bwd"]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "rope":
        dh = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 160, 256])
        axes = rng.choice([1, 1, 1, 2, 3])
        rot = rng.choice([dh, dh, dh // 2, 2 * rng.randint(max(axes, dh // 8), dh // 2)])
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 1, 2, 3, 4])
        tokens = _log(rng, 1, max(1, min(32768, 80 * 1000 * 1000 // ((hq + hk) * dh))))
        b = rng.choice([1, 2, 3, 8])
        c.update(b=b, t=max(1, tokens // b), hq=hq, hk=hk, dh=dh, rot=rot, axes=axes,
                 interleaved=rng.random() < 0.3, start=rng.choice([0, 0, 5000, 120000]))
    elif kind == "gated":
        step = rng.choice([1, 8, 8, 64])
        d, f = (max(step, _log(rng, 64, hi) // step * step) for hi in (2048, 4096))
        most = 8192 * 1024 * 4096 // (4 if c["dtype"] == "f32" else 2)
        c.update(m=_log(rng, 1, max(1, min(8192, most // (d * f)))), d=d, f=f,
                 act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"]), bias=rng.random() < 0.4)
        if c["dir"] == "fwd":
            c["save"] = rng.random() < 0.5
    else:
        v = _log(rng, 64, 160000)
        c.update(n=_log(rng, 1, max(1, min(16384, 200 * 1000 * 1000 // v))), c=v, scale=rng.choice([1.0, 1.0, 0.7, 1.6]),
                 masked=rng.choice([0, 0, v // 50]))
        if c["dir"] == "fwd":
            c["top"] = rng.choice([0, 1, 5, 20])
    return c


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case)
    if case["kind"] == "rope":
        b, t, hq, hk, dh, rot = (case[k] for k in ("b", "t", "hq", "hk", "dh", "rot"))
        # the packed projection [b, t, (hq + 2·hk)·dh] and its views
        qkv = normal(b, t, (hq + 2 * hk) * dh)
        s["q"] = qkv[..., :hq * dh].unflatten(-1, (hq, dh))
        s["k"] = qkv[..., hq * dh:(hq + hk) * dh].unflatten(-1, (hk, dh))
        s["gamma_q"], s["gamma_k"] = ((1 + normal(dh, std=0.1, dtype=torch.float32)).to(dt) for _ in range(2))
        s["inv_freq"] = 10000.0 ** (-2.0 / rot * torch.arange(rot // 2, dtype=torch.float64, device="cuda"))
        first = torch.randint(0, case["start"] + 1, (b, 1), generator=g, device="cuda")
        tok = torch.arange(t, device="cuda")[None]
        if case["axes"] == 1:
            s["positions"] = (first + tok)[None]
        else:   # frames of 14 x 14 patches
            s["positions"] = torch.stack([first + tok // 196, (tok // 14 % 14).expand(b, t),
                                          (tok % 14).expand(b, t)][:case["axes"]])
        s["positions"] = s["positions"].contiguous()
        pairs, axes = rot // 2, case["axes"]
        s["sections"] = [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)
        s["axis"] = torch.arange(axes, device="cuda").repeat_interleave(torch.tensor(s["sections"], device="cuda"))
        if case["dir"] == "bwd":
            s["doq"], s["dok"] = normal(b, t, hq, dh), normal(b, t, hk, dh)
    elif case["kind"] == "gated":
        m, d, f = case["m"], case["d"], case["f"]
        s["x"] = normal(m, d)
        s["w"] = normal(2 * f, d, std=d ** -0.5)
        s["bias_"] = normal(2 * f, std=0.2, dtype=torch.float32) if case["bias"] else None
        if case["dir"] == "bwd":
            gu = s["x"].float() @ s["w"].float().t()
            s["gu"] = (gu if s["bias_"] is None else gu + s["bias_"]).to(dt)
            s["dh"] = normal(m, f, std=0.05)
    else:
        n, c = case["n"], case["c"]
        z = torch.randn((n, c), generator=g, device="cuda").mul_(2.5)
        s["labels"] = torch.randint(0, c - case["masked"], (n,), generator=g, device="cuda")
        z[torch.arange(n, device="cuda"), s["labels"]] += 4.0
        if case["masked"]:   # the padding of a vocabulary
            z[:, c - case["masked"]:] = -math.inf
        s["logits"] = z.to(dt)
        s["labels"][torch.rand(n, generator=g, device="cuda") < 0.1] = -100
        if case["dir"] == "bwd":
            lse, ent = [], []
            for r in s["logits"].split(max(1, 50000000 // c)):   # what the forward kept
                lp = (r.double() * case["scale"])
                lse.append(lp.logsumexp(1))
                lp -= lse[-1][:, None]
                ent.append(-torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1))
            s["lse"], s["entropy"] = torch.cat(lse).float(), torch.cat(ent).float()
            s["dlogprob"] = normal(n, dtype=torch.float32) / n
            s["dentropy"] = normal(n, dtype=torch.float32) * (0.1 / n)
    return s


# ---------------------------------------------------------------- plain forms
def _rotation(s):
    """cos and sin [b, t, 1, rot/2] of every token's angles, formed in 64 bits."""
    angle = s["positions"].double()[s["axis"]].movedim(0, -1) * s["inv_freq"]
    return angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]


def _pairs(s, x):
    r = x[..., :s["rot"]]
    if s["interleaved"]:
        return r[..., 0::2], r[..., 1::2]
    return r.chunk(2, -1)


def _unpairs(s, a, b, x):
    r = torch.stack((a, b), -1).flatten(-2) if s["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((r, x[..., s["rot"]:]), -1)


_EPS = 1e-6


def _rope_plain(s):
    cos, sin = _rotation(s)
    out = {}
    for n in "qk":
        x, gamma = s[n].float(), s["gamma_" + n].float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        xh = x * rstd
        if s["dir"] == "fwd":
            z = xh * gamma
            a, b = _pairs(s, z)
            out[n] = _unpairs(s, a * cos - b * sin, a * sin + b * cos, z).to(s[n].dtype)
        else:
            dy = s["do" + n].float()
            a, b = _pairs(s, dy)
            dz = _unpairs(s, a * cos + b * sin, b * cos - a * sin, dy)
            dzg = dz * gamma
            out["d" + n] = (rstd * (dzg - xh * (dzg * xh).mean(-1, keepdim=True))).to(s[n].dtype)
            out["dgamma_" + n] = (dz * xh).sum((0, 1, 2))
    return out


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        e = torch.sigmoid(g)
        return g * e, e * (1 + g * (1 - e))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-g * 0.5 ** 0.5)
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        k = (2 / math.pi) ** 0.5
        e = torch.sigmoid(2 * k * (g + 0.044715 * g ** 3))
        return g * e, e + g * e * (1 - e) * 2 * k * (1 + 3 * 0.044715 * g * g)
    if name == "sigmoid":
        e = torch.sigmoid(g)
        return e, e * (1 - e)
    return g.clamp_min(0), (g > 0).to(g.dtype)


def _gated_plain(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    if s["dir"] == "fwd":
        gu = x @ w.t()
        if s["bias_"] is not None:
            gu = gu + s["bias_"]
        g, u = gu.chunk(2, -1)
        out = {"h": (_act(s["act"], g)[0] * u).to(dt)}
        if s["save"]:
            out["gu"] = gu.to(dt)
        return out
    g, u = s["gu"].float().chunk(2, -1)
    a, da = _act(s["act"], g)
    dh = s["dh"].float()
    dgu = torch.cat((dh * u * da, dh * a), -1)
    out = {"dx": (dgu @ w).to(dt), "dw": dgu.t() @ x}
    if s["bias"]:
        out["db"] = dgu.sum(0)
    return out


def _top(z, k):
    """Columns of the k largest values of each row, equal ones lowest first: 64-bit
    keys of the value (in an order that whole numbers keep) and the column."""
    i = (z + 0.0).view(torch.int32).long()
    i = torch.where(i < 0, -(i & 0x7fffffff) - 1, i)
    key = i * (1 << 32) + (0xffffffff - torch.arange(z.shape[1], device="cuda"))
    return 0xffffffff - (key.topk(k, 1).values & 0xffffffff)


def _logprob_plain(s):
    z, y = s["logits"].float() * s["scale"], s["labels"]
    given = y != -100
    at = torch.where(given, y, 0)[:, None]
    if s["dir"] == "fwd":
        m = z.max(1, keepdim=True).values
        e = torch.exp(z - m)
        total = e.sum(1, keepdim=True)
        logt = torch.log(total)
        out = {"logprob": torch.where(given, (z.gather(1, at) - m - logt)[:, 0], 0.0),
               "lse": (m + logt)[:, 0],
               "entropy": (logt - torch.where(e > 0, e * (z - m), 0.0).sum(1, keepdim=True) / total)[:, 0]}
        if s["top"]:
            idx = _top(s["logits"].float(), s["top"])
            out["top_logprob"], out["top_index"] = z.gather(1, idx) - m - logt, idx
        return out
    lp = z - s["lse"][:, None]
    p = torch.exp(lp)
    dlp = torch.where(given, s["dlogprob"], 0.0)[:, None]
    d = -p * (dlp + s["dentropy"][:, None] * (torch.where(p > 0, lp, 0.0) + s["entropy"][:, None]))
    d.scatter_add_(1, at, dlp)
    return {"dlogits": (d * s["scale"]).to(s["logits"].dtype)}


# ----------------------------------------------------------------------- run
def _own(s):
    from thot_amd import ops
    if s["kind"] == "rope":
        kw = dict(eps=_EPS, sections=s["sections"], interleaved=s["interleaved"])
        if s["dir"] == "fwd":
            q, k = ops.qk_norm_rope_fwd(s["q"], s["k"], s["positions"], s["inv_freq"], s["gamma_q"], s["gamma_k"], **kw)
            return {"q": q, "k": k}
        dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(s["doq"], s["dok"], s["q"], s["k"], s["positions"], s["inv_freq"],
                                                s["gamma_q"], s["gamma_k"], **kw)
        return {"dq": dq, "dk": dk, "dgamma_q": dgq, "dgamma_k": dgk}
    if s["kind"] == "gated":
        if s["dir"] == "fwd":
            h, gu = ops.gated_linear_fwd(s["x"], s["w"], s["bias_"], act=s["act"], save=s["save"])
            return {"h": h, "gu": gu} if s["save"] else {"h": h}
        dx, dw, db = ops.gated_linear_bwd(s["dh"], s["x"], s["w"], s["gu"], act=s["act"], need_db=s["bias"])
        return {"dx": dx, "dw": dw, "db": db} if s["bias"] else {"dx": dx, "dw": dw}
    if s["dir"] == "fwd":
        lp, ent, lse, top, idx = ops.token_logprob_fwd(s["logits"], s["labels"], scale=s["scale"], top=s["top"])
        out = {"logprob": lp, "lse": lse, "entropy": ent}
        return dict(out, top_logprob=top, top_index=idx) if s["top"] else out
    return {"dlogits": ops.token_logprob_bwd(s["logits"], s["labels"], s["lse"], s["dlogprob"], entropy=s["entropy"],
                                             dentropy=s["dentropy"], scale=s["scale"])}


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope_plain, "gated": _gated_plain, "logprob": _logprob_plain}[state["kind"]](state)


# ---------------------------------------------------------------------- work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    fwd = case["dir"] == "fwd"
    if case["kind"] == "rope":
        tokens, heads, dh = case["b"] * case["t"], case["hq"] + case["hk"], case["dh"]
        n = tokens * heads * dh
        return {"bytes": n * e * (2 if fwd else 3) + 8 * case["axes"] * tokens + 2 * dh * e + (0 if fwd else 8 * dh),
                "flops": n * (8 if fwd else 18)}
    if case["kind"] == "gated":
        m, d, f = case["m"], case["d"], case["f"]
        b = 8 * f if case["bias"] else 0
        if fwd:
            return {"bytes": e * (m * d + 2 * f * d + m * f * (3 if case["save"] else 1)) + b, "flops": 4 * m * d * f}
        return {"bytes": e * (3 * m * f + 2 * m * d + 2 * f * d) + 8 * f * d + b, "flops": 8 * m * d * f}
    n, c = case["n"], case["c"]
    if fwd:
        return {"bytes": n * c * e + n * (8 + 12 + 12 * case["top"]), "flops": 6 * n * c}
    return {"bytes": 2 * n * c * e + n * (8 + 16), "flops": 8 * n * c}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        out, half = {}, case["rot"] // 2
        first = [sum(s["sections"][:a]) for a in range(case["axes"])]
        turn = torch.empty((case["b"], case["t"], 1, half), dtype=torch.complex128, device="cuda")
        for a, n in enumerate(s["sections"]):
            th = s["positions"][a].double()[..., None, None] * s["inv_freq"][first[a]:first[a] + n]
            turn[..., first[a]:first[a] + n] = torch.polar(torch.ones_like(th), th)
        idx = torch.arange(case["rot"], device="cuda")
        re, im = (idx[0::2], idx[1::2]) if case["interleaved"] else (idx[:half], idx[half:])

        def rotated(v, by):
            v = v.clone()
            w = torch.complex(v[..., re], v[..., im]) * by
            v[..., re], v[..., im] = w.real, w.imag
            return v

        for n in "qk":
            x, gam = s[n].double(), s["gamma_" + n].double()
            rms = (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            if case["dir"] == "fwd":
                out[n] = rotated(x / rms * gam, turn)
            else:
                dz = rotated(s["do" + n].double(), turn.conj())
                dot = (dz * gam * x).mean(-1, keepdim=True)
                out["d" + n] = dz * gam / rms - x * dot / rms ** 3
                out["dgamma_" + n] = (dz * x / rms).flatten(0, 2).sum(0)
        return out
    if case["kind"] == "gated":
        x, w = s["x"].double(), s["w"].double()
        f = case["f"]
        if case["dir"] == "fwd":
            gu = x @ w.t() + (0 if s["bias_"] is None else s["bias_"].double())
        else:
            gu = s["gu"].double()
        g = gu[:, :f].clone().requires_grad_(case["dir"] == "bwd")
        u = gu[:, f:].clone().requires_grad_(case["dir"] == "bwd")
        F = torch.nn.functional
        a = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "relu": F.relu,
             "sigmoid": torch.sigmoid}[case["act"]](g)
        h = a * u
        if case["dir"] == "fwd":
            return {"h": h, "gu": gu} if case["save"] else {"h": h}
        d = torch.cat(torch.autograd.grad(h, (g, u), s["dh"].double()), 1)
        out = {"dx": d @ w, "dw": d.t() @ x}
        return dict(out, db=d.sum(0)) if case["bias"] else out
    parts = []
    rows = max(1, 40000000 // case["c"])
    for r in range(0, case["n"], rows):
        z = s["logits"][r:r + rows].double() * case["scale"]
        y = s["labels"][r:r + rows]
        ok = y >= 0
        lp = torch.log_softmax(z, 1)
        p = lp.exp()
        plogp = torch.where(p > 0, p * lp, 0.0)
        hit = lp.gather(1, y.clamp_min(0)[:, None])[:, 0]
        if case["dir"] == "fwd":
            q = {"logprob": torch.where(ok, hit, 0.0), "lse": z.logsumexp(1), "entropy": -plogp.sum(1)}
            if case["top"]:
                best = s["logits"][r:r + rows].double().sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
                q["top_logprob"], q["top_index"] = lp.gather(1, best), best
        else:
            dl = torch.where(ok, s["dlogprob"][r:r + rows].double(), 0.0)[:, None]
            dh = s["dentropy"][r:r + rows].double()[:, None]
            d = -dl * p - dh * (plogp - p * plogp.sum(1, keepdim=True))
            d[torch.arange(len(y), device="cuda"), y.clamp_min(0)] += dl[:, 0]
            q = {"dlogits": d * case["scale"]}
        parts.append(q)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
