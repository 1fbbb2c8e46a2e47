"""qk_norm_rope without the norm: elements past the rotated ones are copied, bit for
bit and whatever they hold, on every path (chunks, odd sizes, both pairings)."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def special(shape, dt, lo, seed):
    """Normal values with infinities, NaN and the type's largest from element lo of each head on."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    what = torch.randint(0, 8, shape, generator=g, device="cuda")
    for i, v in enumerate((float("inf"), -float("inf"), float("nan"), torch.finfo(dt).max)):
        x[..., lo:] = torch.where(what[..., lo:] == i, v, x[..., lo:])
    return x.to(dt)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0, 7, -7), b.nan_to_num(0, 7, -7))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dh,rot", [(64, 0), (64, 32), (64, 36), (80, 60), (33, 14), (128, 2), (512, 256), (7, 0), (40, 40)])
def test_unrotated_elements(dh, rot, inter, dt):
    dt = DT[dt]
    b, t, hq, hk = 2, 21, 3, 1
    q, k = special((b, t, hq, dh), dt, rot, 1), special((b, t, hk, dh), dt, rot, 2)
    pos = torch.arange(b * t, device="cuda").view(b, t) + 5 if rot else None
    freq = ops.rope_frequencies(rot) if rot else None
    clean = [torch.cat((x[..., :rot], torch.ones_like(x[..., rot:])), -1) for x in (q, k)]
    for run in (lambda a, c: ops.qk_norm_rope_fwd(a, c, pos, freq, norm=False, interleaved=inter),
                lambda a, c: ops.qk_norm_rope_bwd(a, c, a, c, pos, freq, norm=False, interleaved=inter)[:2]):
        got, want = run(q, k), run(*clean)
        torch.cuda.synchronize()
        for y, w, x in zip(got, want, (q, k)):
            assert same(y[..., rot:], x[..., rot:])
            assert torch.equal(y[..., :rot], w[..., :rot])      # what is rotated sees none of them
