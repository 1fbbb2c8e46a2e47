"""Gates that are not finite before a token that forgets (a reset, or a keep of exactly 0):
nothing of them reaches what follows, forward or backward, wherever the two lie in a span of
tokens, in a tile of 256 and in a segment of time."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("d", [64, 37])
@pytest.mark.parametrize("at", [1, 2, 3, 5, 17, 100, 255, 256, 300, 1000])
@pytest.mark.parametrize("how", ["reset", "zero"])
def test_what_follows_is_clean(dt, d, at, how):
    """The tokens from `at` on: bit for bit as with finite gates before them."""
    dt = DT[dt]
    b, t = 2, 3000
    g = torch.Generator(device="cuda").manual_seed(at)
    x, gate, dh = ((torch.rand(b, t, d, generator=g, device="cuda") * 0.8 + 0.1).to(dt) for _ in range(3))
    dlast = torch.rand(b, d, generator=g, device="cuda")
    reset = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    if how == "reset":
        reset[:, at] = True
    else:
        gate[:, at] = 0

    def run(gate, x):
        h, last, states = ops.linear_scan_fwd(x, gate, sigmoid=False, mix=False, reset=reset if how == "reset" else None, save=True)
        dx, dgate, _ = ops.linear_scan_bwd(dh, x, gate, states, sigmoid=False, mix=False, dlast=dlast,
                                           reset=reset if how == "reset" else None)
        torch.cuda.synchronize()
        # (where the gate itself is 0, its gradient takes the state before it)
        return h[:, at:], last, dx[:, at:], dgate[:, at + 1:]
    want = run(gate, x)
    for bad in (math.nan, math.inf, -math.inf):
        for back in (1, 2, 9):
            if at >= back:
                gg = gate.clone()
                gg[:, at - back] = bad
                for name, a, w in zip(("h", "last", "dx", "dgate"), run(gg, x), want):
                    assert torch.equal(a, w), (name, bad, back)
    xx = x.clone()
    xx[:, at - 1] = math.nan
    for name, a, w in zip(("h", "last", "dx", "dgate"), run(gate, xx), want):
        assert torch.equal(a, w), name


@pytest.mark.parametrize("at", [1, 5, 256, 1000])
def test_what_comes_before_is_clean(at):
    """Backward, gradients and gates that are not finite behind the token that forgets."""
    b, t, d = 2, 3000, 64
    g = torch.Generator(device="cuda").manual_seed(at)
    x, gate, dh = (torch.rand(b, t, d, generator=g, device="cuda") * 0.8 + 0.1 for _ in range(3))
    reset = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    reset[:, at] = True

    def run(gate, dh):
        h, _, states = ops.linear_scan_fwd(x, gate, sigmoid=False, mix=False, reset=reset, save=True)
        dx, dgate, dh0 = ops.linear_scan_bwd(dh, x, gate, states, sigmoid=False, mix=False, reset=reset)
        torch.cuda.synchronize()
        return h[:, :at], dx[:, :at], dgate[:, :at], dh0
    want = run(gate, dh)
    for bad in (math.nan, math.inf):
        for ahead in (0, 1, 9):
            gg, dd = gate.clone(), dh.clone()
            gg[:, at + ahead] = bad
            dd[:, at + ahead] = bad
            for args in ((gg, dh), (gate, dd)):
                for name, a, w in zip(("h", "dx", "dgate", "dh0"), run(*args), want):
                    assert torch.equal(a, w), (name, bad, ahead)
