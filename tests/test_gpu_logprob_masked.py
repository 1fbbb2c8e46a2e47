"""token_logprob of rows in which nearly all tokens are masked (constrained decoding), at
the sizes of a vocabulary: the live tokens first, then masked ones from the lowest
column on, with log probability −inf.

Tolerance: at most 64 half steps of fp32 (2^-24) of |z − m| and log of the live count."""
import math

import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,c,live,top", [(2, 128256, 3, 8), (3, 128256, 0, 20), (260, 50257, 3, 20), (1, 300001, 70, 64),
                                          (1100, 32000, 1, 5), (40, 1500, 3, 64), (2100, 4000, 30, 64)])
def test_few_live_tokens(n, c, live, top, dt):
    g = torch.Generator(device="cuda").manual_seed(c + top)
    z = torch.full((n, c), -math.inf, device="cuda")
    z[1::2] = torch.finfo(dt).min      # the other way to mask: equal, so lowest column first as well
    at = torch.rand((n, c), generator=g, device="cuda").topk(max(live, 1), 1).indices
    if live:
        z.scatter_(1, at, torch.randn((n, live), generator=g, device="cuda") * 3)
    z = z.to(dt)
    y = at[:, 0].contiguous()
    lp, ent, lse, tv, ti = ops.token_logprob_fwd(z, y, top=top)
    torch.cuda.synchronize()
    want = z.float().sort(dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti, want)
    if live == 0:
        assert bool((lse == -math.inf).all()) and bool((ent == 0).all()) and bool((lp == -math.inf).all())
        assert bool((tv == -math.inf).all())
        return
    v = z.gather(1, at).double()
    ref = v - v.logsumexp(1, keepdim=True)
    tol = 64 * U * (ref.abs().amax() + math.log(live) + 1)
    assert float((lp.double() - ref[:, 0]).abs().amax()) <= tol
    k = min(live, top)
    assert float((tv[:, :k].double() - ref.sort(1, descending=True).values[:, :k]).abs().amax()) <= tol
    assert bool((tv[:, k:] == -math.inf).all())
