"""Scales of token_logprob at the ends of their range: 1e-30 to 1e30, so that fp32
holds them."""
import ctypes as C
import math

import pytest
import torch

from thot_amd import ops
from thot_amd._abi import NottInvalidArgument


@pytest.mark.parametrize("scale", [1e-31, 1e-40, 1e-50, 5e-324, 1e30])
def test_refused(scale):
    z, y, one = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(ValueError, match="scale"):
        ops.token_logprob_fwd(z, y, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.token_logprob_bwd(z, y, one, one, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-31, 1e-50, 1e30])
def test_refused_at_the_entry_points(scale):
    buf = torch.zeros(4096, device="cuda").data_ptr()
    ctx = ops.context()
    with pytest.raises(NottInvalidArgument, match="scale"):
        ctx.call("nott_token_logprob_fwd", 0, 3, 5, buf, buf, C.c_double(scale), 0, buf, None, None, None, None)
    with pytest.raises(NottInvalidArgument, match="scale"):
        ctx.call("nott_token_logprob_bwd", 0, 3, 5, buf, buf, C.c_double(scale), buf, None, buf, None, buf)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_least_scale(dt):
    """Live tokens are all as likely, masked ones have none, and one 3e30 above the rest leads them by e^3."""
    c = 300
    z = torch.randn(2, c, device="cuda").to(dt)
    z[:, ::3] = -math.inf
    z[1, 4] = 3e30
    y = torch.tensor([1, 4], device="cuda")
    lp, ent, _, _, ti = ops.token_logprob_fwd(z, y, scale=1e-30, top=1)
    torch.cuda.synchronize()
    live = c - c // 3
    d = float(z[1, 4]) * float(torch.tensor(1e-30, dtype=torch.float32))
    s = math.exp(-d) * (live - 1) + 1
    # 64 half steps of fp32 and c/256 additions, as at any scale
    tol = 66 * 2.0 ** -24
    assert abs(float(lp[0]) + math.log(live)) <= tol * 6 and abs(float(ent[0]) - math.log(live)) <= tol * 6
    assert abs(float(lp[1]) + math.log(s)) <= tol * 6 and int(ti[1, 0]) == 4
