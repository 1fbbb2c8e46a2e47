"""Keys split in an odd number of parts for an odd number of rows with odd value widths: what
is kept of a part beside its output begins where 16-byte reads may."""
import pytest
import torch

from test_gpu_diff_attention import DT, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("t,s,dv", [(1, 700, 41), (3, 700, 33), (1, 1200, 7), (5, 1200, 63)])
def test_odd_everything(dt, t, s, dv):
    q, k, v, lam = make(1, t, s, 1, 1, 20, dv, DT[dt], seed=dv)
    check(q, k, v, lam, backward=False)
    check(q, k, v, lam, causal=True, start=torch.tensor([s - t], dtype=torch.int32, device="cuda"), backward=False)
