"""The initial state of the host layer's linear recurrence is an input like the others: its
gradient is asked for by torch.autograd.grad, passes its hooks, and is left in .grad."""
import pytest
import torch

from thot_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [0, 1, 300])
def test_gradient_of_an_initial_state(t):
    from thot_amd import _nott_host as host
    x, gate, dh = (torch.randn(2, t, 40, device="cuda") for _ in range(3))
    h0, dlast = torch.randn(2, 40, device="cuda").requires_grad_(), torch.randn(2, 40, device="cuda")
    _, _, states = ops.linear_scan_fwd(x, gate, h0.detach(), save=True)
    want = ops.linear_scan_bwd(dh, x, gate, states, dlast=dlast)[2]
    h, last = host.linear_scan(x, gate, h0)
    got, = torch.autograd.grad((h, last), (h0,), (dh, dlast), retain_graph=True)
    assert torch.equal(got, want) and h0.grad is None
    seen = []
    h0.register_hook(lambda g: seen.append(g.clone()) or 2 * g)
    torch.autograd.backward((h, last), (dh, dlast), retain_graph=True)
    torch.autograd.backward((h, last), (dh, dlast))
    torch.cuda.synchronize()
    assert len(seen) == 2 and all(torch.equal(g, want) for g in seen) and torch.equal(h0.grad, 4 * want)
