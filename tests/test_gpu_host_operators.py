"""The host layer's differentiable functions on inputs of any strides, outputs that a
loss leaves out, and parameters that cannot have a gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def host():
    from thot_amd import _nott_host
    return _nott_host


def rnd(*s, dt=torch.float32):
    return torch.randn(s, device="cuda").to(dt)


@pytest.mark.parametrize("dt", DT)
def test_gradient_of_a_view(host, dt):
    """x as a transposed or sliced view: the gradient of the contiguous copy, laid back."""
    dt = DT[dt]
    d, f = 32, 24
    w = rnd(2 * f, d).requires_grad_()
    wc = w.detach().to(dt)
    wl = rnd(f, d).requires_grad_()
    gamma, beta = rnd(d).requires_grad_(), rnd(d).requires_grad_()
    calls = {"gated": lambda x: host.gated_linear(x, w, None, wc), "linear": lambda x: host.linear(x, wl, None, wl.detach().to(dt)),
             "norm": lambda x: host.layer_norm(x, gamma, beta, gamma.detach().to(dt), beta.detach().to(dt))}
    for name, call in calls.items():
        for base, view in ((rnd(d, 10, dt=dt), lambda t: t.t()), (rnd(10, 2 * d, dt=dt), lambda t: t[:, d:])):
            a, b = base.clone().requires_grad_(), base.clone().requires_grad_()
            y = call(view(a))
            dy = torch.randn_like(y)
            y.backward(dy)
            call(view(b).contiguous()).backward(dy)
            torch.cuda.synchronize()
            assert a.grad is not None, name
            assert torch.equal(a.grad, b.grad), name
