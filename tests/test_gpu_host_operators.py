"""The host layer's differentiable functions on inputs of any strides, outputs that a
loss leaves out, and parameters that cannot have a gradient."""
import pytest
import torch

from thot_amd import ops

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


@pytest.mark.parametrize("dt", DT)
def test_log_probability_alone(host, dt):
    """A loss of one output: the gradient of ops without the other."""
    dt = DT[dt]
    z = rnd(6, 300, dt=dt).requires_grad_()
    y = torch.tensor([0, 299, 7, -100, 3, 3], device="cuda")
    f = ops.token_logprob_fwd(z.detach(), y, scale=0.7)
    d = rnd(6)
    lp, ent = host.token_logprob(z, y, 0.7)
    lp.backward(d)
    assert torch.equal(z.grad, ops.token_logprob_bwd(z.detach(), y, f[2], d, scale=0.7))
    z.grad = None
    lp, ent = host.token_logprob(z, y, 0.7)
    ent.backward(d)
    assert torch.equal(z.grad, ops.token_logprob_bwd(z.detach(), y, f[2], torch.zeros_like(d), entropy=f[1], dentropy=d,
                                                     scale=0.7))
    z.grad = None
    lp, ent = host.token_logprob(z, y, 0.7)
    torch.autograd.backward((lp, ent), (d, 2 * d))
    assert torch.equal(z.grad, ops.token_logprob_bwd(z.detach(), y, f[2], d, entropy=f[1], dentropy=2 * d, scale=0.7))


def test_output_left_out_costs_nothing(host):
    """A loss of the log probability alone allocates the logits' gradient and nothing for the entropy's."""
    z = rnd(6, 300).requires_grad_()
    y = torch.zeros(6, dtype=torch.int64, device="cuda")
    d = rnd(6)

    def allocated(use):
        z.grad = None
        lp, ent = host.token_logprob(z, y)
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        torch.autograd.backward((lp, ent)[:use], (d, d)[:use])
        return torch.cuda.memory_stats()["allocation.all.allocated"] - before
    allocated(1)
    assert allocated(1) == allocated(2) == 1


def test_one_of_two_heads_used(host):
    """A loss of queries or keys alone, and of neither's whole: absent gradients count as zeros."""
    q, k = (rnd(2, 9, 4, 16).requires_grad_() for _ in range(2))
    pos = torch.arange(18, device="cuda").view(1, 2, 9)
    freq = ops.rope_frequencies(16)
    gq, gk = rnd(16).requires_grad_(), rnd(16).requires_grad_()
    yq, yk = host.qk_norm_rope(q, k, pos, freq, gq, gk)
    g = torch.randn_like(yk)
    yk.backward(g)
    torch.cuda.synchronize()
    want = ops.qk_norm_rope_bwd(torch.zeros_like(q), g.transpose(1, 2), q.detach(), k.detach(), pos, freq, gq.detach(),
                                gk.detach())
    assert torch.equal(k.grad, want[1]) and torch.equal(gk.grad, want[3])
    assert torch.count_nonzero(q.grad).item() == 0 and torch.count_nonzero(gq.grad).item() == 0
