"""The optimizer over many tensors and the bf16 copies that it hands out: a copy whose storage
was replaced is refused by the step, before anything is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [lambda c: torch.zeros(3, dtype=c.dtype, device="cuda"), lambda c: c.t(),
                                   lambda c: torch.zeros(c.shape, dtype=torch.float16, device="cuda")])
@pytest.mark.parametrize("bits", [8, 32])
def test_replaced_copy(other, bits):
    from thot_amd import _nott_host as host
    ps = [torch.randn(30, 30, device="cuda").requires_grad_() for _ in range(2)]
    opt = host.MultiTensorAdamW([ps], [1e-2], [0.0], bits=bits)
    for p in ps:
        p.grad = torch.randn_like(p)
    copy = opt.bf16_copy(ps[1])
    opt.step()
    assert torch.equal(copy, ps[1].detach().bfloat16())
    before = [p.detach().clone() for p in ps]
    copy.data = other(copy.data)
    with pytest.raises(RuntimeError, match="copy has changed"):
        opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p.detach(), b) for p, b in zip(ps, before)) and opt.state_step(ps[0]) == 1
    copy.data = torch.zeros(30, 30, dtype=torch.bfloat16, device="cuda")
    opt.step()
    assert torch.equal(copy, ps[1].detach().bfloat16())
