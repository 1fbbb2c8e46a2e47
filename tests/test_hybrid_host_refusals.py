"""Arguments that the host layer's differential attention, linear recurrence and optimizer
over many tensors refuse, on host tensors: nothing reaches a device."""
import pytest
import torch


@pytest.fixture(scope="module")
def host():
    return pytest.importorskip("thot_amd._nott_host")


def z(*s, dt=torch.float32):
    return torch.zeros(s, dtype=dt)


I32 = torch.int32


@pytest.mark.parametrize("kw", [
    dict(q=z(2, 3, 4)), dict(q=z(2, 3, 3, 8)), dict(q=z(2, 3, 6, 8)), dict(q=z(2, 3, 4, 0)), dict(k=z(2, 5, 4)),
    dict(k=z(1, 5, 4, 8)), dict(k=z(2, 6, 4, 8)), dict(k=z(2, 5, 2, 8)), dict(k=z(2, 5, 4, 9)), dict(v=z(2, 5, 0, 8)),
    dict(v=z(2, 5, 2, 8, dt=torch.bfloat16)), dict(k=z(2, 5, 4, 8, dt=torch.bfloat16)), dict(lam=z(3)), dict(lam=z(2, 2)),
    dict(lam=z(2, 5, 2)), dict(lam=z(2, dt=torch.float64)), dict(lam=z(2, dt=torch.bfloat16)), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(lengths=z(3, dt=I32)), dict(lengths=z(2, dt=torch.int64)),
    dict(lengths=z(2, 1, dt=I32)), dict(q_start=z(4, dt=I32)[::2]), dict(q_start=z(2))])
def test_diff_attention(host, kw):
    a = dict(q=z(2, 3, 4, 8), k=z(2, 5, 4, 8), v=z(2, 5, 2, 8), lam=z(2))
    with pytest.raises(ValueError, match="HIP device"):     # the good call gets as far as the device
        host.diff_attention(**a)
    a.update(kw)
    with pytest.raises(ValueError) as e:
        host.diff_attention(**a)
    assert "HIP device" not in str(e.value)


@pytest.mark.parametrize("kw", [
    dict(x=z(2, 8)), dict(x=z(2, 3, 0), gate=z(2, 3, 0)), dict(gate=z(2, 4, 8)), dict(gate=z(2, 3, 8, dt=torch.bfloat16)),
    dict(h0=z(8)), dict(h0=z(3, 8)), dict(h0=z(2, 8, dt=torch.bfloat16)), dict(reset=z(2, 3)), dict(reset=z(2, 4, dt=torch.bool)),
    dict(reset=z(3, 2, dt=torch.bool).t()), dict(reset=z(6, dt=torch.uint8))])
def test_linear_scan(host, kw):
    a = dict(x=z(2, 3, 8), gate=z(2, 3, 8), h0=z(2, 8), reset=z(2, 3, dt=torch.bool))
    with pytest.raises(ValueError, match="HIP device"):
        host.linear_scan(**a)
    a.update(kw)
    with pytest.raises(ValueError) as e:
        host.linear_scan(**a)
    assert "HIP device" not in str(e.value)


def test_optimizer(host):
    p = z(4).requires_grad_()
    for cls in (host.MultiTensorAdam, host.MultiTensorAdamW):
        with pytest.raises(ValueError, match="bits"):
            cls([[p]], [1e-3], [0.0], bits=16)
        with pytest.raises(ValueError, match="HIP device"):
            cls([[p]], [1e-3], [0.0])
        with pytest.raises(ValueError, match="per group"):
            cls([[p]], [1e-3], [])
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            cls([[z(4, dt=torch.float64).requires_grad_()]], [1e-3], [0.0])
