"""What linear_scan refuses before anything reaches a device."""
import pytest
import torch

from thot_amd import ops


def scan(**kw):
    a = dict(x=torch.zeros(2, 3, 8), gate=torch.zeros(2, 3, 8))
    a.update(kw)
    return ops.linear_scan_fwd(a.pop("x"), a.pop("gate"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(x=torch.zeros(3, 8)), "b, t, d"),
    (dict(x=torch.zeros(2, 3, 0), gate=torch.zeros(2, 3, 0)), "d > 0"),
    (dict(gate=torch.zeros(2, 4, 8)), "gate must be"),
    (dict(gate=torch.zeros(2, 3, 16)[..., ::2]), "contiguous"),
    (dict(x=torch.zeros(8).expand(2, 3, 8)), "repeats one token"),
    (dict(), "device tensor"),
])
def test_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        scan(**kw)


def test_types():
    with pytest.raises(TypeError):
        scan(x=torch.zeros(2, 3, 8, dtype=torch.float16), gate=torch.zeros(2, 3, 8, dtype=torch.float16))
    with pytest.raises(TypeError, match="dtype and device of x"):
        scan(gate=torch.zeros(2, 3, 8, dtype=torch.bfloat16))
