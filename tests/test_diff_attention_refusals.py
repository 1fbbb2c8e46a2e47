"""What differential attention refuses before anything reaches a device."""
import pytest
import torch

from thot_amd import ops


def call(**kw):
    a = dict(q=torch.zeros(2, 3, 8, 16), k=torch.zeros(2, 5, 4, 16), v=torch.zeros(2, 5, 2, 32), lam=torch.zeros(4))
    a.update(kw)
    return ops.diff_attention_fwd(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("lam"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(3, 8, 16)), "must be"),
    (dict(q=torch.zeros(2, 3, 7, 16)), "two for each head"),
    (dict(q=torch.zeros(2, 3, 6, 16)), "whole groups"),
    (dict(q=torch.zeros(2, 3, 8, 72), k=torch.zeros(2, 5, 4, 72)), "head size"),
    (dict(v=torch.zeros(2, 5, 2, 129)), "head size"),
    (dict(k=torch.zeros(2, 6, 4, 16)), "k must be"),
    (dict(k=torch.zeros(2, 5, 2, 16)), "k must be"),
    (dict(k=torch.zeros(2, 5, 4, 32)[..., ::2]), "contiguous"),
    (dict(q=torch.zeros(16).expand(2, 3, 8, 16)), "repeats one row"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(), "device tensor"),
])
def test_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


def test_types():
    with pytest.raises(TypeError):
        call(q=torch.zeros(2, 3, 8, 16, dtype=torch.float16))
    with pytest.raises(TypeError, match="dtype and device of q"):
        call(k=torch.zeros(2, 5, 4, 16, dtype=torch.bfloat16))
