"""What adam_multi_step refuses before anything reaches a device."""
import pytest
import torch

from thot_amd import ops


def moments(p, **kw):
    return ops.AdamMoments(p, **kw)


def test_parameters():
    for bad, match in (([], "empty"), ([torch.zeros(3)], "device tensor")):
        with pytest.raises(ValueError, match=match):
            moments(bad)
    with pytest.raises(ValueError, match="8 or 32"):
        moments([torch.zeros(3)], bits=16)
    with pytest.raises(ValueError, match="2 copies for 1"):
        moments([torch.zeros(3)], copies=[None, None])
    with pytest.raises(TypeError):
        moments([torch.zeros(3, dtype=torch.float16)])
