"""Arguments that the host layer's language-model functions refuse in the forward, on
host tensors: parameters whose gradient could not be written, and positions that
nothing would use."""
import pytest
import torch


@pytest.fixture(scope="module")
def host():
    return pytest.importorskip("thot_amd._nott_host")


def bf16(*s):
    return torch.ones(s, dtype=torch.bfloat16)


def test_trained_gated_weight_that_is_not_fp32(host):
    x = bf16(3, 8)
    with pytest.raises(ValueError, match="fp32"):
        host.gated_linear(x, bf16(4, 8).requires_grad_())
    with pytest.raises(ValueError, match="fp32"):
        host.gated_linear(x, torch.ones(4, 8, dtype=torch.float64).requires_grad_(), None, bf16(4, 8))
    for w in (bf16(4, 8), torch.ones(4, 8).requires_grad_()):    # these get as far as the device
        with pytest.raises(ValueError, match="HIP device"):
            host.gated_linear(x, w, None, bf16(4, 8))


@pytest.mark.parametrize("which", ["gamma_q", "gamma_k"])
def test_trained_head_weight_that_is_not_fp32(host, which):
    q = bf16(1, 2, 3, 8)
    with pytest.raises(ValueError, match="fp32"):
        host.qk_norm_rope(q, q, **{which: bf16(8).requires_grad_()})
    with pytest.raises(ValueError, match="HIP device"):
        host.qk_norm_rope(q, q, **{which: bf16(8)})
    with pytest.raises(ValueError, match="HIP device"):
        host.qk_norm_rope(q, q, **{which: torch.ones(8).requires_grad_(), which + "_compute": bf16(8)})


@pytest.mark.parametrize("kw", [dict(positions=torch.zeros(1, 1, 2, dtype=torch.int64)), dict(sections=[4])])
def test_positions_that_nothing_uses(host, kw):
    q = torch.ones(1, 2, 3, 8)
    with pytest.raises(ValueError, match="inv_freq"):
        host.qk_norm_rope(q, q, **kw)


def test_no_rotated_elements(host):
    """Empty frequencies are frequencies: the call gets as far as the device."""
    q = torch.ones(1, 2, 3, 8)
    with pytest.raises(ValueError, match="HIP device"):
        host.qk_norm_rope(q, q, torch.zeros(1, 1, 2, dtype=torch.int64), torch.ones(0, dtype=torch.float64))
