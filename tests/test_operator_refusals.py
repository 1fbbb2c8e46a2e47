"""Arguments that the language-model operators refuse, before anything reaches a
device: the checks of thot_amd.ops and of the host layer on host tensors."""
import pytest
import torch

from thot_amd import ops


@pytest.fixture(scope="module")
def host():
    return pytest.importorskip("thot_amd._nott_host")


def heads(b=2, t=3, h=4, dh=8, dtype=torch.float32):
    return torch.zeros((b, t, h, dh), dtype=dtype)


def rope(**kw):
    a = dict(q=heads(), k=heads(h=2), positions=torch.zeros((2, 3), dtype=torch.int64),
             inv_freq=torch.ones(4, dtype=torch.float64))
    a.update(kw)
    return ops.qk_norm_rope_fwd(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 3, 8)), "b, t, heads, dh"),
    (dict(q=heads(dh=520), k=None), "1 to 512"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(norm=False, gamma_q=torch.ones(8)), "weight needs the norm"),
    (dict(inv_freq=torch.ones(5, dtype=torch.float64)), "at most the head size"),
    (dict(inv_freq=torch.ones((2, 2), dtype=torch.float64)), "inv_freq must be"),
    (dict(positions=None), "needs positions"),
    (dict(inv_freq=None), "need inv_freq"),
    (dict(positions=torch.zeros((3, 2), dtype=torch.int64)), "positions must be"),
    (dict(positions=torch.zeros((5, 2, 3), dtype=torch.int64), sections=[1, 1, 1, 1, 0]), "positions must be"),
    (dict(positions=torch.zeros((2, 2, 3), dtype=torch.int64)), "sections must be 2"),
    (dict(positions=torch.zeros((2, 2, 3), dtype=torch.int64), sections=[3, 2]), "add up to 4"),
    (dict(positions=torch.zeros((2, 2, 3), dtype=torch.int64), sections=[5, -1]), "add up to 4"),
    (dict(k=heads(t=4, h=2)), "k has shape"),
    (dict(k=heads(h=2, dh=16)[..., ::2]), "contiguous"),
    (dict(q=torch.zeros(8).expand(2, 3, 4, 8)), "repeats one head"),
    (dict(), "device tensor"),
])
def test_rope(kw, match):
    with pytest.raises(ValueError, match=match):
        rope(**kw)


def test_rope_types():
    with pytest.raises(TypeError):
        rope(q=heads(dtype=torch.float16), k=None)
    with pytest.raises(TypeError, match="dtype and device of q"):
        rope(k=heads(h=2, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.rope_frequencies(7)
    f = ops.rope_frequencies(8, 100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, 100.0 ** -(torch.arange(4, dtype=torch.float64) / 4))


def test_outputs_that_overlap_themselves():
    for t in (torch.zeros(2, 1, 4, 8).expand(2, 3, 4, 8), torch.zeros(100).as_strided((2, 3, 4, 8), (8, 16, 4, 1))):
        with pytest.raises(ValueError, match="overlaps itself"):
            ops._check_out(t, "out")
    ops._check_out(torch.zeros(2, 4, 3, 8).transpose(1, 2), "out")
    ops._check_out(torch.zeros(2, 3, 64)[..., 32:].unflatten(-1, (4, 8)), "out")
    ops._check_out(torch.zeros(0, 3, 4, 8), "out")


@pytest.mark.parametrize("x,w,act,match", [
    ((3, 8), (10, 8), "tanh", "unknown activation"),
    ((3, 8), (9, 8), "silu", "gate rows"),
    ((3, 8), (10, 7), "silu", "gate rows"),
    ((3, 8), (0, 8), "silu", "gate rows"),
    ((3, 8), (10,), "silu", "gate rows"),
    ((3, 8), (10, 8), "silu", "device tensor"),
])
def test_gated(x, w, act, match):
    with pytest.raises(ValueError, match=match):
        ops.gated_linear_fwd(torch.zeros(x), torch.zeros(w), act=act)


def test_accumulation_without_gradients():
    x, w, gu = torch.zeros(3, 8), torch.zeros(10, 8), torch.zeros(3, 10)
    with pytest.raises(ValueError, match="accumulate needs"):
        ops.gated_linear_bwd(torch.zeros(3, 5), x, w, gu, need_db=False, accumulate=True)
    with pytest.raises(ValueError, match="accumulate needs"):
        ops.gated_linear_bwd(torch.zeros(3, 5), x, w, gu, dw=w, accumulate=True)


def test_gated_types():
    with pytest.raises(TypeError):
        ops.gated_linear_fwd(torch.zeros((3, 8), dtype=torch.float16), torch.zeros((10, 8), dtype=torch.float16))


@pytest.mark.parametrize("n,kw,match", [
    (4, dict(), "labels has shape"),
    (3, dict(scale=0.0), "scale"),
    (3, dict(scale=float("inf")), "scale"),
    (3, dict(scale=float("nan")), "scale"),
    (3, dict(top=6), "top must be"),
    (3, dict(top=-1), "top must be"),
    (3, dict(), "device tensor"),
])
def test_logprob(n, kw, match):
    with pytest.raises(ValueError, match=match):
        ops.token_logprob_fwd(torch.zeros(3, 5), torch.zeros(n, dtype=torch.int64), **kw)


def test_logprob_shapes():
    y = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="c > 0"):
        ops.token_logprob_fwd(torch.zeros(3, 0), y)
    with pytest.raises(ValueError, match="top must be"):
        ops.token_logprob_fwd(torch.zeros(3, 100), y, top=65)
    one = torch.zeros(3)
    with pytest.raises(ValueError, match="needs entropy"):
        ops.token_logprob_bwd(torch.zeros(3, 5), y, one, one, dentropy=one)


@pytest.mark.parametrize("kw,match", [
    (dict(w=torch.zeros(0, 8)), "weight must be"),
    (dict(x=torch.zeros(3, 0), w=torch.zeros(4, 0)), "weight must be"),
    (dict(w=torch.zeros(8, 4).t()), "weight must be"),
    (dict(w=torch.zeros(6, 8), w_compute=torch.zeros(4, 8)), "working copy"),
    (dict(b=torch.zeros(3)), "bias must be"),
    (dict(b=torch.zeros(8)[::2]), "bias must be"),
    (dict(b=torch.zeros(4, dtype=torch.float64)), "bias must be"),
    (dict(), "HIP device"),
])
def test_host_gated_linear(host, kw, match):
    a = dict(x=torch.zeros(3, 8), w=torch.zeros(4, 8))
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        host.gated_linear(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(gamma_q=torch.ones(7)), "weight must be"),
    (dict(gamma_k=torch.ones(16)[::2]), "weight must be"),
    (dict(gamma_q=torch.ones(6), gamma_q_compute=torch.ones(8)), "weight must be"),
    (dict(k=torch.zeros(2, 3, 4, 8, dtype=torch.bfloat16)), "q's type"),
    (dict(), "HIP device"),
])
def test_host_qk_norm_rope(host, kw, match):
    q = torch.zeros(2, 3, 4, 8)
    a = dict(q=q, k=q)
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        host.qk_norm_rope(**a)
