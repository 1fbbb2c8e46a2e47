"""AdamMoments when its tensors get other storage between steps: checked again before
anything reaches the kernel (here on host tensors, with the device's part of the checks
left out)."""
import pytest
import torch

from thot_amd import ops

N = 300


@pytest.fixture
def moments(monkeypatch):
    check = ops._check

    def without_device(t, name, **kw):
        if t.device.type != "cpu":
            raise ValueError(f"{name} is on {t.device}")
        monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
        try:
            check(t, name, **kw)
        finally:
            monkeypatch.delattr(torch.Tensor, "is_cuda", raising=False)
    monkeypatch.setattr(ops, "_check", without_device)

    def make(bits=8, copies=True):
        p = [torch.zeros(20, 20), torch.zeros(N), torch.zeros(N, dtype=torch.bfloat16)]
        c = [torch.zeros(t.shape, dtype=torch.bfloat16) for t in p] if copies else None
        return ops.AdamMoments(p, bits=bits, copies=c)
    return make


def grads(m):
    return [torch.ones(shape) for _, shape in m._meta]


def words(m, g=None):
    w, n = m._tensors(g or grads(m))
    return [list(w[8 * i:8 * i + 8]) for i in range(n)]


@pytest.mark.parametrize("bits", [8, 32])
def test_addresses_follow(moments, bits):
    """New storage of the same shape and type is where the step goes."""
    m = moments(bits)
    assert [w[0] for w in words(m)] == [p.data_ptr() for p in m.params]
    m.params[1].data = torch.ones(N)
    m.copies[0] = torch.ones(20, 20, dtype=torch.bfloat16)
    m.copies[2] = None
    m.m = torch.ones_like(m.m.float()).to(m.m.dtype)
    m.v = m.v.clone()
    if bits == 8:
        m.scale = m.scale.clone()
    size = 256 * bits // 8
    for i, w in enumerate(words(m)):
        assert w[0] == m.params[i].data_ptr() and w[5] == (0 if m.copies[i] is None else m.copies[i].data_ptr())
        assert w[2] == m.m.data_ptr() + size * m.first[i] and w[3] == m.v.data_ptr() + size * m.first[i]
        assert w[4] == (m.scale.data_ptr() + 8 * m.first[i] if bits == 8 else 0)
    assert torch.equal(m.exp_avg(1), torch.ones(N) * (m.scale[0, 0] if bits == 8 else 1))


def narrower(t):
    return torch.zeros(t.shape[0] - 1, t.shape[1], dtype=t.dtype)


@pytest.mark.parametrize("change", [
    lambda m: setattr(m.params[0], "data", torch.zeros(20, 20).t()),
    lambda m: setattr(m.params[0], "data", m.params[0].data.t()),
    lambda m: setattr(m.params[1], "data", torch.zeros(2 * N)[::2]),
    lambda m: setattr(m.params[1], "data", torch.zeros(N - 1)),
    lambda m: setattr(m.params[1], "data", torch.zeros(N, dtype=torch.float16)),
    lambda m: setattr(m.params[1], "data", m.params[1].data.view(torch.int32)),
    lambda m: m.params.__setitem__(1, torch.zeros(N, device="meta")),
    lambda m: setattr(m.params[1], "data", m.params[0].data.view(-1)[:N]),
    lambda m: m.params.__setitem__(1, torch.zeros(N - 1)),
    lambda m: setattr(m.copies[1], "data", torch.zeros(N - 1, dtype=torch.bfloat16)),
    lambda m: setattr(m.copies[1], "data", torch.zeros(N, dtype=torch.float32)),
    lambda m: setattr(m.copies[1], "data", m.copies[1].data.view(torch.int16)),
    lambda m: setattr(m.copies[0], "data", m.copies[0].data.t()),
    lambda m: setattr(m.copies[1], "data", m.params[2].data),
    lambda m: m.copies.__setitem__(1, torch.zeros(N, device="meta", dtype=torch.bfloat16)),
    lambda m: setattr(m, "m", narrower(m.m)),
    lambda m: setattr(m, "v", m.v.view(torch.uint8)),
    lambda m: setattr(m, "v", torch.zeros(m.v.shape)),
    lambda m: setattr(m, "scale", torch.zeros(m.scale.shape[::-1]).t()),
    lambda m: setattr(m, "scale", narrower(m.scale)),
    lambda m: setattr(m, "scale", torch.zeros(m.scale.numel() + 2)[2:].view(m.scale.shape)),
])
def test_what_does_not_fit_is_refused(moments, change):
    m = moments()
    words(m)
    change(m)
    for _ in range(2):      # (and again at the next step)
        with pytest.raises((ValueError, TypeError)):
            words(m)


def test_a_parameter_without_a_gradient_may_be_anything(moments):
    m = moments()
    m.params[1].data = torch.zeros(3)
    g = grads(m)
    g[1] = None
    assert len(words(m, g)) == 2
    with pytest.raises(ValueError):
        words(m)
    m.params[1].data = torch.zeros(N)
    assert words(m)[1][0] == m.params[1].data_ptr()
