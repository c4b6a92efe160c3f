"""rope under autograd: the gradient is the inverse rotation of the output's,
bit for bit, and by differences what the definition in 64 bits says."""
import numpy as np
import pytest

from test_gpu_rope import close, plain, table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def problem(torch, dtype, seed=0, n=9, h=3, d=40, rot=24, axes=2):
    rng = np.random.default_rng(seed)
    freq, axis, dfreq, daxis = table(torch, rot, axes, seed)
    pos = rng.integers(0, 30000, (n, axes)).astype(np.int32)
    x, w = (torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).cuda().to(dtype) for _ in range(2))
    return x, w, pos, torch.from_numpy(pos).cuda(), freq, axis, dfreq, daxis


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_backward_is_the_rotation_back(mb, torch, inverse, interleaved, dtype):
    x, w, pos, dpos, freq, axis, dfreq, daxis = problem(torch, getattr(torch, dtype))
    how = dict(interleaved=interleaved, inverse=inverse)
    without = mb.rope(x, dpos, dfreq, daxis, **how)
    assert not without.requires_grad
    leaf = x.clone().requires_grad_()
    y = mb.rope(leaf, dpos, dfreq, daxis, **how)
    assert y.requires_grad and torch.equal(y, without)
    y.backward(w)
    back = mb.rope(w, dpos, dfreq, daxis, interleaved=interleaved, inverse=not inverse)
    assert leaf.grad.dtype is x.dtype and torch.equal(leaf.grad, back)
    want, norm = plain(w.double().cpu().numpy(), pos, freq, axis, interleaved, not inverse)
    close(leaf.grad.double().cpu().numpy(), want, norm, dtype)


def test_through_other_operators(mb, torch):
    """A slice of a projection, whose gradient comes back through rope; a sum's gradient, whose strides are 0; without
    recording; and a second derivative (of a quadratic form: the rotation of the rotation back, so the vector itself)."""
    x, w, pos, dpos, freq, axis, dfreq, daxis = problem(torch, torch.float32)
    n, h, d = x.shape
    weight = torch.randn(16, 2 * h * d, device="cuda").requires_grad_()
    base = torch.randn(n, 16, device="cuda")
    part = (base @ weight).unflatten(1, (2 * h, d))[:, h:]              # strided
    mb.rope(part, dpos, dfreq, daxis).backward(w)
    back = mb.rope(w, dpos, dfreq, daxis, inverse=True)
    whole = torch.zeros(n, 2 * h, d, device="cuda")
    whole[:, h:] = back
    # one product of at most 9 terms in fp32
    torch.testing.assert_close(weight.grad, base.T @ whole.flatten(1), rtol=1e-5, atol=1e-5)

    leaf = x.clone().requires_grad_()
    mb.rope(leaf, dpos, dfreq, daxis).sum().backward()
    assert torch.equal(leaf.grad, mb.rope(torch.ones_like(x), dpos, dfreq, daxis, inverse=True))

    with torch.no_grad():
        assert not mb.rope(leaf, dpos, dfreq, daxis).requires_grad
        out = torch.empty_like(x)
        assert mb.rope(leaf, dpos, dfreq, daxis, out=out) is out

    leaf = x.clone().requires_grad_()
    y = mb.rope(leaf, dpos, dfreq, daxis)
    first, = torch.autograd.grad((y * y).sum() / 2, leaf, create_graph=True)
    second, = torch.autograd.grad((first * w).sum(), leaf)
    # the identity, turned there and back: two rotations of fp32, 6 units of 2^-24 of the pair's norm each
    norm = torch.from_numpy(plain(w.double().cpu().numpy(), pos, freq, axis, False)[1]).cuda()
    limit = 14 * 2.0 ** -24 * torch.maximum(norm, w.abs().double())
    assert ((second.double() - w.double()).abs() <= limit).all()


def test_gradient_by_differences(mb, torch):
    """<w, rope(x)> of the operator itself, by central differences of step 1 (the rotation is linear): each side's error is
    at most 6 units of 2^-24 of a pair's norm for every value it sums, of norms below 2 * 4.5 + 1."""
    x, w, pos, dpos, freq, axis, dfreq, daxis = problem(torch, torch.float32, n=2, h=1, d=10, rot=8)
    leaf = x.clone().requires_grad_()
    (mb.rope(leaf, dpos, dfreq, daxis) * w).sum().backward()
    for k in range(x.numel()):
        e = torch.zeros(x.numel(), device="cuda")
        e[k] = 1.0
        up, down = (mb.rope(x + s * e.view_as(x), dpos, dfreq, daxis).double() for s in (1.0, -1.0))
        diff = ((up - down) * w.double()).sum().item() / 2
        assert abs(diff - leaf.grad.flatten()[k].item()) <= 20 * 6 * 10 * 4.5 * 2.0 ** -24


def test_refusals(mb, torch):
    x, w, pos, dpos, freq, axis, dfreq, daxis = problem(torch, torch.float32)
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError):
        mb.rope(leaf, dpos, dfreq, daxis, out=torch.empty_like(x))
    y = mb.rope(leaf, dpos, dfreq, daxis)
    dpos += 1                                   # what the backward pass needs is not what it was
    with pytest.raises(RuntimeError):
        y.sum().backward()
