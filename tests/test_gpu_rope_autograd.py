"""Rotary positions of tensors that require a gradient."""
import pytest

from test_gpu_rope import bound, definition, values

import numpy as np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_the_gradient_is_recorded(cuda, pkg, halves, inverse):
    rng = np.random.default_rng(1)
    q, _ = values(cuda, rng, (6, 4, 64), "float32")
    k, _ = values(cuda, rng, (6, 2, 64), "float32")
    gq, gq64 = values(cuda, rng, (6, 4, 64), "float32")
    gk, gk64 = values(cuda, rng, (6, 2, 64), "float32")
    positions = rng.integers(0, 4096, 6)
    p, f = cuda.from_numpy(positions).cuda(), pkg.rope_frequencies(48)
    freqs = f.cpu().numpy()
    with cuda.no_grad():
        plain = pkg.rope_qk(q, k, p, f, halves=halves, magnitude=1.1, inverse=inverse)
    assert not plain[0].requires_grad
    q.requires_grad_(), k.requires_grad_()
    got = pkg.rope_qk(q, k, p, f, halves=halves, magnitude=1.1, inverse=inverse)
    assert cuda.equal(got[0], plain[0]) and cuda.equal(got[1], plain[1])
    (got[0] * gq).sum().backward(retain_graph=True)  # the queries alone, then both
    assert k.grad is None or not bool(k.grad.any())
    q.grad = k.grad = None
    ((got[0] * gq).sum() + (got[1] * gk).sum()).backward()
    for x, g in ((q, gq64), (k, gk64)):
        want = definition(g, positions, freqs, halves, 1.1, not inverse)
        assert (np.abs(x.grad.double().cpu().numpy() - want) <= bound(g, want, freqs, halves, 1.1, "float32")).all()


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_one_tensor_strides_and_a_broadcast_gradient(cuda, pkg, kind):
    rng = np.random.default_rng(2)
    wide, _ = values(cuda, rng, (5, 3, 96), kind)
    positions = rng.integers(0, 4096, 5)
    p, f = cuda.from_numpy(positions).cuda(), pkg.rope_frequencies(64)
    wide.requires_grad_()
    pkg.rope(wide[..., 16:80], p, f).sum().backward()  # (the gradient of a sum is one number, expanded)
    ones = np.ones((5, 3, 64))
    want = definition(ones, positions, f.cpu().numpy(), False, 1.0, True)
    assert (np.abs(wide.grad[..., 16:80].double().cpu().numpy() - want) <= bound(ones, want, f.cpu().numpy(), False, 1.0, kind)).all()
    assert not bool(wide.grad[..., :16].any()) and not bool(wide.grad[..., 80:].any())
    # only one of a pair requires one
    q, k = values(cuda, rng, (5, 3, 64), kind)[0], values(cuda, rng, (5, 1, 64), kind)[0].requires_grad_()
    a, b = pkg.rope_qk(q, k, p, f)
    (a.float().sum() + b.float().sum()).backward()
    assert q.grad is None and k.grad is not None


def test_a_second_gradient(cuda, pkg):
    x = cuda.randn(4, 2, 64, device="cuda", requires_grad=True)
    p, f = cuda.arange(4, device="cuda"), pkg.rope_frequencies(64)
    y = pkg.rope(x, p, f)
    (g,) = cuda.autograd.grad((y ** 2).sum(), x, create_graph=True)
    (h,) = cuda.autograd.grad(g.sum(), x)
    assert bool((h - 2.0).abs().max() <= 2.0 ** -18)  # R' R = 1, twice: a few f32 steps of 2


def test_outputs_that_would_lose_a_gradient_are_refused(cuda, pkg):
    x = cuda.randn(4, 2, 64, device="cuda", requires_grad=True)
    p, f = cuda.arange(4, device="cuda"), pkg.rope_frequencies(64)
    for out in (cuda.empty_like(x), x * 1.0, x):
        with pytest.raises(ValueError):
            pkg.rope(x, p, f, out=out)
    with pytest.raises(ValueError):
        pkg.rope(x.detach(), p, f, out=x * 1.0)
    with pytest.raises(ValueError):
        pkg.rope_qk(x.detach(), x, p, f, out=(cuda.empty_like(x), None))
    with cuda.no_grad():
        out = cuda.empty_like(x)
        assert pkg.rope(x, p, f, out=out) is out
    with cuda.inference_mode():
        assert cuda.equal(pkg.rope(x, p, f), out)
