"""Rotary positions of many tokens against their definition in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def definition(x, positions, freqs, halves, magnitude, inverse):
    """x: float64 (tokens, heads, dim)."""
    n = 2 * len(freqs)
    y = x.copy()
    angle = positions.astype(np.float64)[:, None] * freqs[None]
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * (-magnitude if inverse else magnitude)
    lo, hi = (slice(0, n // 2), slice(n // 2, n)) if halves else (slice(0, n, 2), slice(1, n, 2))
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., lo] * s + x[..., hi] * c
    return y


def bound(x, y, freqs, halves, magnitude, kind):
    """The angle is rounded to f32 within half a turn (2^-23), its sine and cosine are within 2 steps (2^-23), their product with
    the magnitude, the two products and the sum are rounded (3 * 2^-24 of the two terms): (2^-22 + 3 * 2^-24) (|lo| + |hi|).
    64-bit angles of positions up to 2^31 add 2^-21 at most.  Last, the result's rounding."""
    n = 2 * len(freqs)
    size = np.zeros_like(x)
    lo, hi = (slice(0, n // 2), slice(n // 2, n)) if halves else (slice(0, n, 2), slice(1, n, 2))
    both = np.abs(x[..., lo]) + np.abs(x[..., hi])
    size[..., lo] = size[..., hi] = both * abs(magnitude)
    b = size * (2.0 ** -22 + 3 * 2.0 ** -24)
    if n:
        b[..., :n] += np.abs(y[..., :n]) * HALF_STEP[kind] + (2.0 ** -25 if kind == "float16" else 0.0)
    return b


def values(torch, rng, shape, kind):
    t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(getattr(torch, kind))
    return t.cuda(), t.double().numpy()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", [(1, 1, 1, 64, 64), (3, 7, 1, 128, 128), (5, 4, 2, 96, 24), (2, 3, 3, 80, 20),
                                                           (33, 32, 8, 128, 64), (700, 4, 4, 256, 256), (9, 2, 1, 40, 6), (4, 2, 2, 66, 66)])
def test_rope(cuda, pkg, kind, halves, tokens, heads, kv_heads, dim, rot):
    rng = np.random.default_rng(tokens + dim)
    q, q64 = values(cuda, rng, (tokens, heads, dim), kind)
    k, k64 = values(cuda, rng, (tokens, kv_heads, dim), kind)
    positions = rng.integers(0, 1 << 20, tokens)
    freqs = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    f = cuda.from_numpy(freqs).cuda()
    for wide, magnitude, inverse in ((False, 1.0, False), (True, 1.25, True)):
        p = cuda.from_numpy(positions.astype(np.int64 if wide else np.int32)).cuda()
        got = pkg.rope_qk(q, k, p, f, halves=halves, magnitude=magnitude, inverse=inverse)
        for x, y in zip((q64, k64), got):
            want = definition(x, positions, freqs, halves, magnitude, inverse)
            assert (np.abs(y.double().cpu().numpy() - want) <= bound(x, want, freqs, halves, magnitude, kind)).all()
        alone = pkg.rope(k, p, f, halves=halves, magnitude=magnitude, inverse=inverse)
        assert cuda.equal(alone, got[1])
        here = q.clone()
        assert pkg.rope(here, p, f, halves=halves, magnitude=magnitude, inverse=inverse, out=here) is here
        assert cuda.equal(here, got[0])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("halves", [False, True])
def test_strides(cuda, pkg, kind, halves):
    rng = np.random.default_rng(1)
    q, _ = values(cuda, rng, (5, 3, 64), kind)
    k, _ = values(cuda, rng, (5, 2, 64), kind)
    p, f = cuda.arange(7, 12, device="cuda"), pkg.rope_frequencies(32)
    want = pkg.rope_qk(q, k, p, f, halves=halves)
    joint = cuda.zeros(5, 5, 67, dtype=q.dtype, device="cuda")  # queries and keys of one projection, at odd addresses
    joint[:, :3, 2:66], joint[:, 3:, 2:66] = q, k
    out = cuda.full((3, 5, 70), 4.0, dtype=q.dtype, device="cuda")  # heads outside the tokens
    got = pkg.rope_qk(joint[:, :3, 2:66], joint[:, 3:, 2:66], p, f, halves=halves, out=(out[:, :, 1:65].transpose(0, 1), None))
    assert cuda.equal(got[0], want[0]) and cuda.equal(got[1], want[1])
    assert bool((out[..., 0] == 4).all()) and bool((out[..., 65:] == 4).all())
    pkg.rope_qk(joint[:, :3, 2:66], joint[:, 3:, 2:66], p, f, halves=halves, out=(joint[:, :3, 2:66], joint[:, 3:, 2:66]))
    assert cuda.equal(joint[:, :3, 2:66], want[0]) and cuda.equal(joint[:, 3:, 2:66], want[1])
    assert not bool(joint[..., :2].any()) and not bool(joint[..., 66:].any())
    one = q[:1].expand(5, 3, 64)  # the same values at five positions
    assert cuda.equal(pkg.rope(one, p, f, halves=halves), pkg.rope(one.contiguous(), p, f, halves=halves))


@pytest.mark.parametrize("halves", [False, True])
def test_gradient(cuda, pkg, halves):
    rng = np.random.default_rng(2)
    x, x64 = values(cuda, rng, (6, 3, 64), "float32")
    g, g64 = values(cuda, rng, (6, 3, 64), "float32")
    positions = rng.integers(0, 4096, 6)
    p, f = cuda.from_numpy(positions).cuda(), pkg.rope_frequencies(48)
    freqs = f.cpu().numpy()
    dx = pkg.rope(g, p, f, halves=halves, magnitude=1.1, inverse=True).double().cpu().numpy()
    # the formula: the transposed rotation
    want = definition(g64, positions, freqs, halves, 1.1, True)
    tolerance = bound(g64, want, freqs, halves, 1.1, "float32")
    assert (np.abs(dx - want) <= tolerance).all()
    # differences of the definition, which is linear: exact for any step, up to 64-bit rounding
    for _ in range(40):
        at = tuple(int(rng.integers(0, n)) for n in x64.shape)
        up, down = x64.copy(), x64.copy()
        up[at] += 0.5
        down[at] -= 0.5
        slope = ((definition(up, positions, freqs, halves, 1.1, False) - definition(down, positions, freqs, halves, 1.1, False)) * g64).sum()
        assert abs(dx[at] - slope) <= tolerance[at] + 1e-11
    # and the framework's own two directions: <g, R x> = <R' g, x>
    y = pkg.rope(x, p, f, halves=halves, magnitude=1.1).double().cpu().numpy()
    assert abs((g64 * y).sum() - (dx * x64).sum()) <= (np.abs(g64) * bound(x64, y, freqs, halves, 1.1, "float32")).sum() + (np.abs(x64) * tolerance).sum()


def test_far_and_negative_positions(cuda, pkg):
    positions = np.array([0, -1, 1, 2 ** 31 - 1, -(2 ** 31), 1 << 24, (1 << 24) + 1])
    x = np.zeros((7, 1, 4))
    x[..., 0] = 1.0
    freqs = np.array([1.0, 1e-3])
    got = pkg.rope(cuda.from_numpy(x).float().cuda(), cuda.from_numpy(positions).cuda(), cuda.from_numpy(freqs).cuda())
    want = definition(x, positions, freqs, False, 1.0, False)
    # 2^31 radians in 64 bits: 2^-22 of a radian either side
    assert np.abs(got.double().cpu().numpy() - want).max() <= 2.0 ** -22 + 3 * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -24


def test_frequencies(cuda, pkg):
    def plain(n, base):
        return [base ** (-2.0 * p / n) for p in range(n // 2)]
    def close(got, want):
        assert got.dtype == cuda.float64
        np.testing.assert_allclose(got.cpu().numpy(), want, rtol=1e-12, atol=0)
    close(pkg.rope_frequencies(128), plain(128, 1e4))
    close(pkg.rope_frequencies(6, 5e5), plain(6, 5e5))
    close(pkg.rope_frequencies(64, scaling="linear", factor=8.0), [f / 8 for f in plain(64, 1e4)])
    n, base, factor, original, low, high = 128, 1e4, 16.0, 4096.0, 1.0, 32.0
    pair = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    first, last = max(0, math.floor(pair(high))), min(n - 1, math.ceil(pair(low)))
    assert 0 < first < last < 64
    keep = [1 - min(1.0, max(0.0, (p - first) / (last - first))) for p in range(n // 2)]
    close(pkg.rope_frequencies(n, base, "yarn", factor, original, low, high), [f * k + f / factor * (1 - k) for f, k in zip(plain(n, base), keep)])
    keep = [min(1.0, max(0.0, (original * f / (2 * math.pi) - 1.0) / 3.0)) for f in plain(n, base)]
    close(pkg.rope_frequencies(n, base, "bands", factor, original, 1.0, 4.0), [f * k + f / factor * (1 - k) for f, k in zip(plain(n, base), keep)])
    assert pkg.rope_frequencies(0).numel() == 0


def test_nothing_to_do(cuda, pkg):
    f = pkg.rope_frequencies(64)
    p = cuda.zeros(0, dtype=cuda.int32, device="cuda")
    q, k = pkg.rope_qk(cuda.empty(0, 4, 64, device="cuda"), cuda.empty(0, 2, 64, device="cuda"), p, f)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    x = cuda.randn(3, 2, 64, device="cuda")
    p = cuda.arange(3, device="cuda")
    assert cuda.equal(pkg.rope(x, p, f[:0]), x)  # no pair turns
    assert pkg.rope(x[:, :0], p, f).shape == (3, 0, 64)


def test_refusals(cuda, pkg):
    x, p, f = cuda.zeros(3, 2, 64, device="cuda"), cuda.arange(3, device="cuda"), pkg.rope_frequencies(64)
    def bad(error, *a, **k):
        with pytest.raises(error):
            pkg.rope(*a, **k)
    bad(TypeError, x.double(), p, f)
    bad(TypeError, x.cpu(), p, f)
    bad(ValueError, x[0], p, f)
    bad(ValueError, x[..., ::2], p, f[:16])
    bad(TypeError, x, p.float(), f)
    bad(ValueError, x, p[:2], f)
    bad(TypeError, x, p, f.float())
    bad(ValueError, x, p, pkg.rope_frequencies(66))
    bad(ValueError, x, p, f, out=x[:2])
    bad(TypeError, x, p, f, out=x.half())
    bad(ValueError, x, p, f, out=x[:, :1].expand(3, 2, 64))
    with pytest.raises(ValueError):
        pkg.rope_qk(x, x[:2], p, f)
    with pytest.raises(TypeError):
        pkg.rope_qk(x, x.half(), p, f)
    with pytest.raises(ValueError):
        pkg.rope_frequencies(64, scaling="other")
    for args in ((63,), (64, 1.0), (64, 1e4, "linear", 0.0), (64, 1e4, "yarn", 2.0, 0.0), (64, 1e4, "bands", 2.0, 4096.0, 4.0, 4.0), (5000,)):
        with pytest.raises(pkg.TcrvCudaError):
            pkg.rope_frequencies(*args)
