"""Which overlaps of its operands the rotation of many tokens refuses, through the C ABI, without a GPU."""
import ctypes
import random

from test_paged_cache_arguments import A, INVALID, RopeTensor


def refused(pkg, tensors, tokens=6, dim=32, kind=0):
    """For operands that do overlap only: others would be launched."""
    many = (RopeTensor * len(tensors))(*tensors)
    return pkg.lib().tcrv_cuda_rope_rows(kind, tokens, dim, dim, ctypes.addressof(many), len(tensors), A, A, 1.0, 0, None) == INVALID


def elements(base, tokens, heads, token, head, dim):
    return {base + t * token + h * head + d for t in range(tokens) for h in range(heads) for d in range(dim)}


def test_overlapping_operands_are_refused(pkg):
    rng = random.Random(1)
    found = 0
    for _ in range(4000):
        kind, size = rng.choice(((0, 4), (1, 2)))
        tokens, heads, dim = rng.randint(1, 6), rng.randint(1, 4), 32
        head = rng.choice((32, 40, 64, 200))
        token = rng.choice((head * heads + rng.choice((0, 32, 500)), 32, head))
        other = (rng.randint(1, 4), token, head) if rng.random() < 0.7 else (rng.randint(1, 4), token + 32, head)
        shift = rng.randint(-700, 700)
        x, y = (0, tokens, heads, token, head, dim), (shift, tokens, other[0], other[1], other[2], dim)
        far = A + (1 << 30)
        if not elements(*x) & elements(*y):
            continue
        found += 1
        # the output of a second tensor over the input of the first, and over its output
        a = RopeTensor(A, far, heads, token, head, 4096, 512)
        b = RopeTensor(far * 2, A + shift * size, other[0], 4096, 512, other[1], other[2])
        assert refused(pkg, [a, b], tokens, dim, kind) and refused(pkg, [b, a], tokens, dim, kind)
        a = RopeTensor(far, A, heads, 4096, 512, token, head)
        assert refused(pkg, [a, b], tokens, dim, kind) and refused(pkg, [b, a], tokens, dim, kind)
        if other[0] == heads and (shift != 0 or (tokens > 1 and other[1] != token)):
            assert refused(pkg, [RopeTensor(A, A + shift * size, heads, token, head, other[1], other[2])], tokens, dim, kind)
    assert found > 500


def test_its_own_memory_in_another_order_is_refused(pkg):
    assert refused(pkg, [RopeTensor(A, A, 6, 192, 32, 32, 192)])
    assert refused(pkg, [RopeTensor(A, A, 6, 192, 32, 384, 32)])
