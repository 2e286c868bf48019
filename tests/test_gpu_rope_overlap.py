"""Rotary positions into outputs that share memory with an input or with one another."""
import pytest

pytestmark = pytest.mark.gpu

KINDS = ["float32", "bfloat16"]


def operands(torch, pkg, kind, tokens, rot=48):
    torch.manual_seed(tokens)
    p, f = torch.arange(3, 3 + tokens, device="cuda"), pkg.rope_frequencies(rot)
    return torch.randn(tokens, 24, 64, device="cuda").to(getattr(torch, kind)), p, f


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("halves", [False, True])
def test_overlaps_are_refused(cuda, pkg, kind, halves):
    x, p, f = operands(cuda, pkg, kind, 8)
    def bad(call, *a, **k):
        before = x.clone()
        with pytest.raises(pkg.TcrvCudaError):
            call(*a, halves=halves, **k)
        assert cuda.equal(x, before)
    square = x[:, :8]
    bad(pkg.rope, square, p, f, out=square.transpose(0, 1))          # its own memory in another order
    one = x[:1, :8]                                                  # the strides of a single token do not matter
    assert pkg.rope(one.clone(), p[:1], f, halves=halves, out=None).shape == one.shape
    bad(pkg.rope, x[:7], p[:7], f, out=x[1:])                        # a token on
    bad(pkg.rope, x[:, :8], p, f, out=x[:, 1:9])                     # a head on
    wide = x.view(8, 12, 128)
    bad(pkg.rope, wide[..., :64], p, f, out=wide[..., 32:96])        # half a head on
    bad(pkg.rope, x[:1].expand(8, 24, 64), p, f, out=x)              # a broadcast input's own row
    bad(pkg.rope_qk, x[:, :8], x[:, 8:16], p, f, out=(x[:, 8:16], None))             # the keys' memory
    bad(pkg.rope_qk, x[:, :8], x[:, 8:16], p, f, out=(None, x[:, 4:12]))
    other = cuda.empty_like(x[:, :8])
    bad(pkg.rope_qk, x[:, :8], x[:, 8:16], p, f, out=(other, other))                 # one output for both
    bad(pkg.rope_qk, x[:, :8], x[:, 8:16], p, f, out=(other, other.transpose(0, 1)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("tokens", [1, 2, 9])
def test_places_of_one_buffer_that_do_not_overlap(cuda, pkg, kind, halves, tokens):
    x, p, f = operands(cuda, pkg, kind, tokens)
    q, k, rest = x[:, :8], x[:, 8:12], x[:, 12:24]
    want = pkg.rope_qk(q, k, p, f, halves=halves)
    kept = x.clone()
    pkg.rope_qk(q, k, p, f, halves=halves, out=(rest[:, :8], rest[:, 8:]))           # behind the inputs of each token
    assert cuda.equal(rest[:, :8], want[0]) and cuda.equal(rest[:, 8:], want[1]) and cuda.equal(x[:, :12], kept[:, :12])
    wide = cuda.zeros(tokens, 8, 128, dtype=x.dtype, device="cuda")                  # the two halves of wider heads
    wide[..., :64] = q
    pkg.rope(wide[..., :64], p, f, halves=halves, out=wide[..., 64:])
    assert cuda.equal(wide[..., 64:], want[0]) and cuda.equal(wide[..., :64], q)
    pkg.rope_qk(q, k, p, f, halves=halves, out=(q, k))                               # in place
    assert cuda.equal(q, want[0]) and cuda.equal(k, want[1])
    single = kept[:, :1].clone()                                                     # one head: its stride does not matter
    pkg.rope(single, p, f, halves=halves, out=single.as_strided(single.shape, (64, 640, 1)))
    assert cuda.equal(single, want[0][:, :1])
