"""Which overlaps of its output with its queries attention refuses, through the C ABI, without a GPU."""
import ctypes

from test_paged_cache_arguments import A, INVALID, WORKSPACE, Attention, cache


def status(pkg, q, out, rows=3, heads=4, q_strides=(256, 64), out_strides=(256, 64), kind=0):
    """With a workspace that is too small, which is looked at last: no call gets to a launch."""
    c = Attention(kind, 2, rows, heads, 1, q, *q_strides, out, *out_strides, None, cache(), A, 4, 4, A, None, 0.125, 0, A, 0)
    return pkg.lib().tcrv_cuda_attention_q4_0(ctypes.addressof(c), None)


def test_overlaps(pkg):
    for kind, size in ((0, 4), (1, 2), (2, 2)):
        row, head = 256 * size, 64 * size
        assert status(pkg, A, A, kind=kind) == WORKSPACE                                     # in place
        assert status(pkg, A, A + 3 * row, kind=kind) == status(pkg, A + 3 * row, A, kind=kind) == WORKSPACE
        for shift in (size, head, row, 2 * row, 2 * row + 3 * head, 3 * row - size):
            assert status(pkg, A, A + shift, kind=kind) == status(pkg, A + shift, A, kind=kind) == INVALID, shift
        wide = (512, 64)  # side by side in one buffer, then a head into one another
        assert status(pkg, A, A + row, q_strides=wide, out_strides=wide, kind=kind) == WORKSPACE
        assert status(pkg, A, A + row - head, q_strides=wide, out_strides=wide, kind=kind) == INVALID
        assert status(pkg, A, A, out_strides=(64, 192), kind=kind) == INVALID                # its own memory in another order
        assert status(pkg, A, A, rows=1, out_strides=(7, 64), kind=kind) == WORKSPACE        # the stride of a single row does not matter
        assert status(pkg, A, A, rows=1, out_strides=(7, 128), kind=kind) == INVALID
