"""Attention over the paged Q4_0 cache: where a request's rows sit when a call leaves some of its rows or tokens out, and far contexts."""
import numpy as np
import pytest

import attention_rms as rms
import paged_reference as ref

pytestmark = pytest.mark.gpu


def case(torch, pkg, kind, lens, first, rows, max_new, heads, kv_heads, dim, window=0, width=None, seed=0, page_tokens=16):
    """Requests whose rows begin at first[r]; `width` pages to a request, although its length may say more."""
    rng = np.random.default_rng(seed)
    width = width or max(1, max(-(-n // page_tokens) for n in lens))
    table = np.arange(len(lens) * width).reshape(len(lens), width).astype(np.int32)
    cache = ref.random_cache(rng, table.size, kv_heads, page_tokens, dim)
    q = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).to(getattr(torch, kind))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    _, lse = pkg.attention_q4_0(q.cuda(), torch.from_numpy(cache).cuda(), i32(table.tolist()), i32(lens), first_rows=i32(first),
                                max_new=max_new, window=window, out=out, with_lse=True)
    pkg.check_device_errors()
    d = rms.definition(q.double().numpy(), cache, table, lens, first, dim ** -0.5, window, max_new)
    left = np.isnan(d["out"]).all((1, 2))
    assert bool((out.cpu()[torch.from_numpy(left)] == 7.0).all())
    biggest = min(max_new, int(np.diff(first).max())) * heads // kv_heads
    rms.check(out, lse, d, kind, kind != "float32" and dim in (64, 128) and biggest > 32)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("max_new", [1, 2, 5, 40, 90])
def test_fewer_rows_than_a_request_has(cuda, pkg, kind, window, max_new):
    # rows behind max_new are left out; the others stay where they are
    case(cuda, pkg, kind, [50, 130, 97], [0, 7, 107, 110], 110, max_new, 4, 2, 64, window=window, seed=max_new)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 20])
def test_rows_behind_the_queries(cuda, pkg, kind, window):
    case(cuda, pkg, kind, [150, 150], [0, 2, 92], 52, 90, 4, 2, 64, window=window, seed=4)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 30, 300])
@pytest.mark.parametrize("new", [1, 6, 80])
def test_contexts_longer_than_their_table(cuda, pkg, kind, window, new):
    # tokens behind the table are unseen, and the rows still sit at the end of the length
    case(cuda, pkg, kind, [100, 2 ** 31 - 1, 120], [0, new, new + 1, 2 * new + 1], 2 * new + 1, new, 4, 2, 64, window=window, width=6, seed=new)


@pytest.mark.parametrize("kind,new", [("float32", 1), ("float16", 33)])
def test_windows_beyond_2_to_the_30(cuda, pkg, kind, new):
    """A context of 2^30 + 100 tokens (one page of nearly 2^20 again and again) whose first token decides: a window that holds it, and
    one that ends before it."""
    groups = 65535
    page_tokens = 16 * groups
    n = (1 << 30) + 100
    width = -(-n // page_tokens)
    rng = np.random.default_rng(0)
    two = np.zeros((2, 1, groups, 18 * 64), np.uint8)
    plain = ref.random_cache(rng, 1, 1, 16, 64)[0, 0, 0]
    plain[16 * 64:17 * 64] = 0  # keys of zero
    two[0, 0, :] = two[1, 0, :] = plain
    key, value, shift, kd, vd = ref.places(64)
    first = two[1, 0, 0]
    quants = np.full((2, 16, 64), 8, np.uint8)
    quants[:, 0] = 15
    scales = np.full((2, 16, 2), 1.0, np.float16)
    first[:] = ref.encode(quants[:, None], scales[:, None])[0]
    cache = cuda.from_numpy(two).cuda()
    table = cuda.zeros(1, width, dtype=cuda.int32, device="cuda")
    table[0, 0] = 1
    i32 = lambda x: cuda.tensor(x, dtype=cuda.int32, device="cuda")  # noqa: E731
    q = cuda.ones(new, 1, 64, dtype=getattr(cuda, kind), device="cuda")
    def run(window):
        return pkg.attention_q4_0(q, cache, table, i32([n]), first_rows=i32([0, new]), max_new=new, window=window, scale=1.0)
    seen = run(n)  # a score of 448 against zeros: the first token's values
    pkg.check_device_errors()
    assert bool((seen == 7.0).all())
    last = run(n - 1)  # the last row does not see it, the others do
    pkg.check_device_errors()
    assert bool((last[:-1] == 7.0).all()) and bool((last[-1].abs() < 2.5).all())  # (a mean of values of at most 8 * 0.3)
