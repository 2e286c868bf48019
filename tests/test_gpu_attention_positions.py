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
