"""Attention right behind the store that fills its cache, without a synchronisation between, again and again in the same pages."""
import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,new,dim", [("bfloat16", 700, 128), ("float16", 300, 64), ("bfloat16", 1, 128), ("float32", 3, 64)])
def test_every_call_sees_the_store_before_it(cuda, pkg, kind, new, dim):
    rng = np.random.default_rng(new)
    n, rounds, dtype = 900, 12, getattr(cuda, kind)
    table, pages = ref.tables(rng, [n], 32)
    at = np.arange(n)
    slots = cuda.from_numpy(table[0, at // 32].astype(np.int64) * 32 + at % 32).cuda()
    cuda.manual_seed(new)
    kv = [cuda.randn(2, n, 2, dim, device="cuda").to(dtype) for _ in range(rounds)]
    q = cuda.randn(new, 8, dim, device="cuda").to(dtype)
    i32 = lambda x: cuda.tensor(x, dtype=cuda.int32, device="cuda")  # noqa: E731
    lens, first, t = i32([n]), i32([0, new]), cuda.from_numpy(table).cuda()
    def attend(cache, out):
        return pkg.attention_q4_0(q, cache, t, lens, first_rows=first, max_new=new, out=out)
    want = []
    for k, v in kv:  # each in a cache of its own
        cache = pkg.kv_cache_q4_0(pages, 2, 32, dim)
        pkg.kv_store_q4_0(cache, k, v, slots)
        cuda.cuda.synchronize()
        want.append(attend(cache, cuda.empty_like(q)))
    cache, got = pkg.kv_cache_q4_0(pages, 2, 32, dim), [cuda.empty_like(q) for _ in kv]
    cuda.cuda.synchronize()
    for (k, v), out in zip(kv, got):
        pkg.kv_store_q4_0(cache, k, v, slots)
        attend(cache, out)
    cuda.cuda.synchronize()
    assert all(cuda.equal(a, b) for a, b in zip(got, want)) and not cuda.equal(got[0], got[1])
