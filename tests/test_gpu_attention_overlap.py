"""Attention into the queries' memory: in place, or refused."""
import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu

CASES = [("float32", [700, 5, 40], [1, 1, 1], 64), ("bfloat16", [900, 300, 33], [1, 200, 2], 64), ("float16", [5000], [1], 128),
         ("bfloat16", [2500], [40], 128), ("float32", [300, 90], [40, 7], 96)]


def operands(torch, kind, lens, new, dim):
    rng = np.random.default_rng(dim)
    table, pages = ref.tables(rng, lens, 16)
    i32 = lambda x: torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")  # noqa: E731
    cache = torch.from_numpy(ref.random_cache(rng, pages, 2, 16, dim)).cuda()
    first = np.concatenate(([0], np.cumsum(new)))
    q = torch.from_numpy(rng.standard_normal((first[-1], 12, dim)).astype(np.float32)).to(getattr(torch, kind)).cuda()
    return q, (cache, torch.from_numpy(table).cuda(), i32(lens)), dict(first_rows=i32(first), max_new=max(new))


@pytest.mark.parametrize("kind,lens,new,dim", CASES)
def test_in_place(cuda, pkg, kind, lens, new, dim):
    wide, rest, k = operands(cuda, kind, lens, new, dim)
    q = wide[:, 2:10]
    want, lse = pkg.attention_q4_0(q, *rest, with_lse=True, **k)
    kept = wide.clone()
    got, here = pkg.attention_q4_0(q, *rest, with_lse=True, out=q, **k)
    pkg.check_device_errors()
    assert got is q and cuda.equal(q, want) and cuda.equal(here, lse)
    assert cuda.equal(wide[:, :2], kept[:, :2]) and cuda.equal(wide[:, 10:], kept[:, 10:])


@pytest.mark.parametrize("kind,lens,new,dim", CASES[:2])
def test_other_overlaps_are_refused(cuda, pkg, kind, lens, new, dim):
    wide, rest, k = operands(cuda, kind, lens, new, dim)
    kept, q = wide.clone(), wide[:, :8]
    outs = [wide[:, 1:9], wide[:, 4:], wide.as_strided(q.shape, (dim, dim * len(wide), 1))]
    for out in outs:
        with pytest.raises(pkg.TcrvCudaError):
            pkg.attention_q4_0(q, *rest, out=out, **k)
    assert cuda.equal(wide, kept)
    side = cuda.zeros(len(wide), 16, dim, dtype=wide.dtype, device="cuda")  # beside one another in one buffer
    side[:, :8] = q
    pkg.attention_q4_0(side[:, :8], *rest, out=side[:, 8:], **k)
    assert cuda.equal(side[:, 8:], pkg.attention_q4_0(q, *rest, **k)) and cuda.equal(side[:, :8], q)
