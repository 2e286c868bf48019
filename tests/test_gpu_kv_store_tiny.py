"""The paged cache's writer on blocks so small that the reciprocal of their scale is no number."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_kv_cache import stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1e-37, 2.3e-38, 1e-38, 3e-39, 1e-40, 1e-44])
def test_blocks_below_the_normal_numbers(cuda, pkg, kind, size):
    class Rows:  # (the row quantiser itself: in C the conversion of an infinity to an integer has no meaning)
        @staticmethod
        def quantize_q4_0(x):
            return pkg.quantize_q4_0(cuda.from_numpy(x).cuda()).cpu().numpy()

    rng = np.random.default_rng(3)
    before = ref.random_cache(rng, 2, 2, 16, 96)
    n = 20
    k, v = (rng.uniform(-size, size, (n, 2, 96)).astype(np.float32) for _ in range(2))
    k[3, :, 32:64] = size          # of one sign
    k[4, :, 32:64] = np.resize([size, -size], 32)
    v[5, :, 40:] = 0
    kt, vt = (cuda.from_numpy(x).to(getattr(cuda, kind)).cuda() for x in (k, v))
    slots = rng.permutation(32)[:n].astype(np.int64)
    cache = cuda.from_numpy(before).cuda()
    pkg.kv_store_q4_0(cache, kt, vt, cuda.from_numpy(slots).cuda())
    want = stored(Rows, before, kt.float().cpu().numpy(), vt.float().cpu().numpy(), slots)
    assert np.array_equal(cache.cpu().numpy(), want)
