"""What the entries around the paged Q4_0 cache refuse before any CUDA call, through the C ABI, without a GPU."""
import ctypes

import numpy as np
import pytest

import paged_reference as ref

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, -1, -2, -5
sz, p = ctypes.c_size_t, ctypes.c_void_p


class RopeTensor(ctypes.Structure):
    _fields_ = [("x", p), ("y", p)] + [(n, sz) for n in ("heads", "x_token", "x_head", "y_token", "y_head")]


class Cache(ctypes.Structure):
    _fields_ = [("data", p)] + [(n, sz) for n in ("pages", "kv_heads", "groups", "dim", "page_stride")]


class Plan(ctypes.Structure):
    _fields_ = ([(n, sz) for n in ("requests", "page_tokens", "width", "rows", "free_capacity")] +
                [(n, p) for n in ("context_lens", "new_lens", "block_table")] + [("table_stride", sz)] +
                [(n, p) for n in ("free_pages", "free_count", "first_rows", "kv_lens", "slots", "positions", "row_requests", "info")])


class Attention(ctypes.Structure):
    _fields_ = ([("type", ctypes.c_int)] + [(n, sz) for n in ("requests", "rows", "heads", "max_new")] +
                [("q", p), ("q_row_stride", sz), ("q_head_stride", sz), ("out", p), ("out_row_stride", sz), ("out_head_stride", sz),
                 ("lse", p), ("cache", Cache), ("block_table", p), ("width", sz), ("table_stride", sz), ("kv_lens", p),
                 ("first_rows", p), ("scale", ctypes.c_float), ("window", sz), ("workspace", p), ("workspace_bytes", sz)])


A = 1 << 20  # an address that is aligned; nothing here gets as far as using it


def cache(**changes):
    c = Cache(A, 8, 2, 2, 64, 2 * 2 * 18 * 64)
    for k, v in changes.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [({"dim": 0}, INVALID), ({"dim": 40}, INVALID), ({"kv_heads": 0}, INVALID), ({"groups": 0}, INVALID), ({"data": None}, INVALID),
              ({"data": A + 8}, INVALID), ({"page_stride": 4600}, INVALID), ({"page_stride": 2304}, INVALID), ({"dim": 2048}, UNSUPPORTED),
              ({"kv_heads": 1 << 20}, UNSUPPORTED), ({"pages": 1 << 32}, UNSUPPORTED)]


def test_rope_arguments(pkg):
    L = pkg.lib()
    t = RopeTensor(A, A, 4, 256, 64, 256, 64)
    def call(kind=0, tokens=3, dim=64, rot=64, tensors=t, count=1, positions=A, freqs=A, flags=0):
        return L.tcrv_cuda_rope_rows(kind, tokens, dim, rot, ctypes.addressof(tensors) if tensors else None, count, positions, freqs, 1.0, flags, None)
    for bad in ({"kind": 3}, {"kind": -1}, {"rot": 63}, {"rot": 66}, {"tensors": None}, {"count": 5}, {"positions": None}, {"freqs": None},
                {"flags": 8}, {"tensors": RopeTensor(None, A, 4)}, {"tensors": RopeTensor(A, None, 4)}):
        assert call(**bad) == INVALID, bad
    assert call(dim=8192) == UNSUPPORTED and call(tokens=1 << 40) == UNSUPPORTED
    assert call(tensors=RopeTensor(A, A, 1 << 20)) == UNSUPPORTED
    many = (RopeTensor * 4)(*[RopeTensor(A, A, 65535) for _ in range(4)])
    assert call(tensors=many, count=4, dim=4096) == UNSUPPORTED
    assert call(tokens=0) == OK and call(count=0) == OK and call(tensors=RopeTensor(None, None, 0)) == OK
    def freqs(n=64, base=1e4, scaling=0, factor=1.0, original=0.0, low=1.0, high=32.0, out=A):
        return L.tcrv_cuda_rope_frequencies_f64(n, base, scaling, factor, original, low, high, out, None)
    nan = float("nan")
    for bad in ({"n": 63}, {"base": 1.0}, {"base": nan}, {"factor": 0.0}, {"factor": nan}, {"scaling": 4}, {"scaling": -1}, {"out": None},
                {"scaling": 2}, {"scaling": 3, "original": nan}, {"scaling": 2, "original": 1e3, "low": 0.0}, {"scaling": 3, "original": 1e3, "low": 32.0}):
        assert freqs(**bad) == INVALID, bad
    assert freqs(n=8192) == UNSUPPORTED


def test_store_and_load_arguments(pkg):
    L = pkg.lib()
    def store(c, kind=0, rows=3, k=A, v=A, slots=A):
        return L.tcrv_cuda_kv_store_q4_0(kind, rows, k, 128, 64, v, 128, 64, slots, ctypes.addressof(c) if c else None, None)
    def load(c, kind=0, rows=3, k=A, v=A, slots=A):
        return L.tcrv_cuda_kv_load_q4_0(kind, rows, k, v, slots, ctypes.addressof(c) if c else None, None)
    for call in (store, load):
        for changes, status in BAD_CACHES:
            assert call(cache(**changes)) == status, changes
        assert call(None) == INVALID and call(cache(), kind=3) == INVALID and call(cache(), k=None) == INVALID
        assert call(cache(), v=None) == INVALID and call(cache(), slots=None) == INVALID
        assert call(cache(), rows=1 << 32) == UNSUPPORTED and call(cache(), rows=0, k=None) == OK
    assert load(cache(), k=A + 4) == INVALID


def test_plan_arguments(pkg):
    L = pkg.lib()
    def call(**changes):
        c = Plan(2, 16, 4, 5, 8, A, A, A, 4, A, A, A, A, A, A, A, A)
        for k, v in changes.items():
            setattr(c, k, v)
        return L.tcrv_cuda_kv_plan(ctypes.addressof(c), None)
    assert L.tcrv_cuda_kv_plan(None, None) == INVALID
    for name in ("context_lens", "new_lens", "block_table", "free_pages", "free_count", "first_rows", "kv_lens", "slots", "positions", "row_requests", "info"):
        assert call(**{name: None}) == INVALID, name
    assert call(page_tokens=0) == INVALID and call(table_stride=3) == INVALID
    for big in ({"requests": 16385}, {"page_tokens": 1 << 20}, {"rows": 1 << 31}, {"width": 1 << 30}, {"free_capacity": 1 << 31}):
        assert call(**big) == UNSUPPORTED, big


def test_attention_arguments(pkg):
    L = pkg.lib()
    def make(**changes):
        c = Attention(0, 2, 2, 4, 1, A, 256, 64, A, 256, 64, None, cache(), A, 4, 4, A, None, 0.125, 0, A, 0)
        for k, v in changes.items():
            setattr(c, k, v)
        return c
    def call(**changes):
        c = make(**changes)
        return L.tcrv_cuda_attention_q4_0(ctypes.addressof(c), None)
    assert L.tcrv_cuda_attention_q4_0(None, None) == INVALID
    for changes, status in BAD_CACHES:
        assert call(cache=cache(**changes)) == status, changes
    for bad in ({"type": 3}, {"heads": 0}, {"heads": 5}, {"max_new": 0}, {"q": None}, {"out": None}, {"kv_lens": None}, {"block_table": None}, {"table_stride": 3}):
        assert call(**bad) == INVALID, bad
    for dim in (32, 160, 512):
        assert call(cache=cache(dim=dim, page_stride=2 * 2 * 18 * dim)) == UNSUPPORTED
    for big in ({"heads": 1 << 17}, {"requests": 1 << 31}, {"rows": 1 << 31}, {"max_new": 1 << 30}, {"width": 1 << 30}):
        assert call(**big) == UNSUPPORTED, big
    for bad in ({"workspace": None, "workspace_bytes": 1 << 40}, {"workspace": A + 16, "workspace_bytes": 1 << 40}, {"workspace_bytes": 16}):
        assert call(**bad) == WORKSPACE, bad
    assert call(requests=0, q=None) == OK and call(rows=0, q=None) == OK
    def size(**changes):
        c = make(**changes)
        return L.tcrv_cuda_attention_q4_0_workspace_bytes(ctypes.addressof(c))
    assert size() > 0 and size(q=None, block_table=None, cache=cache(data=None)) == size()
    assert size(rows=0) == 0 and size(max_new=1 << 20) == size(max_new=2)
    assert size(heads=5) == 0 and size(requests=0) == 0 and L.tcrv_cuda_attention_q4_0_workspace_bytes(None) == 0


@pytest.mark.parametrize("dim", [32, 96, 128])
def test_the_reference_layout_holds_every_value_once(dim):
    key, value, shift, kd, vd = ref.places(dim)
    assert sorted((key * 8 + shift).ravel()) == [8 * b + s for b in range(8 * dim) for s in (0, 4)]
    assert sorted((value * 8 + shift).ravel()) == [8 * b + s for b in range(8 * dim, 16 * dim) for s in (0, 4)]
    assert sorted(np.concatenate((kd, vd)).ravel()) == list(range(16 * dim, 18 * dim, 2))
    rng = np.random.default_rng(dim)
    quants, scales = rng.integers(0, 16, (2, 3, 16, dim), dtype=np.uint8), rng.uniform(0.1, 1, (2, 3, 16, dim // 32)).astype(np.float16)
    for part, got in enumerate(ref.decode(ref.encode(quants, scales))):
        assert np.array_equal(got, (quants[part] - 8.0) * np.repeat(scales[part].astype(np.float64), 32, -1))


def test_the_attention_definition_by_hand():
    # one token, then two of equal score: the value itself, then the mean of two
    quants = np.full((2, 1, 1, 1, 16, 32), 8, np.uint8)
    quants[1, 0, 0, 0, 0], quants[1, 0, 0, 0, 1] = 10, 14
    cache64 = ref.encode(quants, np.full((2, 1, 1, 1, 16, 1), 0.5, np.float16))
    out, lse, _ = ref.attention(np.ones((2, 1, 32)), cache64, np.array([[0]]), [2], [0, 2], 1.0)
    assert np.allclose(out[0], 1.0) and np.allclose(out[1], 2.0) and np.allclose(lse[:, 0], [0.0, np.log(2.0)])
    out, _, _ = ref.attention(np.ones((2, 1, 32)), cache64, np.array([[0]]), [2], [0, 2], 1.0, window=1)
    assert np.allclose(out[1], 3.0)
