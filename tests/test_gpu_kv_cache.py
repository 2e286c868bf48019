"""The paged Q4_0 cache's writer, reader and book-keeping."""
import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def stored(O, before, k, v, slots):
    """The cache after a store, from the row quantiser's oracle."""
    after = before.copy()
    dim, page_tokens = k.shape[-1], before.shape[2] * 16
    nb = dim // 32
    key, value, shift, kd, vd = ref.places(dim)
    for row, slot in enumerate(slots):
        if not 0 <= slot < before.shape[0] * page_tokens:
            continue
        page, token = divmod(int(slot), page_tokens)
        for h in range(k.shape[1]):
            group = after[page, h, token // 16]
            t = token % 16
            for x, byte, at in ((k, key, kd), (v, value, vd)):
                blocks = O.quantize_q4_0(np.ascontiguousarray(x[row, h][None], dtype=np.float32)).reshape(nb, 18)
                for b in range(nb):
                    group[at[t, b]], group[at[t, b] + 1] = blocks[b, 0], blocks[b, 1]
                    group[byte[t, 32 * b:32 * b + 16]] = blocks[b, 2:]
    return after


def rows(torch, rng, n, heads, dim, kind):
    t = torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).to(getattr(torch, kind))
    return t.cuda(), t.float().numpy()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,heads,page_tokens", [(32, 1, 16), (64, 3, 32), (96, 2, 16), (128, 8, 64), (256, 1, 48)])
def test_store_is_the_row_quantiser_in_the_slots(cuda, pkg, O, kind, dim, heads, page_tokens):
    rng = np.random.default_rng(dim)
    before = ref.random_cache(rng, 4, heads, page_tokens, dim)
    for n in (1, 2, 17, 41):
        slots = rng.permutation(4 * page_tokens)[:n].astype(np.int64)
        if n == 17:
            slots[3], slots[9], slots[16] = -1, 4 * page_tokens, 1 << 40  # outside the cache: left out
        k, k32 = rows(cuda, rng, n, heads, dim, kind)
        v, v32 = rows(cuda, rng, n, heads, dim, kind)
        if n == 41:  # ties of magnitude (the first one decides the sign), zeros, extremes
            k32[5, 0, :32] = np.resize([0.5, -0.5], 32)
            v32[5, 0, :32] = 0
            v32[7, 0, :32] = -0.0
            k32[6, 0, :32] = 1e-30 if kind != "float16" else 1e-7
            v32[6, 0, :32] = np.resize([3e4, -6e4, 1.0], 32)
            k, v = cuda.from_numpy(k32).to(k.dtype).cuda(), cuda.from_numpy(v32).to(k.dtype).cuda()
            k32, v32 = k.float().cpu().numpy(), v.float().cpu().numpy()
        cache = cuda.from_numpy(before).cuda()
        assert pkg.kv_store_q4_0(cache, k, v, cuda.from_numpy(slots).cuda()) is cache
        want = stored(O, before, k32, v32, slots)
        assert np.array_equal(cache.cpu().numpy(), want)
        inside = np.where((slots >= 0) & (slots < 4 * page_tokens), slots, 0)
        keys, values = ref.decode(want[inside // page_tokens, :, inside % page_tokens // 16])
        for dtype in TYPES:
            got = pkg.kv_load_q4_0(cache, cuda.from_numpy(slots).cuda(), dtype=getattr(cuda, dtype))
            for x, w in zip(got, (keys, values)):
                w = w[np.arange(n), :, inside % 16 if page_tokens % 16 == 0 else None]
                w[(slots < 0) | (slots >= 4 * page_tokens)] = 0
                assert cuda.equal(x.cpu(), cuda.from_numpy(w).to(getattr(cuda, dtype)))
    pkg.check_device_errors()


@pytest.mark.parametrize("kind", TYPES)
def test_store_runs_of_neighbouring_slots(cuda, pkg, O, kind):
    # whole groups, and runs that begin and end inside one
    rng = np.random.default_rng(2)
    before = ref.random_cache(rng, 6, 2, 32, 64)
    slots = np.concatenate((np.arange(64, 128), np.arange(5, 30), np.arange(185, 161, -1))).astype(np.int64)
    k, k32 = rows(cuda, rng, len(slots), 2, 64, kind)
    v, v32 = rows(cuda, rng, len(slots), 2, 64, kind)
    cache = cuda.from_numpy(before).cuda()
    pkg.kv_store_q4_0(cache, k, v, cuda.from_numpy(slots).cuda())
    assert np.array_equal(cache.cpu().numpy(), stored(O, before, k32, v32, slots))


@pytest.mark.parametrize("kind", TYPES)
def test_store_strides(cuda, pkg, O, kind):
    rng = np.random.default_rng(3)
    before = ref.random_cache(rng, 2, 2, 16, 64)
    k, k32 = rows(cuda, rng, 9, 2, 64, kind)
    v, v32 = rows(cuda, rng, 9, 2, 64, kind)
    slots = np.arange(3, 12).astype(np.int64)
    both = cuda.zeros(2, 2, 9, 131, dtype=k.dtype, device="cuda")  # heads outside the rows, at odd addresses
    both[0, :, :, 1:65], both[1, :, :, 67:131] = k.transpose(0, 1), v.transpose(0, 1)
    pages = cuda.zeros(2, 3, 2, 1, 18 * 64, dtype=cuda.uint8, device="cuda")  # a layer of several
    pages[:, 2] = cuda.from_numpy(before).cuda()
    pkg.kv_store_q4_0(pages[:, 2], both[0, :, :, 1:65].transpose(0, 1), both[1, :, :, 67:131].transpose(0, 1),
                      cuda.from_numpy(slots).cuda())
    assert np.array_equal(pages[:, 2].cpu().numpy(), stored(O, before, k32, v32, slots))
    assert not bool(pages[:, :2].any())


def test_store_and_load_of_nothing(cuda, pkg):
    cache = pkg.kv_cache_q4_0(2, 1, 16, 64)
    none = cuda.empty(0, dtype=cuda.int64, device="cuda")
    pkg.kv_store_q4_0(cache, cuda.empty(0, 1, 64, device="cuda"), cuda.empty(0, 1, 64, device="cuda"), none)
    k, v = pkg.kv_load_q4_0(cache, none)
    assert k.shape == v.shape == (0, 1, 64) and not bool(cache.any())


def test_store_and_load_refusals(cuda, pkg):
    cache = pkg.kv_cache_q4_0(2, 2, 16, 64)
    x, slots = cuda.zeros(3, 2, 64, device="cuda"), cuda.tensor([0, 1, 2], device="cuda")
    def bad(error, call, *a):
        with pytest.raises(error):
            call(*a)
    store = pkg.kv_store_q4_0
    bad(TypeError, store, cache, x.double(), x.double(), slots)
    bad(TypeError, store, cache, x, x.half(), slots)
    bad(TypeError, store, cache, x, x, slots.int())
    bad(ValueError, store, cache, x, x, slots[:2])
    bad(ValueError, store, cache, x[:, :1], x[:, :1], slots)
    bad(ValueError, store, cache, x[..., ::2], x[..., ::2], slots)
    bad(ValueError, store, cache.view(2, 2, -1), x, x, slots)
    bad(ValueError, store, cache[..., :-32], x, x, slots)
    bad(TypeError, store, cache.cpu(), x, x, slots)
    bad(TypeError, pkg.kv_load_q4_0, cache, slots, cuda.float64)
    bad(TypeError, pkg.kv_load_q4_0, cache, slots.int())
    for sizes in ((2, 2, 17, 64), (2, 2, 0, 64), (2, 2, 16, 40)):
        bad(ValueError, pkg.kv_cache_q4_0, *sizes)


# ------------------------------------------------------------------ plan


def plan_case(torch, pkg, context, new, page_tokens, rows, width, free, free_count, table):
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    t = ints(table).reshape(len(context), width)
    got = pkg.kv_plan(ints(context), ints(new), t, ints(free), ints([free_count]), page_tokens, rows)
    want, want_table = ref.plan(context, new, np.array(table, np.int32).reshape(len(context), width), free, free_count, page_tokens, rows)
    for name, x, w in zip(("first_rows", "kv_lens", "slots", "positions", "requests", "info"), got, want):
        assert np.array_equal(x.cpu().numpy(), w) and x.cpu().numpy().dtype == w.dtype, name
    assert np.array_equal(t.cpu().numpy(), want_table)
    return got


@pytest.mark.parametrize("n,page_tokens,prompt", [(0, 16, 1), (1, 16, 1), (1, 64, 5000), (7, 16, 40), (64, 32, 1), (1000, 16, 3),
                                                  (1025, 32, 9), (3000, 16, 2), (40, 16, 2000), (16384, 16, 1)])
def test_plan(cuda, pkg, n, page_tokens, prompt):
    rng = np.random.default_rng(n + prompt)
    context = [int(x) for x in rng.integers(0, 100, n)]
    new = [int(x) for x in rng.integers(0, prompt + 1, n)]
    width = -(-(100 + prompt) // page_tokens)
    held = [-(-c // page_tokens) for c in context]
    order = rng.permutation(n * width + 5)
    table, used = np.full((n, width), -1, np.int64), 0
    for r, h in enumerate(held):
        table[r, :h] = order[used:used + h]
        used += h
    free = [int(x) for x in order[used:]] + [123456789] * 4
    got = plan_case(cuda, pkg, context, new, page_tokens, sum(new) + 3, width, free, len(free) - 4, table.tolist())
    assert int(got.info[0]) == 0


def test_plan_boundaries(cuda, pkg):
    # contexts that end with a page, a request that fills its table, exactly enough pages and rows
    plan_case(cuda, pkg, [16, 15, 0, 47], [1, 1, 16, 1], 16, 19, 3, [9, 8], 2, [[0, -1, -1], [1, -1, -1], [-1, -1, -1], [3, 4, 5]])


@pytest.mark.parametrize("n", [4, 3000])
def test_plan_that_cannot_be_done_takes_nothing(cuda, pkg, n):
    context, new, table = [10] * n, [7] * n, [[1, -1]] * n
    free = list(range(n + 2))
    plan_case(cuda, pkg, context, new, 16, 7 * n, 2, free, n - 1, table)                  # 1: one page short
    plan_case(cuda, pkg, [10] * (n - 1) + [30], new, 16, 7 * n, 2, free, n, table)        # 2: a table that is too narrow
    plan_case(cuda, pkg, context, new, 16, 7 * n - 1, 2, free, n, table)                  # 3: a row short
    plan_case(cuda, pkg, [10] * (n - 1) + [-1], new, 16, 7 * n, 2, free, n, table)        # 4
    plan_case(cuda, pkg, context, [7] * (n - 1) + [-1], 16, 7 * n, 2, free, n, table)     # 4
    plan_case(cuda, pkg, context, new, 16, 7 * n, 2, free, n + 3, table)                  # 4: more pages than the list has
    plan_case(cuda, pkg, context, new, 16, 7 * n, 2, free, -1, table)                     # 4
    # sums beyond 32 bits
    plan_case(cuda, pkg, [0] * n, [2147483647] * n, 16, 5, 2, free, n, table)


def test_plan_in_a_captured_loop(cuda, pkg):
    # the free count goes from one step's info to the next's; a replay is a step
    n, page_tokens, width = 5, 16, 4
    ints = lambda x: cuda.tensor(x, dtype=cuda.int32, device="cuda")  # noqa: E731
    context, new, table = ints([0, 3, 15, 16, 40]), ints([1, 2, 1, 1, 0]), ints(np.full((n, width), -1))
    table[1, 0], table[2, 0], table[3, 0], table[4, :3] = 0, 1, 2, ints([3, 4, 5])
    free = ints(range(6, 30))
    plan = pkg.kv_plan(context, ints([0] * n), table, free, ints([24]), page_tokens, 6)
    assert plan.info.tolist() == [0, 0, 0, 24]
    state, want_table, left = [0, 3, 15, 16, 40], table.cpu().numpy(), 24
    cuda.cuda.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        again = pkg.kv_plan(context, new, table, free, plan.info[3:4], page_tokens, 6, out=plan)
        context.copy_(again.kv_lens)
    for _ in range(12):
        graph.replay()
        want, want_table = ref.plan(state, [1, 2, 1, 1, 0], want_table, list(range(6, 30)), left, page_tokens, 6)
        state, left = [int(x) for x in want[1]], int(want[5][3])
        for x, w in zip(plan, want):
            assert np.array_equal(x.cpu().numpy(), w)
        assert np.array_equal(table.cpu().numpy(), want_table)


@pytest.mark.parametrize("n", [7, 3000])
def test_plan_that_replaces_its_own_inputs(cuda, pkg, n):
    # the lengths and the free count of one step are the next one's, in the same buffers
    rng = np.random.default_rng(n)
    ints = lambda x: cuda.tensor(x, dtype=cuda.int32, device="cuda")  # noqa: E731
    width, rows = 8, 4 * n
    state, left, table = [0] * n, 8 * n, np.full((n, width), -1, np.int32)
    free = [int(x) for x in rng.permutation(8 * n)]
    t, f = ints(table), ints(free)
    plan = pkg.kv_plan(ints(state), ints(state), t, f, ints([left]), 16, rows)
    for step in range(6):
        new = [int(x) for x in rng.integers(0, 5, n)] if step != 3 else [200] * n  # (once what cannot be done)
        pkg.kv_plan(plan.kv_lens, ints(new), t, f, plan.info[3:4], 16, rows, out=plan)
        want, table = ref.plan(state, new, table, free, left, 16, rows)
        for x, w in zip(plan, want):
            assert np.array_equal(x.cpu().numpy(), w)
        assert np.array_equal(t.cpu().numpy(), table)
        state, left = [int(x) for x in want[1]], int(want[5][3])


def test_plan_refusals(cuda, pkg):
    ints = lambda x: cuda.tensor(x, dtype=cuda.int32, device="cuda")  # noqa: E731
    ok = [ints([1, 2]), ints([1, 1]), ints([[0, 1], [2, 3]]), ints([4]), ints([1]), 16, 2]
    def bad(error, at, value, **k):
        a = list(ok)
        a[at] = value
        with pytest.raises(error):
            pkg.kv_plan(*a, **k)
    bad(ValueError, 0, ints([1]))
    bad(TypeError, 0, cuda.tensor([1, 2], device="cuda"))
    bad(ValueError, 1, ints([1, 2, 3, 4])[::2])
    bad(ValueError, 2, ints([0, 1]))
    bad(ValueError, 2, ints([[0, 1], [2, 3]]).t())
    bad(ValueError, 4, ints([1, 1]))
    bad(ValueError, 5, 0)
    bad(ValueError, 6, -1)
    bad(TypeError, 0, cuda.tensor([1, 2], dtype=cuda.int32))
    plan = pkg.kv_plan(*ok)
    bad(ValueError, 6, 3, out=plan)
    many = cuda.zeros(16385, dtype=cuda.int32, device="cuda")
    with pytest.raises(pkg.TcrvCudaError):
        pkg.kv_plan(many, many, many[:, None], ints([4]), ints([1]), 16, 2)
