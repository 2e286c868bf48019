"""Attention over the paged Q4_0 cache against its definition in 64 bits."""
import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def as_type(torch, x, kind):
    """The values of a numpy array in a type: (CUDA tensor, the same values in 64 bits)."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, kind))
    return t.cuda(), t.double().numpy()


def check(got, lse, want, want_lse, weight, kind, spread=1.0, prompt=False):
    bound, lse_bound = ref.attention_bounds(want, want_lse, weight, kind, 0.3 * spread, prompt)
    got = got.double().cpu().numpy()
    rows = ~np.isnan(want).any((1, 2))
    off = np.abs(got[rows] - want[rows])
    assert np.isfinite(got[rows]).all()
    assert (off <= bound[rows]).all(), f"off by {(off / bound[rows]).max():.3g} bounds, {off.max():.3g}"
    if lse is not None:
        lse = lse.double().cpu().numpy()[rows]
        empty = np.isneginf(want_lse[rows])
        assert np.array_equal(np.isneginf(lse), empty)
        off = np.abs(lse[~empty] - want_lse[rows][~empty])
        assert (off <= lse_bound[rows][~empty]).all(), f"lse off by {off.max():.3g}"


def run_prompt(*a, **k):
    run_case(*a, prompt=True, **k)


def run_case(torch, pkg, kind, lens, new, heads, kv_heads, dim, page_tokens, window=0, scale=None, seed=0, spread=1.0, q_std=1.0, prompt=None):
    prompt = prompt or kind != "float32" and dim in (64, 128) and max(new) * heads // kv_heads > 32
    rng = np.random.default_rng(seed)
    table, pages = ref.tables(rng, lens, page_tokens)
    cache = ref.random_cache(rng, pages, kv_heads, page_tokens, dim, spread)
    first = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    q, q64 = as_type(torch, rng.standard_normal((first[-1], heads, dim)) * q_std, kind)
    got, lse = pkg.attention_q4_0(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                                  torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  first_rows=torch.from_numpy(first).cuda(), max_new=max(new), scale=scale, window=window,
                                  with_lse=True)
    pkg.check_device_errors()
    want, want_lse, weight = ref.attention(q64, cache, table, lens, first, dim ** -0.5 if scale is None else scale, window)
    check(got, lse, want, want_lse, weight, kind, spread, prompt)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_one_token_per_request(cuda, pkg, kind, dim):
    # lengths around the groups, units and pages, one of them long enough to be split
    run_case(cuda, pkg, kind, [1, 15, 16, 17, 31, 33, 64, 100, 2500], [1] * 9, 8, 2, dim, 32, seed=dim)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (16, 2), (33, 1), (64, 2)])
def test_head_layouts(cuda, pkg, kind, heads, kv_heads):
    run_case(cuda, pkg, kind, [5, 200, 77], [1, 1, 1], heads, kv_heads, 64, 16, seed=heads)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,new", [(128, [5, 1, 3, 2]), (64, [17, 40, 1, 33]), (256, [9, 2, 16, 1]), (128, [70, 3, 129, 64])])
def test_several_new_tokens(cuda, pkg, kind, dim, new):
    run_case(cuda, pkg, kind, [new[0], 90, 300, 64], new, 4, 2, dim, 16, seed=sum(new))


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [1, 7, 32, 100, 100000])
def test_windows(cuda, pkg, kind, window):
    run_case(cuda, pkg, kind, [1, 40, 333, 700], [1, 4, 6, 1], 6, 2, 128, 64, window=window, seed=window)


@pytest.mark.parametrize("kind", TYPES)
def test_rows_that_see_nothing(cuda, pkg, kind):
    # an empty context, one shorter than its new rows (its first rows lie before the first token), an idle request
    run_case(cuda, pkg, kind, [0, 2, 50, 0], [2, 5, 1, 0], 4, 2, 64, 16, seed=3)


@pytest.mark.parametrize("kind", ["float32", "float16"])
def test_long_contexts_are_split_and_joined(cuda, pkg, kind):
    run_case(cuda, pkg, kind, [20000, 9, 4097], [1, 1, 1], 4, 1, 128, 64, seed=11)


@pytest.mark.parametrize("kind", TYPES)
def test_many_short_requests(cuda, pkg, kind):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 120, 300)]
    new = [int(x) for x in rng.integers(0, 3, 300)]
    run_case(cuda, pkg, kind, lens, new, 4, 2, 64, 16, seed=6)


@pytest.mark.parametrize("spread,q_std,scale", [(1e-3, 1e-6, 3e3), (2e5, 1e-3, 1e-6), (1.0, 3e4, 1e-4), (1.0, 20.0, None), (1.0, 1.0, -0.2)])
def test_magnitudes_f32(cuda, pkg, spread, q_std, scale):
    # scales near both ends of fp16, queries far from 1, a peaked soft-max, a negative scale
    run_case(cuda, pkg, "float32", [300, 40], [1, 2], 4, 2, 128, 16, scale=scale, spread=spread, q_std=q_std, seed=8)


# prompts: rows enough for the kernel whose operands are fp16 (16-bit calls, head sizes 64 and 128)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 1, 128), (7, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("lens,new", [([100], [100]), ([700, 5, 129, 40], [300, 1, 129, 2]), ([1500, 260], [33, 260])])
def test_prompts(cuda, pkg, kind, heads, kv_heads, dim, lens, new):
    run_prompt(cuda, pkg, kind, lens, new, heads, kv_heads, dim, 32, seed=heads + len(lens))


@pytest.mark.parametrize("window", [1, 50, 128, 300])
def test_prompts_with_windows(cuda, pkg, window):
    run_prompt(cuda, pkg, "bfloat16", [700, 90], [400, 90], 4, 2, 128, 16, window=window, seed=window)


def test_prompts_longer_than_their_context(cuda, pkg):
    run_prompt(cuda, pkg, "float16", [20, 0, 300], [200, 140, 129], 2, 1, 128, 64, seed=1)


@pytest.mark.parametrize("spread,q_std,scale", [(1e-3, 1.0, None), (2e5, 1e-6, None), (1.0, 3e4, 1e-5), (1.0, 20.0, None), (1.0, 1.0, -0.2)])
def test_prompts_magnitudes(cuda, pkg, spread, q_std, scale):
    run_prompt(cuda, pkg, "bfloat16", [300, 140], [100, 140], 4, 2, 64, 16, scale=scale, spread=spread, q_std=q_std, seed=8)


def test_prompts_with_bad_values(cuda, pkg):
    """Scales that are no numbers: behind the context they do not matter, in it they reach the rows that see their token only."""
    rng = np.random.default_rng(4)
    n, new = 300, 250
    table, pages = ref.tables(rng, [n], 16)
    table = np.concatenate((table, np.full((1, 3), -1, np.int32)), 1)
    cache = ref.random_cache(rng, pages, 1, 16, 64)
    q, _ = as_type(cuda, rng.standard_normal((new, 2, 64)), "bfloat16")
    first, lens = cuda.tensor([0, new], dtype=cuda.int32, device="cuda"), cuda.tensor([n], dtype=cuda.int32, device="cuda")
    t = cuda.from_numpy(table).cuda()
    want = pkg.attention_q4_0(q, cuda.from_numpy(cache).cuda(), t, lens, first_rows=first, max_new=new)
    _, _, _, kd, vd = ref.places(64)
    for bits in (0x7c00, 0x7e00, 0xfc00):  # infinities, NaN
        for at in (kd, vd):
            for token in (300, 303, 280, 60):  # two behind the last token (in its page), two that some rows see
                spoiled = cache.copy()
                page = spoiled[table[0, token // 16], :, 0]
                page[:, at[token % 16]], page[:, at[token % 16] + 1] = bits & 255, bits >> 8
                got = pkg.attention_q4_0(q, cuda.from_numpy(spoiled).cuda(), t, lens, first_rows=first, max_new=new)
                sees = max(0, min(new, token - (n - new)))  # rows before this one do not see the token
                assert cuda.equal(got[:sees], want[:sees])
                assert not bool(cuda.isfinite(got[sees:].float()).all(-1).any())


def test_a_page_outside_the_cache_inside_a_prompt(cuda, pkg):
    rng = np.random.default_rng(14)
    table, pages = ref.tables(rng, [300], 16)
    cache = ref.random_cache(rng, pages, 1, 16, 128)
    table[0, 3], table[0, 15] = -3, pages + 5
    q, q64 = as_type(cuda, rng.standard_normal((200, 2, 128)), "float16")
    got, lse = pkg.attention_q4_0(q, cuda.from_numpy(cache).cuda(), cuda.from_numpy(table).cuda(), cuda.tensor([300], dtype=cuda.int32, device="cuda"),
                                  first_rows=cuda.tensor([0, 200], dtype=cuda.int32, device="cuda"), max_new=200, with_lse=True)
    want, want_lse, weight = ref.attention(q64, cache, table, [300], [0, 200], 128 ** -0.5)
    check(got, lse, want, want_lse, weight, "float16", prompt=True)


def test_prompts_strides_streams_and_graphs(cuda, pkg):
    rng = np.random.default_rng(15)
    lens64, new = [400, 300], [150, 300]
    table, pages = ref.tables(rng, lens64, 16)
    cache, t = cuda.from_numpy(ref.random_cache(rng, pages, 2, 16, 64)).cuda(), cuda.from_numpy(table).cuda()
    q, _ = as_type(cuda, rng.standard_normal((sum(new), 4, 64)), "bfloat16")
    first, lens = cuda.tensor([0, 150, 450], dtype=cuda.int32, device="cuda"), cuda.tensor(lens64, dtype=cuda.int32, device="cuda")
    call = lambda x, **k: pkg.attention_q4_0(x, cache, t, lens, first_rows=first, max_new=300, **k)  # noqa: E731
    want = call(q)
    wide = cuda.zeros(450, 5, 67, dtype=q.dtype, device="cuda")
    wide[:, 1:, 1:65] = q
    out = cuda.full((4, 451, 70), 9.0, dtype=q.dtype, device="cuda")
    call(wide[:, 1:, 1:65], out=out[:, :450, 3:67].transpose(0, 1))
    assert cuda.equal(out[:, :450, 3:67].transpose(0, 1), want)
    assert bool((out[..., :3] == 9).all()) and bool((out[..., 67:] == 9).all()) and bool((out[:, 450] == 9).all())
    streams, results = [cuda.cuda.Stream() for _ in range(2)], []
    cuda.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with cuda.cuda.stream(s):
                results.append(call(q))
    cuda.cuda.synchronize()
    assert all(cuda.equal(x, want) for x in results)
    static = cuda.empty_like(q)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        call(q, out=static)
    graph.replay()
    cuda.cuda.synchronize()
    assert cuda.equal(static, want)
    lens.copy_(cuda.tensor([200, 310], dtype=cuda.int32))
    first.copy_(cuda.tensor([0, 2, 302], dtype=cuda.int32))  # one request falls to the other kernel
    graph.replay()
    cuda.cuda.synchronize()
    assert cuda.equal(static[:302], call(q)[:302])


def operands(torch, kind="bfloat16", lens=(50, 70, 20), heads=4, kv_heads=2, dim=64, page_tokens=16, seed=21):
    rng = np.random.default_rng(seed)
    table, pages = ref.tables(rng, lens, page_tokens)
    cache = ref.random_cache(rng, pages, kv_heads, page_tokens, dim)
    q, q64 = as_type(torch, rng.standard_normal((len(lens), heads, dim)), kind)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), lens_t, (q64, cache, table, list(lens))


def test_bad_values_behind_a_context_do_not_matter(cuda, pkg):
    for kind in TYPES:
        q, cache, table, lens, _ = operands(cuda, kind)
        want = pkg.attention_q4_0(q, cache, table, lens)
        spoiled = cache.cpu().numpy().copy()
        key, value, shift, kd, vd = ref.places(64)
        nan = np.array([np.nan, np.inf], np.float16).view(np.uint8).reshape(2, 2)
        for r, n in enumerate([50, 70, 20]):  # NaN and infinity as the scales of the tokens behind the last one
            page, token = int(table[r, n // 16]), n % 16
            for tok in range(token, 16):
                for at in (kd, vd):
                    spoiled[page, :, 0][:, at[tok]] = nan[tok % 2, 0]
                    spoiled[page, :, 0][:, at[tok] + 1] = nan[tok % 2, 1]
        got = pkg.attention_q4_0(q, cuda.from_numpy(spoiled).cuda(), table, lens)
        assert cuda.equal(got, want)


def test_bad_values_of_a_later_token_do_not_reach_earlier_rows(cuda, pkg):
    rng = np.random.default_rng(4)
    for kind in TYPES:
        table, pages = ref.tables(rng, [20], 16)
        cache = ref.random_cache(rng, pages, 1, 16, 64)
        q, _ = as_type(cuda, rng.standard_normal((3, 4, 64)), kind)
        first, lens = cuda.tensor([0, 3], dtype=cuda.int32, device="cuda"), cuda.tensor([20], dtype=cuda.int32, device="cuda")
        t = cuda.from_numpy(table).cuda()
        want = pkg.attention_q4_0(q, cuda.from_numpy(cache).cuda(), t, lens, first_rows=first, max_new=3)
        _, _, _, kd, vd = ref.places(64)
        for bits in (0x7c00, 0x7e00):  # infinity, NaN
            spoiled = cache.copy()
            for at in (kd, vd):  # the last token's scales
                spoiled[table[0, 1], :, 0][:, at[3]], spoiled[table[0, 1], :, 0][:, at[3] + 1] = bits & 255, bits >> 8
            got = pkg.attention_q4_0(q, cuda.from_numpy(spoiled).cuda(), t, lens, first_rows=first, max_new=3)
            assert cuda.equal(got[:2], want[:2])
            assert not bool(cuda.isfinite(got[2].float()).all())


def test_pages_outside_the_cache_count_as_unseen(cuda, pkg):
    q, cache, table, lens, (q64, cache64, table64, lens64) = operands(cuda, "float32")
    table64 = table64.copy()
    table64[1, 1], table64[2, 0] = 1 << 30, -5
    got, lse = pkg.attention_q4_0(q, cache, cuda.from_numpy(table64).cuda(), lens, with_lse=True)
    want, want_lse, weight = ref.attention(q64, cache64, table64, lens64, list(range(4)), 64 ** -0.5)
    check(got, lse, want, want_lse, weight, "float32")


def test_lengths_beyond_the_table_and_negative_ones(cuda, pkg):
    q, cache, table, _, (q64, cache64, table64, _) = operands(cuda, "float32")
    lens64 = [1 << 30, -7, 20]
    table64 = np.where(table64 < 0, 0, table64).astype(np.int32)
    got, lse = pkg.attention_q4_0(q, cache, cuda.from_numpy(table64).cuda(), cuda.tensor(lens64, dtype=cuda.int32, device="cuda"), with_lse=True)
    want, want_lse, weight = ref.attention(q64, cache64, table64, lens64, list(range(4)), 64 ** -0.5)
    check(got, lse, want, want_lse, weight, "float32")


def test_rows_of_no_request_are_left_alone(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda)
    q = cuda.cat((q, q, q))
    first = cuda.tensor([1, 2, 2, 5], dtype=cuda.int32, device="cuda")  # row 0 and rows 5.. belong to none; request 1 is idle
    out = cuda.full_like(q, 7.0)
    pkg.attention_q4_0(q, cache, table, lens, first_rows=first, max_new=3, out=out)
    assert bool((out[0] == 7).all()) and bool((out[5:] == 7).all()) and not bool((out[1:5] == 7).all(-1).any())
    # more rows than max_new says, and rows beyond the tensor: those are left out
    out = cuda.full_like(q, 7.0)
    first = cuda.tensor([-4, 3, 3, 1 << 30], dtype=cuda.int32, device="cuda")
    pkg.attention_q4_0(q, cache, table, lens, first_rows=first, max_new=2, out=out)
    cuda.cuda.synchronize()
    assert bool((out[5:] == 7).all()) and bool((out[:3] == 7).all())


def test_strides(cuda, pkg):
    for kind in TYPES:
        q, cache, table, lens, _ = operands(cuda, kind)
        want = pkg.attention_q4_0(q, cache, table, lens)
        wide = cuda.zeros(3, 5, 67, dtype=q.dtype, device="cuda")  # rows at odd addresses
        wide[:, 1:, 1:65] = q
        out = cuda.full((5, 3, 70), 9.0, dtype=q.dtype, device="cuda")  # heads outside, rows inside
        view = out[:4, :, 3:67].transpose(0, 1)
        pages = cuda.zeros(cache.shape[0], 3, *cache.shape[1:], dtype=cuda.uint8, device="cuda")  # a layer of several
        pages[:, 1] = cache
        tall = cuda.zeros(3, table.shape[1] + 3, dtype=cuda.int32, device="cuda")
        tall[:, :table.shape[1]] = table
        got = pkg.attention_q4_0(wide[:, 1:, 1:65], pages[:, 1], tall[:, :table.shape[1]], lens, out=view)
        assert got is view and cuda.equal(got, want)
        assert bool((out[4] == 9).all()) and bool((out[..., :3] == 9).all()) and bool((out[..., 67:] == 9).all())


def test_the_same_call_gives_the_same_bits(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda, "float32", lens=(3000, 70, 900))
    first = pkg.attention_q4_0(q, cache, table, lens)
    for _ in range(5):
        assert cuda.equal(pkg.attention_q4_0(q, cache, table, lens), first)


def test_captured_and_replayed_with_new_lengths(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda, "bfloat16", lens=(600, 70, 20))
    others = [cuda.tensor(x, dtype=cuda.int32, device="cuda") for x in ([600, 70, 20], [1, 0, 7], [599, 64, 16])]
    want = [pkg.attention_q4_0(q, cache, table, x) for x in others]
    out = cuda.empty_like(q)
    pkg.attention_q4_0(q, cache, table, lens, out=out)
    cuda.cuda.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        pkg.attention_q4_0(q, cache, table, lens, out=out)
    for x, w in zip(others, want):
        lens.copy_(x)
        graph.replay()
        cuda.cuda.synchronize()
        assert cuda.equal(out, w)


def test_two_streams_at_once(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda, "float32", lens=(5000, 4000, 900))
    want = pkg.attention_q4_0(q, cache, table, lens)
    cuda.cuda.synchronize()
    streams, results = [cuda.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for s, r in zip(streams, results):
            with cuda.cuda.stream(s):
                r.append(pkg.attention_q4_0(q, cache, table, lens))
    cuda.cuda.synchronize()
    assert all(cuda.equal(x, want) for r in results for x in r)


def test_a_cache_of_more_than_4_gib(cuda, pkg):
    dim, heads, page_tokens = 128, 8, 64
    pages = (1 << 32) // (heads * 4 * 18 * dim) + 40
    cache = cuda.zeros(pages, heads, 4, 18 * dim, dtype=cuda.uint8, device="cuda")
    rng = np.random.default_rng(9)
    far = ref.random_cache(rng, 3, heads, page_tokens, dim)
    cache[-3:] = cuda.from_numpy(far).cuda()
    q, q64 = as_type(cuda, rng.standard_normal((1, heads, dim)), "float32")
    table = np.array([[2, 0, 1]], np.int32)
    got, lse = pkg.attention_q4_0(q, cache, cuda.from_numpy(table + pages - 3).cuda(), cuda.tensor([150], dtype=cuda.int32, device="cuda"),
                                  with_lse=True)
    want, want_lse, weight = ref.attention(q64, far, table, [150], [0, 1], dim ** -0.5)
    check(got, lse, want, want_lse, weight, "float32")
    slots = cuda.tensor([(pages - 1) * 64 + 5], device="cuda")
    k, _ = pkg.kv_load_q4_0(cache, slots)
    assert np.array_equal(k[0].double().cpu().numpy(), ref.decode(far[2, :, 0])[0][:, 5])


def test_nothing_to_do(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda)
    out = pkg.attention_q4_0(q[:0], cache, table[:0], lens[:0])
    assert out.shape == (0, 4, 64)
    out, lse = pkg.attention_q4_0(q[:1], cache, table[:1, :0], lens[:1], with_lse=True)  # a table without pages
    assert not bool(out.any()) and bool(cuda.isneginf(lse).all())


def test_refusals(cuda, pkg):
    q, cache, table, lens, _ = operands(cuda)
    first = cuda.tensor([0, 1, 2, 3], dtype=cuda.int32, device="cuda")
    def bad(error, *a, **k):
        with pytest.raises(error):
            pkg.attention_q4_0(*a, **k)
    bad(TypeError, q.double(), cache, table, lens)
    bad(TypeError, q.cpu(), cache, table, lens)
    bad(ValueError, q[0], cache, table, lens)
    bad(ValueError, q.transpose(1, 2), cache, table, lens)
    bad(ValueError, q[:, :3], cache, table, lens)             # heads no multiple of the cache's
    bad(ValueError, q[..., :32].contiguous(), cache, table, lens)
    bad(ValueError, q, cache.float(), table, lens)
    bad(ValueError, q, cache[..., :-1], table, lens)
    bad(ValueError, q, cache.expand(-1, -1, 3, -1), table, lens)  # groups that share their bytes
    bad(ValueError, q, cache, table.long(), lens)
    bad(TypeError, q, cache, table, lens.long())
    bad(ValueError, q, cache, table, lens[:2])
    bad(ValueError, q, cache, table, lens, max_new=2)         # several rows need first_rows
    bad(ValueError, q, cache, table, lens, first_rows=first[:3])
    bad(ValueError, q, cache, table, lens, first_rows=first, max_new=0)
    bad(ValueError, q, cache, table, lens, window=-1)
    bad(ValueError, q, cache, table, lens, out=q[:2])
    bad(TypeError, q, cache, table, lens, out=q.float())
    bad(ValueError, q, cache, table, lens, out=cuda.empty(3, 1, 64, dtype=q.dtype, device="cuda").expand(3, 4, 64))
    bad(pkg.TcrvCudaError, q, cache, table, lens, workspace=cuda.empty(64, dtype=cuda.uint8, device="cuda"))
    small = cuda.zeros(2, 2, 1, 18 * 32, dtype=cuda.uint8, device="cuda")
    bad(pkg.TcrvCudaError, q[..., :32], small, table, lens)   # a head size without a kernel
    odd = cuda.zeros(cache.numel() + 1, dtype=cuda.uint8, device="cuda")[1:].view(cache.shape)
    bad(pkg.TcrvCudaError, q, odd, table, lens)               # a cache off 16-byte boundaries
