"""Attention over the paged Q4_0 cache: small values, values of many magnitudes side by side, values that are no numbers."""
import numpy as np
import pytest

import attention_rms as rms
import paged_reference as ref

pytestmark = pytest.mark.gpu

HALF = ["float16", "bfloat16"]


def tensor(torch, x, kind):
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, kind))
    return t.cuda(), t.double().numpy()


def ints(torch, x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")


def build(rng, lens, kv_heads, page_tokens, dim, keys, values):
    """(cache, table) whose key and value scales are keys(r, shape) and values(r, shape) of request r, shape (kv_heads, tokens, dim / 32); any quants."""
    table, pages = ref.tables(rng, lens, page_tokens)
    lead = (pages, kv_heads, page_tokens // 16)
    quants = rng.integers(0, 16, (2,) + lead + (16, dim), dtype=np.uint8)
    scales = np.zeros((2,) + lead + (16, dim // 32))
    for r, n in enumerate(lens):
        held = -(-n // page_tokens)
        for part, of in enumerate((keys, values)):
            s = of(r, (kv_heads, held * page_tokens, dim // 32)).reshape(kv_heads, held, page_tokens // 16, 16, dim // 32)
            scales[part][table[r, :held]] = s.transpose(1, 0, 2, 3, 4)
    return ref.encode(quants, scales.astype(np.float16)), table


def call(torch, pkg, q, cache, table, lens, first, **k):
    return pkg.attention_q4_0(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table.astype(np.int32)).cuda(), ints(torch, lens),
                              first_rows=ints(torch, first), max_new=int(np.diff(first).max()), with_lse=True, **k)


def ordinary(rng):
    return lambda r, shape: rng.uniform(0.02, 0.3, shape) * rng.choice((-1.0, 1.0), shape)


def few_rows(torch, pkg, kind, lens, new, heads, kv_heads, dim, values, seed=0, sink=None, page_tokens=32, prompt=False):
    rng = np.random.default_rng(seed)
    cache, table = build(rng, lens, kv_heads, page_tokens, dim, ordinary(rng), values(rng))
    first = np.concatenate(([0], np.cumsum(new)))
    x = rng.standard_normal((first[-1], heads, dim))
    if sink is not None:  # one token `sink` above the rest: its key is along every query of its head
        toward = rng.standard_normal((kv_heads, dim))
        x = np.repeat(toward, heads // kv_heads, 0)[None] + 0.05 * x
        key, _, shift, kd, _ = ref.places(dim)
        quants, size = np.clip(np.rint(toward / 0.4) + 8, 0, 15).astype(np.uint8), 0.4
        size = sink / (dim ** -0.5 * ((quants - 8.0) * toward).sum(-1))  # its score
        for r in range(len(lens)):
            for h in range(kv_heads):
                group, token = cache[table[r, 0], h, 0], 5
                for d in range(dim):
                    group[key[token, d]] = group[key[token, d]] & (0xf0 >> shift[token, d]) | quants[h, d] << shift[token, d]
                group[np.add.outer(kd[token], np.arange(2))] = np.array([size[h]], np.float16).view(np.uint8)
    q, q64 = tensor(torch, x, kind)
    got, lse = call(torch, pkg, q, cache, table, lens, first)
    pkg.check_device_errors()
    d = rms.definition(q64, cache, table, lens, first, dim ** -0.5)
    rms.check(got, lse, d, kind, prompt)


@pytest.mark.parametrize("kind", HALF + ["float32"])
@pytest.mark.parametrize("spread", [1.0, 1e-2, 1e-3, 1e-4, 1e-5])
def test_small_values_of_few_rows(cuda, pkg, kind, spread):
    few_rows(cuda, pkg, kind, [2900, 70], [1, 1], 8, 2, 128, lambda rng: lambda r, s: ordinary(rng)(r, s) * spread, seed=1)


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("dim,heads,new", [(64, 4, [5, 3]), (96, 4, [1, 2]), (128, 12, [5, 1]), (192, 4, [1, 5]), (256, 2, [9, 2])])
def test_small_values_of_every_head_size(cuda, pkg, kind, dim, heads, new):
    few_rows(cuda, pkg, kind, [1500, 300], new, heads, 1, dim, lambda rng: lambda r, s: ordinary(rng)(r, s) * 1e-4, seed=dim)


@pytest.mark.parametrize("kind", HALF + ["float32"])
@pytest.mark.parametrize("spread", [1.0, 1e-1, 1e-2, 1e-3])
def test_one_token_above_the_rest(cuda, pkg, kind, spread):
    # the heavy token's values are a hundredth of the others'
    def values(rng):
        def of(r, shape):
            s = ordinary(rng)(r, shape) * spread
            s[:, 5] *= 0.01
            return s
        return of
    few_rows(cuda, pkg, kind, [2900, 700], [1, 1], 8, 2, 128, values, seed=2, sink=8.0)


@pytest.mark.parametrize("kind", HALF + ["float32"])
def test_values_that_grow_along_the_context(cuda, pkg, kind):
    # the largest scale seen moves again and again, up to fp16's largest
    few_rows(cuda, pkg, kind, [1400], [1], 4, 1, 128,
             lambda rng: lambda r, s: ordinary(rng)(r, s) * np.exp(np.linspace(np.log(2e-6), np.log(2e5), s[1]))[None, :, None], seed=3)


@pytest.mark.parametrize("kind", HALF + ["float32"])
def test_values_of_zero(cuda, pkg, kind):
    # no scale at all in the first request, one token's in the second
    def values(rng):
        def of(r, shape):
            s = np.zeros(shape)
            if r:
                s[:, 33] = 1e-3
            return s
        return of
    few_rows(cuda, pkg, kind, [100, 100], [1, 2], 4, 2, 64, values, seed=4)


# prompts: rows enough for the kernel whose operands are fp16


def prompt_case(torch, pkg, kind, n, new, heads, kv_heads, dim, keys, values, seed, window=0, std=1.0):
    """(definition, got, lse) of one request."""
    rng = np.random.default_rng(seed)
    cache, table = build(rng, [n], kv_heads, 32, dim, keys(rng), values(rng))
    q, q64 = tensor(torch, rng.standard_normal((new, heads, dim)) * std, kind)
    got, lse = call(torch, pkg, q, cache, table, [n], [0, new], window=window)
    pkg.check_device_errors()
    return rms.definition(q64, cache, table, [n], [0, new], dim ** -0.5, window), got, lse


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("n,new,dim", [(700, 400, 128), (1500, 33, 128), (300, 300, 64), (4000, 40, 64)])
def test_prompts_on_average(cuda, pkg, kind, n, new, dim):
    d, got, lse = prompt_case(cuda, pkg, kind, n, new, 4, 2, dim, ordinary, ordinary, seed=n)
    rms.check(got, lse, d, kind, True)


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("n,new,dim,window", [(60, 60, 128, 0), (400, 300, 128, 6), (17, 17, 64, 0), (3000, 40, 64, 3), (700, 128, 128, 0)])
def test_the_soft_max_sum_of_prompts_is_f32(cuda, pkg, kind, n, new, dim, window):
    """The result is 16 bits wide, its logarithm of the sum is not: keys count with all the bits of scale times quant.
    A score is a sum of up to 2 * 8 steps of 16 products and the sum so far, each aligned and cut at 2^-24 of the largest: 272 cuts,
    of terms and partial sums the size of the root of the terms' squares.  2^-18 allows for 2^x, the sum's additions and the logarithm."""
    d, got, lse = prompt_case(cuda, pkg, kind, n, new, 8, 2, dim, ordinary, ordinary, seed=n, window=window)
    rms.check(got, lse, d, kind, True)
    off = lse.double().cpu().numpy() - d["lse"]
    allowed = 272 * 2.0 ** -24 * d["spread"] + 2.0 ** -18 + np.abs(d["lse"]) * 2.0 ** -22
    ratio = ((off / allowed) ** 2).mean()
    assert ratio <= 1, f"mean square error of lse {ratio:.3g} of the allowed"


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("n,new,dim", [(700, 400, 128), (1500, 33, 128), (300, 300, 64)])
def test_prompts_without_the_sum(cuda, pkg, kind, n, new, dim):
    rng = np.random.default_rng(n)
    cache, table = build(rng, [n], 2, 32, dim, ordinary(rng), ordinary(rng))
    q, q64 = tensor(cuda, rng.standard_normal((new, 4, dim)), kind)
    got = pkg.attention_q4_0(q, cuda.from_numpy(cache).cuda(), cuda.from_numpy(table.astype(np.int32)).cuda(), ints(cuda, [n]),
                             first_rows=ints(cuda, [0, new]), max_new=new)
    pkg.check_device_errors()
    rms.check(got, None, rms.definition(q64, cache, table, [n], [0, new], dim ** -0.5), kind, True)


@pytest.mark.parametrize("n,new,dim", [(200, 150, 128), (90, 90, 64), (2000, 34, 128)])
def test_values_of_fp16_prompts_are_whole(cuda, pkg, n, new, dim):
    """Keys of zero and a window of 16: weights of 1, sums and a sixteenth of them without rounding, so that a result is the mean of 16
    values rounded once."""
    none = lambda rng: lambda r, shape: np.zeros(shape)  # noqa: E731
    d, got, lse = prompt_case(cuda, pkg, "float16", n, new, 4, 2, dim, none, ordinary, seed=n, window=16)
    full = max(0, 15 - (n - new))  # rows from here on see 16 tokens
    assert np.array_equal(got[full:].cpu().numpy(), d["out"][full:].astype(np.float32).astype(np.float16))
    assert (np.abs(lse[full:].cpu().numpy() - np.log(16)) <= 2.0 ** -21).all()


SMALL = {"float16": (6.2e-5, 1e-4), "bfloat16": (1e-5, 2e-5)}  # (a scale below 2^-14 times a quant is a whole number of fp16's steps)


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("n,new", [(260, 200), (2100, 40)])
def test_prompts_with_large_scales_beside_small_ones(cuda, pkg, kind, n, new):
    """Block 0 of a value has scales of 0.13 and 2.1, block 1 of 1e-4 or less, in the same group of tokens."""
    def values(rng):
        def of(r, shape):
            s = rng.uniform(*SMALL[kind], shape)
            s[..., 0] = np.where(np.arange(shape[1]) % 2, 0.13, 2.1)
            return s
        return of
    d, got, lse = prompt_case(cuda, pkg, kind, n, new, 8, 2, 64, ordinary, values, seed=n, window=8)
    rms.check(got, lse, d, kind, True)
    rms.check(got, None, d, kind, True, where=np.broadcast_to(np.arange(64) >= 32, got.shape))


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("part", ["keys", "values"])
@pytest.mark.parametrize("n", [48, 2096])
def test_prompts_before_a_token_that_leaves_fp16(cuda, pkg, kind, part, n):
    """The last token has scales of 2^13 and more, so that its values leave fp16; rows before it see the small ones beside it as they are."""
    def large(rng):
        def of(r, shape):
            s = rng.uniform(*SMALL[kind], shape)
            s[:, n - 1] = rng.uniform(8192, 60000, shape[2])
            return s
        return of
    keys, values = (large, ordinary) if part == "keys" else (ordinary, large)
    d, got, lse = prompt_case(cuda, pkg, kind, n, 40, 8, 1, 64, keys, values, seed=n, window=8, std=1e4 if part == "keys" else 1.0)
    near = np.zeros(got.shape, bool)
    near[31:39] = True  # rows that see this group's tokens only, and not the last one
    d["lse"][~near[..., 0]] = np.nan
    rms.check(got, lse, d, kind, True, where=near)


@pytest.mark.parametrize("kind", HALF)
def test_prompts_with_tokens_that_leave_fp16(cuda, pkg, kind):
    """Keys and values of 2^13 and more here and there, seen by all rows."""
    def few(rng):
        def of(r, shape):
            s = ordinary(rng)(r, shape)
            s[:, 7::50] = rng.uniform(8192, 60000, s[:, 7::50].shape)
            return s
        return of
    d, got, lse = prompt_case(cuda, pkg, kind, 300, 60, 2, 1, 64, few, few, seed=9, std=2e-5)
    if kind == "float16":
        d["out"][np.abs(d["out"]).max(-1) > 6e4] = np.nan  # (a result that its type does not hold)
    rms.check(got, lse, d, kind, True)


@pytest.mark.parametrize("n,new,kind", [(300, 250, "bfloat16"), (300, 250, "float16"), (2500, 40, "bfloat16"), (300, 3, "bfloat16"), (300, 3, "float32")])
def test_a_value_scale_that_is_no_number_reaches_its_block_only(cuda, pkg, n, new, kind):
    """Rows that see the token have no numbers in the 32 elements of the block; everything else, the soft-max sum too, is as without it."""
    rng = np.random.default_rng(n)
    cache, table = build(rng, [n], 2, 16, 128, ordinary(rng), ordinary(rng))
    q, q64 = tensor(cuda, rng.standard_normal((new, 4, 128)), kind)
    d = rms.definition(q64, cache, table, [n], [0, new], 128 ** -0.5)
    _, _, _, _, vd = ref.places(128)
    prompt = new * 2 > 32
    for bits in (0x7c00, 0xfc00, 0x7e00):
        for token, block in ((n - 20, 0), (60, 3), (n - 1, 2)):
            spoiled = cache.copy()
            spoiled[table[0, token // 16], 1, 0, vd[token % 16, block]] = bits & 255
            spoiled[table[0, token // 16], 1, 0, vd[token % 16, block] + 1] = bits >> 8
            got, lse = call(cuda, pkg, q, spoiled, table, [n], [0, new])
            reached = np.zeros(got.shape, bool)
            reached[max(0, token - (n - new)):, 2:, 32 * block:32 * block + 32] = True
            assert not np.isfinite(got.float().cpu().numpy()[reached]).any()
            rms.check(got, lse, d, kind, prompt, where=~reached)


@pytest.mark.parametrize("new", [1, 4, 30])
def test_values_that_no_row_sees_do_not_matter(cuda, pkg, new):
    """f32: tokens before the window with the largest scales there are, among values of 1e-5."""
    rng = np.random.default_rng(new)
    n, window = 213, 40
    first = n - new - window + 1  # the first token that a row sees
    def values(r, shape):
        s = rng.uniform(2e-6, 1e-5, shape)
        s[:, :first] = 6e4
        return s
    cache, table = build(rng, [n], 1, 16, 64, ordinary(rng), values)
    q, q64 = tensor(cuda, rng.standard_normal((new, 2, 64)), "float32")
    got, lse = call(cuda, pkg, q, cache, table, [n], [0, new], window=window)
    d = rms.definition(q64, cache, table, [n], [0, new], 64 ** -0.5, window)
    rms.check(got, lse, d, "float32")
