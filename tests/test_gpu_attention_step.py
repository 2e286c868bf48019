"""The operations around the paged Q4_0 cache as a serving loop uses them: each step plans pages, rotates, stores and attends."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_attention_q4_0 import check
from test_gpu_kv_cache import stored

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, WIDTH, PAGES = 4, 2, 64, 16, 8, 24


class Loop:
    """The device state of a loop over `n` requests with at most `rows` rows a step."""

    def __init__(self, torch, pkg, n, rows, kind):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.torch, self.pkg, self.rows, self.kind = torch, pkg, rows, kind
        self.cache = pkg.kv_cache_q4_0(PAGES, KV, PAGE, DIM)
        self.table, self.lens, self.new = ints(np.full((n, WIDTH), -1)), ints([0] * n), ints([0] * n)
        self.free = ints(np.random.default_rng(0).permutation(PAGES))
        self.freqs = pkg.rope_frequencies(DIM, scaling="yarn", factor=4.0, original=64.0)
        self.plan = pkg.kv_plan(self.lens, self.new, self.table, self.free, ints([PAGES]), PAGE, rows)
        dtype = getattr(torch, kind)
        self.q = torch.zeros(rows, HEADS, DIM, dtype=dtype, device="cuda")
        self.k, self.v = (torch.zeros(rows, KV, DIM, dtype=dtype, device="cuda") for _ in range(2))
        self.out = torch.zeros_like(self.q)
        self.turned = None

    def step(self, most):
        p = self.pkg
        plan = p.kv_plan(self.lens, self.new, self.table, self.free, self.plan.info[3:4], PAGE, self.rows, out=self.plan)
        self.turned = p.rope_qk(self.q, self.k, plan.positions, self.freqs, magnitude=1.1)
        p.kv_store_q4_0(self.cache, self.turned[1], self.v, plan.slots)
        p.attention_q4_0(self.turned[0], self.cache, self.table, plan.kv_lens, first_rows=plan.first_rows, max_new=most, out=self.out)
        self.lens.copy_(plan.kv_lens)

    def fill(self, rng, new):
        t = self.torch
        for x in (self.q, self.k, self.v):
            x.copy_(t.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        self.new.copy_(t.tensor(new, dtype=t.int32))
        self.out.fill_(3.0)


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_a_serving_loop(cuda, pkg, O, kind):
    rng = np.random.default_rng(1)
    loop = Loop(cuda, pkg, 4, 128, kind)
    state, table, left = [0] * 4, loop.table.cpu().numpy(), PAGES
    # prompts, a second prompt behind one, single tokens, drafted ones, idle requests, more rows than the requests use
    for new in ([40, 1, 0, 17], [1, 1, 60, 1], [1, 0, 1, 33], [5, 3, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0]):
        loop.fill(rng, new)
        before = loop.cache.cpu().numpy()
        loop.step(64)
        want, table = ref.plan(state, new, table, loop.free.cpu().numpy().tolist(), left, PAGE, loop.rows)
        for got, w in zip(loop.plan, want):
            assert np.array_equal(got.cpu().numpy(), w)
        assert np.array_equal(loop.table.cpu().numpy(), table) and want[5][0] == 0
        state, left = [int(x) for x in want[1]], int(want[5][3])
        q, k = loop.turned
        after = stored(O, before, k.float().cpu().numpy(), loop.v.float().cpu().numpy(), want[2])
        assert np.array_equal(loop.cache.cpu().numpy(), after)
        out, lse, weight = ref.attention(q.double().cpu().numpy(), after, table, state, want[0], DIM ** -0.5)
        check(loop.out, None, out, lse, weight, kind, prompt=kind != "float32")
        assert bool((loop.out[sum(new):] == 3).all())  # rows behind the last one are left as they were
    pkg.check_device_errors()


def test_a_captured_decode_loop(cuda, pkg):
    eager, graphed = (Loop(cuda, pkg, 3, 4, "bfloat16") for _ in range(2))
    rng = np.random.default_rng(2)
    graph = None
    for i in range(20):
        new = [1, 1, 1] if i % 4 else [1, 0, 2]  # always the same shapes: up to 4 rows, up to 2 to a request
        seed = int(rng.integers(1 << 30))
        for loop in (eager, graphed):
            loop.fill(np.random.default_rng(seed), new)
        eager.step(2)
        if graph is None:
            cuda.cuda.synchronize()
            graph = cuda.cuda.CUDAGraph()
            with cuda.cuda.graph(graph):
                graphed.step(2)
        graph.replay()
        cuda.cuda.synchronize()
        for a, b in zip(eager.plan, graphed.plan):
            assert cuda.equal(a, b)
        assert cuda.equal(eager.cache, graphed.cache) and cuda.equal(eager.table, graphed.table) and cuda.equal(eager.out, graphed.out)
    assert int(eager.lens[0]) == 20


def test_a_step_without_pages_writes_nothing(cuda, pkg):
    loop = Loop(cuda, pkg, 4, 128, "float32")
    rng = np.random.default_rng(3)
    loop.fill(rng, [30, 30, 30, 30])
    loop.step(32)
    cache, table = loop.cache.clone(), loop.table.clone()
    loop.fill(rng, [64, 64, 0, 0])  # 16 pages are left, 8 taken by the first step's; these need more than a table's width
    loop.new.copy_(cuda.tensor([100, 1, 0, 0], dtype=cuda.int32))
    loop.step(128)
    assert int(loop.plan.info[0]) == 2 and loop.lens.tolist() == [30, 30, 30, 30]
    assert cuda.equal(loop.cache, cache) and cuda.equal(loop.table, table) and bool((loop.out == 3).all())
