"""The page plan at request counts whose shared memory lies around the limit that a kernel has without asking for more."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def step(torch, pkg, n, rows):
    """One token for each of n requests at the first token of a page of their own: page and row r are request r's."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, table = [16 * (r % 3) for r in range(n)], np.full((n, 3), -1, np.int32)
    for r, c in enumerate(lens):
        table[r, :c // 16] = 0
    free = list(range(n))
    t = i32(table.tolist())
    got = pkg.kv_plan(i32(lens), i32([1] * n), t, i32(free), i32([n]), 16, rows)
    want, want_table = ref.plan(lens, [1] * n, table, free, n, 16, rows)
    for x, w in zip(got, want):
        assert np.array_equal(x.cpu().numpy(), w)
    assert np.array_equal(t.cpu().numpy(), want_table)


FIRST = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch, __graft_entry__ as entry
from test_gpu_kv_plan_sizes import step
pkg = entry.load_package()
for n in {sizes!r}:
    step(torch, pkg, n, n + 1)
print("plans are right")
"""


@pytest.mark.parametrize("sizes", [(4051, 4052, 4095, 4096, 4097), (4095, 16384, 4052)])
def test_sizes_in_a_process_that_has_planned_nothing_larger(cuda, sizes):
    code = FIRST.format(root=ROOT, tests=os.path.join(ROOT, "tests"), sizes=sizes)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "plans are right" in r.stdout, r.stderr[-2000:]


def test_sizes_from_several_threads(cuda, pkg):
    # a small plan's launch does not take from a large one's what it has asked for
    i32 = lambda n, x: cuda.full((n,), x, dtype=cuda.int32, device="cuda")  # noqa: E731
    failed = []
    def work(n):
        try:
            with cuda.cuda.stream(cuda.cuda.Stream()):
                table = cuda.full((n, 1), -1, dtype=cuda.int32, device="cuda")
                lens, new, free, count = i32(n, 0), i32(n, 1), cuda.arange(n, dtype=cuda.int32, device="cuda"), i32(1, n)
                plan = pkg.kv_plan(lens, new, table, free, count, 16, n)
                for _ in range(400):
                    pkg.kv_plan(lens, new, table, free, count, 16, n, out=plan)
                assert plan.info.tolist() == [0, n, n, 0]
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(n,)) for n in (16384, 4200, 5000, 16384)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
