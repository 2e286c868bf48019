"""The calls around the paged cache captured into a graph by a process that has made none of them before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
sys.path[:0] = [{root!r}]
import torch, __graft_entry__ as entry
pkg = entry.load_package()
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
n, new, dim = {n}, {new}, 128
rows = n * new
cache = pkg.kv_cache_q4_0(n * 4, 2, 16, dim)
q, k, v = (torch.randn(rows, h, dim, device="cuda").to(torch.{kind}) for h in (8, 2, 2))
lens, add, table, free, count = i32([0] * n), i32([new] * n), i32([[-1] * 4] * n), i32(list(range(4 * n))), i32([4 * n])
freqs = torch.pow(1e4, -torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
zero = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device="cuda")
plan = pkg.KvPlan((zero(n + 1), zero(n), zero(rows, t=torch.int64), zero(rows), zero(rows), zero(4)))
out = torch.zeros_like(q)
torch.cuda.synchronize()
def step():
    pkg.kv_plan(lens, add, table, free, count, 16, rows, out=plan)
    a, b = pkg.rope_qk(q, k, plan.positions, freqs)
    pkg.kv_store_q4_0(cache, b, v, plan.slots)
    pkg.attention_q4_0(a, cache, table, plan.kv_lens, first_rows=plan.first_rows, max_new=new, out=out)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
first = out.clone()
out.zero_(), cache.zero_(), table.fill_(-1)
step()
torch.cuda.synchronize()
pkg.check_device_errors()
assert bool(first.any()) and torch.equal(out, first)
print("the same")
"""


@pytest.mark.parametrize("n,new,kind", [(5, 1, "float32"), (5, 40, "bfloat16"), (4200, 1, "float16")])
def test_the_first_call_is_captured(cuda, n, new, kind):
    r = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT, n=n, new=new, kind=kind)], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]
