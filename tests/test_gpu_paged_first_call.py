"""The first call of a process, captured in a graph: nothing that a kernel gets may hang on a call before it."""
import subprocess
import sys

import pytest

from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from VAR_Q import _cabi
from VAR_Q.paged import PagedCache

c, D, page, n, dev = int(sys.argv[2]), 64, 16, 100, "cuda"
codes = lambda: torch.randint(-2 ** 31, 2 ** 31 - 1, (7, 2, page, D // 4), dtype=torch.int32, device=dev)
scale = lambda: torch.rand((7, 2, page), device=dev) / 100 + 0.001
cache = PagedCache.over(codes(), codes(), scale(), scale(), D)
q = torch.randn((c, 4, D), device=dev).half()
table, lens, starts = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[3, 1, 4, 0, 5, 2, 6]], [n], [0, c]))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = cache.attend(q, table, lens, starts, c, n, 0.125)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, cache.attend(q, table, lens, starts, c, n, 0.125))
assert _cabi.device_status() == 0
table[0, 2] = 1 << 20
graph.replay()
assert _cabi.device_status() == 66
"""


@pytest.mark.parametrize("c", [1, 100])
def test_the_first_call_is_captured(c):
    done = subprocess.run([sys.executable, "-c", PROGRAM, PKG_ROOT, str(c)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]
