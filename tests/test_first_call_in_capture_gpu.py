"""A process whose first call of an operator is captured into a graph."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from batchspec_b200.kernels import ops
ops.load_library()
device = torch.device("cuda:0")
w32 = torch.randn(512, 512, device=device)
(x, xs), (w, ws) = ops.quantize_fp8(torch.randn(4, 512, device=device)), ops.quantize_fp8(w32, 128)
# memory that holds 7s in the pool from which the second graph takes its own
pool = torch.cuda.graph_pool_handle()
first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
with torch.cuda.graph(first, pool=pool):
    old = torch.full((1 << 18,), 7, dtype=torch.int32, device=device), [torch.full((1,), 7, dtype=torch.int32, device=device) for _ in range(64)]
first.replay()
torch.cuda.synchronize()
del old
with torch.cuda.graph(second, pool=pool):
    out = ops.linear_fp8(x, xs, w, ws)
    counters = ops._counters(device, 100), ops._work_counter(device)
assert not any(int(c.abs().sum()) for c in counters), "zeros before the first replay"
ops.check_status()
want = ops.linear_fp8(x, xs, w, ws)
second.replay()
torch.cuda.synchronize()
assert torch.equal(out, want)
# what a kernel reported is not cleared by a replay
ops._status_word(device).fill_(104)
second.replay()
torch.cuda.synchronize()
try:
    ops.check_status()
except ops.KernelError as e:
    assert "8-bit product" in str(e)
else:
    raise AssertionError("the report is gone")
print("fine")
"""


def test_words_that_calls_share_are_not_the_graphs():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stderr[-2000:]
