"""GPU: the first calls of the operators in a process, made by several threads at once.

What a library asks a device once (limits, entry points) must be there for every thread that needs it, or be
waited for: each process below starts eight threads whose first call of each operator meets the others'.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import threading
import torch
from loki_b200 import ops

N = 8
g = torch.Generator(device="cuda").manual_seed(1)
a = torch.randint(-127, 128, (40, 256), generator=g, device="cuda", dtype=torch.int8)
w = torch.randint(-127, 128, (1000, 256), generator=g, device="cuda", dtype=torch.int8)
x = torch.randn(700, 1024, generator=g, device="cuda")
scores = torch.randn(8, 50000, generator=g, device="cuda")
u = torch.rand(8, generator=g, device="cuda")
calls = [lambda: (ops.linear(a, w),), lambda: ops.sample(scores, u, top_p=p), lambda: ops.rms_norm_i8(x)[:2]]
p = torch.full((8,), 0.9, device="cuda")
streams = [torch.cuda.Stream() for _ in range(N)]
torch.cuda.synchronize()
meet = threading.Barrier(N)
got = [[None] * len(calls) for _ in range(N)]

def work(i):
    with torch.cuda.stream(streams[i]):
        for c, call in enumerate(calls):
            meet.wait()
            try:
                got[i][c] = call()
            except Exception as e:
                got[i][c] = e

threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
want = [call() for call in calls]
for i in range(N):
    for c in range(len(calls)):
        if isinstance(got[i][c], Exception):
            raise SystemExit(f"thread {i}, call {c}: {got[i][c]}")
        assert all(torch.equal(s, t) for s, t in zip(got[i][c], want[c])), (i, c)
"""


@pytest.mark.parametrize("turn", range(3))
def test_several_threads_at_once(lk, turn):
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
