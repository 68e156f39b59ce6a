"""CPU: the first calls of the operators in a process, made by several threads at once.

What the library asks a device once must be there, whole, for every thread that needs it.  The calls run against a stand-in for the
CUDA runtime that answers slowly, and that writes the answer to a question about clusters in two steps; it launches nothing, and
prints each launch's shape.
"""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = r"""
#include <atomic>
#include <cstdio>
#include <unistd.h>
struct Dim { unsigned x, y, z; };
struct Attr { int id, pad; union { char room[64]; Dim cluster; } val; };
struct Config { Dim grid, block; size_t smem; void *stream; Attr *attrs; unsigned n; };
static int encode(...) { return 0; }
extern "C" {
int cudaGetDeviceCount(int *n) { *n = 1; return 0; }
int cudaGetDevice(int *d) { *d = 0; return 0; }
int cudaSetDevice(int) { return 0; }
int cudaGetLastError() { return 0; }
int cudaFuncSetAttribute(const void *, int, int) { usleep(2000); return 0; }
int cudaDeviceGetAttribute(int *v, int, int) { usleep(20000); *v = 148; return 0; }
int cudaOccupancyMaxActiveClusters(int *n, const void *, const Config *c) {
    *n = 0;
    usleep(5000);
    *n = 148 / (int)c->attrs[0].val.cluster.x;
    return 0;
}
int cudaGetDriverEntryPoint(const char *, void **f, unsigned long long, int *r) {
    usleep(50000);
    *f = (void *)encode;
    *r = 0;
    return 0;
}
int cudaLaunchKernelExC(const Config *c, const void *, void **) {
    const unsigned cluster = c->n ? c->attrs[0].val.cluster.x : 1;
    std::printf("launch %u %u %u %zu\n", c->grid.x, c->block.x, cluster, c->smem);
    std::fflush(stdout);
    return 0;
}
}
"""

CHILD = """
import ctypes as C, sys, threading
from loki_b200 import _lib
L, P = _lib.lib, C.c_void_p(4096)
calls = {
    "linear": lambda: L.lk_linear(0, _lib.LK_BF16, 48, 8192, 1024, P, 1024, None, P, 1024, None, None, 0, None, 0, _lib.LK_BF16, P, 8192, None),
    "linear_few": lambda: L.lk_linear(0, _lib.LK_I8, 1, 4096, 4096, P, 4096, None, P, 4096, None, None, 0, None, 0, _lib.LK_F32, P, 4096, None),
    "sample": lambda: L.lk_sample(0, _lib.LK_F32, 8, 1000000, P, 1000000, None, None, None, None, P, P, P, P, None),
    "norm": lambda: L.lk_rms_norm_i8(0, _lib.LK_F32, 9000, 1024, P, 1024, None, 0, None, 0, 1e-6, None, 0, P, 1024, P, None),
}
call, n = calls[sys.argv[1]], 8
meet, got = threading.Barrier(n), [None] * n
def work(i):
    meet.wait()
    got[i] = (call(), L.lk_last_error())
threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
[t.start() for t in threads]
[t.join() for t in threads]
print("status", *[s for s, _ in got], flush=True)
for s, why in got:
    if s: print(why, file=sys.stderr)
call()  # alone, with everything known
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    d = tmp_path_factory.mktemp("cudart")
    src, lib = d / "stand_in.cpp", d / "stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    return str(lib)


@pytest.mark.parametrize("name", ["linear", "linear_few", "sample", "norm"])
def test_several_threads_at_once(stand_in, name):
    env = dict(os.environ, LD_PRELOAD=stand_in)
    r = subprocess.run([sys.executable, "-c", CHILD, name], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [line.split() for line in r.stdout.splitlines()]
    status = [line[1:] for line in lines if line[0] == "status"]
    assert status == [["0"] * 8], (status, r.stderr[-500:])
    launches = [tuple(line[1:]) for line in lines if line[0] == "launch"]
    assert len(launches) == 9 and len(set(launches)) == 1, launches
