"""That the shapes of the GPU tests choose the ways that they are there for, without a GPU: the kernels that
libredukt_gpu.so launches for them, on a stand-in for the launching part of the HIP runtime."""
import json
import os
import re
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ops  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402
from tests import test_gpu_op_ways as ways  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# What a launch of the operators needs: functions are known by their names, and any address is memory of device 0.
LAUNCHES = r"""
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <string.h>
static struct { const void* fn; const char* name; } g_fn[4096];
static int g_n;
static char g_log[1 << 16];
void** __hipRegisterFatBinary(const void* d) { static void* h; (void)d; return &h; }
void __hipUnregisterFatBinary(void** m) { (void)m; }
void __hipRegisterFunction(void** m, const void* fn, char* a, const char* name, unsigned c, void* d, void* e, dim3* f, dim3* g, int* h) {
    (void)m, (void)a, (void)c, (void)d, (void)e, (void)f, (void)g, (void)h;
    if (g_n < 4096 && strstr(name, "3rdk")) g_fn[g_n].fn = fn, g_fn[g_n++].name = name;
}
void __hipRegisterVar(void** m, void* v, char* a, const char* b, int c, size_t d, int e, int f) {
    (void)m, (void)v, (void)a, (void)b, (void)c, (void)d, (void)e, (void)f;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
    (void)p;
    memset(a, 0, sizeof *a);
    a->type = hipMemoryTypeDevice;
    return hipSuccess;
}
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipLaunchKernel(const void* fn, dim3 g, dim3 b, void** args, size_t lds, hipStream_t s) {
    (void)args, (void)s;
    const size_t at = strlen(g_log);
    const char* name = "?";
    for (int i = 0; i < g_n; i++) if (g_fn[i].fn == fn) name = g_fn[i].name;
    snprintf(g_log + at, sizeof g_log - at, "%s %u %u %u %zu\n", name, g.x, g.y, b.x, lds);
    return hipSuccess;
}
const char* launches(void) { return g_log; }
void clear_launches(void) { g_log[0] = 0; }
"""

CHILD = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
shim.launches.restype = ctypes.c_char_p
from redukt_amd import ops
L, P, out = ops._load(), 1 << 30, []
def recorded(call):
    shim.clear_launches()
    code = call()
    return [code] + [l.split() for l in shim.launches().decode().splitlines()]
for op, v in json.loads(sys.stdin.read()):
    if op == "fp8":
        dtype, m, n, k = v
        a = ops.Fp8Matmul(dtype, m, n, k, P, k, P, P, k, P, None, P, n)
        out.append(recorded(lambda: L.redukt_op_fp8_matmul(ctypes.byref(a), None)))
    elif op == "step":
        rows, ch, groups, n, dtype = v
        a = ops.ScanRows(dtype, rows, ch, groups, n, P, P, P, P, P, P, ch, ch, ch, groups * n, groups * n, ch, P, P, P)
        out.append(recorded(lambda: L.redukt_op_scan_step(ctypes.byref(a), P, rows + 2, P, None)))
    elif op == "chunk":
        rows, n_seq, ch, groups, n, dtype = v
        a = ops.ScanRows(dtype, rows, ch, groups, n, P, P, P, P, P, P, ch, ch, ch, groups * n, groups * n, ch, P, P, P)
        out.append(recorded(lambda: L.redukt_op_scan_chunk(ctypes.byref(a), P, n_seq, P, P, n_seq + 2, P, P, 1 << 40, None)))
    elif op == "grad":
        rows, n_seq, ch, groups, n, dtype = v
        a = ops.ScanRows(dtype, rows, ch, groups, n, P, P, P, P, P, None, ch, ch, ch, groups * n, groups * n, 0, P, P, P)
        g = ops.ScanGradients(P, P, P, P, P, P, ch, ch, ch, ch, groups * n, groups * n, P, P, P)
        out.append(recorded(lambda: L.redukt_op_scan_grad(ctypes.byref(a), ctypes.byref(g), P, n_seq, P, P, P, P, 1 << 40, None)))
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    d = tmp_path_factory.mktemp("launches")
    (d / "l.c").write_text(LAUNCHES)
    so = str(d / "liblaunches.so")
    subprocess.run(["gcc", "-O1", "-std=gnu11", "-shared", "-fPIC", "-I/opt/rocm/include", str(d / "l.c"), "-o", so], check=True)

    def run(calls):
        r = subprocess.run([sys.executable, "-c", CHILD, so], input=json.dumps(calls), cwd=ROOT, capture_output=True, text=True, timeout=120,
                           env={**os.environ, "PYTHONPATH": ROOT})
        assert r.returncode == 0, r.stderr[-2000:]
        got = json.loads(r.stdout.strip().splitlines()[-1])
        assert all(g[0] == 0 for g in got)
        return [[l for l in g[1:]] for g in got]
    return run


def kernel(name):
    """(function, its template's numbers) of a kernel's mangled name."""
    fn = re.search(r"\d+(k_[a-z0-9_]+?)(?=I|E|P|N|v)", name).group(1)
    return fn, tuple(int(v) for v in re.findall(r"L[ibj](\d+)E", name))


TILES = {(256, 256, 2, 4, 2), (128, 128, 2, 2, 2), (64, 128, 2, 2, 3), (64, 64, 2, 2, 2), (64, 64, 2, 2, 4), (64, 32, 2, 1, 4)}


def test_the_products_shapes_reach_every_kernel_with_more_blocks_than_it_has_stages(launched):
    for dtype in (0, 1, 2):
        met = {}
        for shape, ((name, *_),) in zip(ways.DEEP, launched([["fp8", [dtype, *s]] for s in ways.DEEP])):
            met.setdefault(kernel(name), []).append(-(-shape[2] // 128))
        assert {t for fn, t in met if fn == "k_fp8_tiles"} == TILES - ({(256, 256, 2, 4, 2)} if dtype == 2 else set())
        assert {fn for fn, _ in met} == {"k_fp8_tiles", "k_fp8_few", "k_fp8_bytes"}
        assert all(max(blocks) > t[4] + 1 for (fn, t), blocks in met.items() if fn == "k_fp8_tiles")
        assert len([s for s in ways.DEEP if s[2] % 128 == 0]) == 0


def test_products_of_few_tokens_take_no_tiles_that_are_mostly_empty(launched):
    shapes = [(m, n, k) for m in (1, 2, 4, 8, 9, 16, 17, 32, 64, 65, 100, 128, 129, 200) for n, k in ((4096, 4096), (8192, 768), (50280, 768), (131072, 4096))]
    for dtype in (0, 2):
        for (m, n, k), ((name, *_),) in zip(shapes, launched([["fp8", [dtype, *s]] for s in shapes])):
            fn, t = kernel(name)
            if m <= 8:
                assert fn == "k_fp8_few", (m, n, k, dtype)
            elif m > 16 or fn != "k_fp8_few":
                assert fn == "k_fp8_tiles" and (t[0] == 64 or m > t[0] // 2), (m, n, k, dtype)


def test_the_scans_shapes_choose_their_ways(launched):
    sizes = (8, 16, 32, 64)
    for (((name, *_),), n) in zip(launched([["step", [*s, n, 2]] for s in ways.STEPS for n in sizes]), sizes * len(ways.STEPS)):
        assert kernel(name) == ("k_scan_step", (n // 4, 4))
    calls = [(lens, joined, n) for lens, joined in ways.CHUNKS for n in sizes] + [(lens, joined, 16) for lens, joined in ways.SPREAD]
    for (lens, joined, n), launches in zip(calls, launched([["chunk", [sum(l), len(l), 70, 1, n, 2]] for l, _, n in calls])):
        assert [kernel(l[0]) for l in launches] == [(f, (n // 4,)) for f in ["k_scan_pieces"] + ["k_scan_join"] * joined + ["k_scan_run"]]
    for lens, _ in ways.SPREAD:
        for n, piece in ((16, 64), (64, 32)):
            assert ops.scan_chunk_workspace(sum(lens), len(lens), 70, 1, n) == 2 * sum(lens) // piece * 70 * (n + 1) * 4


def test_the_gradients_shapes_choose_their_ways(launched):
    calls = [(name, n) for name in ways.GRAD_WAYS for n in (8, 16, 32, 64)]
    args = [["grad", [sum(ways.GRAD_WAYS[w][0]), len(ways.GRAD_WAYS[w][0]), *ways.GRAD_WAYS[w][1:3], n, 2]] for w, n in calls]
    for (name, n), launches in zip(calls, launched(args)):
        lens, ch, groups, want = ways.GRAD_WAYS[name]
        short, per, joined, size = ways.grad_way(lens, ch, groups, n)
        assert short == (name in ways.SHORT_WAYS) and (per, joined) == want[n > 16], (name, n)
        assert size == ops.scan_grad_workspace(sum(lens), len(lens), ch, groups, n)
        fns = [kernel(l[0]) for l in launches]
        assert [f for f, _ in fns] == ["k_scan_grad_pieces"] + ["k_scan_grad_join"] * joined + ["k_scan_grad_run", "k_scan_grad_rows", "k_scan_grad_columns"]
        assert all(t == (n // 4, int(short)) for f, t in fns[:-2])
        pieces = sum(lens) // ((64 if n <= 16 else 32) // (1 + short)) + len(lens) + 2
        assert int(launches[-3][1]) == pieces * groups * -(-(-(-(ch // groups) // 64)) // per)


def test_drawing_by_whole_arrays_is_drawing():
    r = np.random.default_rng(1)
    for i in range(300):
        l = np.round(r.standard_normal(int(r.integers(1, 60))) * 3, int(r.integers(0, 4)))
        l[r.random(len(l)) < 0.1] = r.choice([-np.inf, np.nan])
        s = dict(temperature=r.choice([0.0, 0.5, 1.0, 3.0, np.inf]), top_k=int(r.integers(-1, 30)), top_p=r.choice([0.0, 0.3, 0.9, 1.0]),
                 min_p=r.choice([0.0, 0.1, 1.0, 2.0]))
        u = r.choice([0.0, 0.5, r.random(), 0.999999, 1.0])
        assert f64.draw(l, u, **s) == f64.draw_fast(l, u, **s), (i, s)
