"""What kd_f8_mm_run would launch, without a GPU: kd_f8_host.cpp compiled with
launchers that record their arguments in place of the kernels'."""
import ctypes
import functools
import os
import subprocess
import tempfile
from collections import namedtuple

import kd_f8
import kd_fa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r"""
#include "kd_f8_host.cpp"
static int64_t got[8];
namespace kdfa {
int device_gfx950() { return KD_FA_OK; }
hipError_t launch_f8_quantize(const F8RowsArgs &, hipStream_t) { return hipSuccess; }
hipError_t launch_f8_norm(const F8RowsArgs &, hipStream_t) { return hipSuccess; }
hipError_t launch_f8_mm(const F8MmArgs &a, int tile, hipStream_t) {
    const int64_t v[] = {tile, a.tiles_m, a.tiles_n, a.n_blocks, a.cols, a.M, a.N, a.d_nb1};
    for (int i = 0; i < 8; ++i) got[i] = v[i];
    return hipSuccess;
}
}
extern "C" const int64_t *recorded() { return got; }
"""

Plan = namedtuple("Plan", "tile tiles_m tiles_n n_blocks cols M N d_nb1")
TILES = (101, 202, 401, 402, 405, 10804, 10806, 10810, 10816, 11616)


def outputs(tile):
    return 16 * (tile // 100 % 100)


def tokens(tile):
    return 16 * (tile % 100)


@functools.lru_cache(maxsize=None)
def _host():
    d = tempfile.mkdtemp()
    src, out = os.path.join(d, "plan.cpp"), os.path.join(d, "plan.so")
    with open(src, "w") as f:
        f.write(SRC)
    subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "-fPIC", "--offload-arch=gfx950", "-shared",
                    "-I", os.path.join(ROOT, "kandinsky.cpp_amd", "csrc"), src, "-o", out], check=True, capture_output=True)
    lib = ctypes.CDLL(out)
    lib.recorded.restype = ctypes.POINTER(ctypes.c_int64)
    lib.kd_f8_mm_run.argtypes = [ctypes.POINTER(kd_f8.KdF8MmDesc), ctypes.c_void_p]
    return lib


def _view(t, rows, cols, size, kind, row_bytes):
    t.type = kind
    for i, (ne, nb) in enumerate([(cols, size), (rows, row_bytes), (1, row_bytes * rows), (1, row_bytes * rows)]):
        t.ne[i], t.nb[i] = ne, nb
    t.data = 1 << 20   # not read


def desc(M, N, K, d_nb1=None):
    """A contiguous call of M tokens, N outputs and K inputs."""
    d = kd_f8.KdF8MmDesc()
    words = (kd_f8.blocks(K) + 3) // 4 * 4
    for r, n in ((d.w, N), (d.x, M)):
        _view(r.codes, n, K, 1, kd_f8.TYPE_E4M3, K)
        _view(r.scales, n, kd_f8.blocks(K), 1, kd_f8.TYPE_E8M0, words)
    _view(d.dst, M, N, 2, kd_f8.TYPE_BF16, 2 * N if d_nb1 is None else d_nb1)
    return d


def run(d):
    """(status, what was launched)."""
    lib = _host()
    st = lib.kd_f8_mm_run(ctypes.byref(d), None)
    return st, Plan(*lib.recorded()[:8])


def plan(M, N, K):
    st, p = run(desc(M, N, K))
    assert st == kd_fa.OK, st
    return p
