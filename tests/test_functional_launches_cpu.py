"""CPU: the grids that the library asks for.  A stand-in for the HIP runtime's launch records them; nothing is launched and no pointer
is read, so that any size can be looked at."""
import json
import os
import shutil
import subprocess
import sys

import pytest

import common as C

STAND_IN = r"""
#include <stdio.h>
typedef struct { unsigned x, y, z; } dim3;
static dim3 grid, block;
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t shared, void* stream) { grid = g; block = b; (void)shared; (void)stream; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* shared, void** stream) { *g = grid; *b = block; *shared = 0; *stream = 0; return 0; }
static unsigned seen[64][4];
static int count;
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t shared, void* stream) {
  (void)f; (void)args; (void)shared; (void)stream;
  if (count < 64) { seen[count][0] = g.x; seen[count][1] = g.y; seen[count][2] = b.x; seen[count][3] = b.y * b.z * g.z; }
  ++count;
  return 0;
}
int hipGetLastError(void) { return 0; }
int recorded(unsigned* out) { for (int i = 0; i < count && i < 64; ++i) for (int k = 0; k < 4; ++k) out[4 * i + k] = seen[i][k]; int n = count; count = 0; return n; }
"""

# (the process has no torch, whose own copy of the runtime would come first)
RUN = r"""
import ctypes, importlib.util, json, sys
stand_in = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
spec = importlib.util.spec_from_file_location("_lib", sys.argv[2])
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib = ctypes.CDLL(L.LIB_PATH)
for name in ("ivid_gn_act_scratch_bytes", "ivid_gn_act_forward", "ivid_gn_act_backward", "ivid_last_error"):
    getattr(lib, name).restype, getattr(lib, name).argtypes = L.SIGNATURES[name]
out = (ctypes.c_uint * 256)()
def launches():
    n = stand_in.recorded(out)
    assert n <= 64
    return [tuple(out[4 * i:4 * i + 4]) for i in range(n)]
result = []
for case in json.loads(sys.argv[3]):
    n, hw, c, groups, dtype = case
    far = 1 << 50
    d = L.GnActDesc(dtype, n, hw, c, 0, groups, 1, far, c, hw * c, None, 0, 0, far << 1, far << 1, None, 0, 0, 1e-5, 0.0, 0, 0, None, 0)
    need = [lib.ivid_gn_act_scratch_bytes(ctypes.byref(d), i) for i in range(2)]
    fwd = lib.ivid_gn_act_forward(ctypes.byref(d), far << 2, far << 3, far << 4, need[0], None), launches()
    bwd = lib.ivid_gn_act_backward(ctypes.byref(d), far << 3, far << 5, far << 6, None, far << 2, far << 2, None, far << 4, need[1], None), launches()
    result.append((need, fwd, bwd, lib.ivid_last_error().decode()))
print(json.dumps(result))
"""


@pytest.fixture(scope="module")
def launches_of(tmp_path_factory):
    """[(n, hw, c, groups, dtype)] -> [(scratch bytes, forward (status, grids), backward (status, grids), last error)]"""
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    where = tmp_path_factory.mktemp("launches")
    src, so = where / "stand_in.c", where / "stand_in.so"
    src.write_text(STAND_IN)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)])
    return lambda cases: json.loads(subprocess.check_output(
        [sys.executable, "-c", RUN, str(so), os.path.join(C.ROOT, "ivid_amd", "_lib.py"), json.dumps(cases)], text=True))


# [samples, pixels, channels, groups, dtype (0 fp32, 1 bf16, 2 fp16)]
ORDINARY = [(1, 64, 1024, 32, 1), (7, 851, 100, 20, 2), (64, 16384, 256, 32, 1), (2, 2500, 1024, 1, 0), ((1 << 23) - 1, 1, 8, 1, 1)]
# ... whose forward pass has 2^23 tiles or more, and the tiles of a sample: a pixel is one piece, a
# tile 2048 of them where a sample has few, else 8192
MANY = [((1 << 23, 1, 8, 1, 1), 1), ((1 << 23, 1, 64, 32, 1), 1), (((1 << 24) - 1, 1, 32, 1, 0), 1), ((1860000, 8200, 2, 1, 1), 5),
        ((980000, 16390, 2, 1, 1), 9), ((32700, (1 << 21) + 1, 2, 1, 1), 257)]
FORWARD = 512      # threads of a workgroup


def test_no_launch_has_2_to_the_32_threads(launches_of):
    """A grid with more in one dimension is not launched, and no error says so."""
    cases = ORDINARY + [c for c, _ in MANY]
    for case, (need, fwd, bwd, message) in zip(cases, launches_of(cases)):
        assert min(need) >= 0, (case, message)
        for status, grids in (fwd, bwd):
            assert status == 0 and grids, (case, message)
            for gx, gy, threads, rest in grids:
                assert rest == 1 and 0 < gx * threads < 1 << 32 and 0 < gy < 1 << 16, (case, gx, gy, threads)


def test_the_launches_hold_every_tile_once(launches_of):
    """... and no launch ends inside a sample whose tiles wait for each other."""
    for (case, tiles), (_, fwd, _, _) in zip(MANY, launches_of([c for c, _ in MANY])):
        grids = [g[0] for g in fwd[1] if g[2] == FORWARD]
        n = case[0]
        if tiles > 256:      # sums, their totals (a workgroup a sample), results
            half = (len(grids) - 1) // 2
            assert grids[half] == n and grids[:half] == grids[half + 1:], case
            grids = grids[:half]
        else:
            assert all(g % tiles == 0 for g in grids), case
        assert sum(grids) == n * tiles and len(grids) > 1, (case, grids)


def test_what_no_launch_holds_is_refused(launches_of):
    cases = [(1 << 24, 1, 8, 1, 1), (1 << 22, 1, 256, 1, 0), (1 << 30, 4, 1, 1, 0)]
    for case, (need, fwd, bwd, message) in zip(cases, launches_of(cases)):
        assert need == [-1, -1] and fwd[0] and bwd[0] and not fwd[1] and not bwd[1], case
        assert "too many tiles" in message
