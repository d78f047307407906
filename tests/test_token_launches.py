"""The launches of the calls on tokens and of the group norm over their extents, the largest among them: fewer than 2^32 work items
along an axis, at most 65535 workgroups along the second and third, at most 160 KiB of LDS.  The library is loaded in a process where
the runtime's launch calls are recorded and not carried out: no device and no memory are needed."""
import itertools
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RECORDER = r"""
#include <stddef.h>
#include <stdint.h>
typedef struct { uint32_t x, y, z; } dims;
static dims grid, block;
static size_t lds;
uint64_t recorded[64][7];
int launches;
unsigned __hipPushCallConfiguration(dims g, dims b, size_t shared, void *stream) { grid = g; block = b; lds = shared; return 0; }
unsigned __hipPopCallConfiguration(dims *g, dims *b, size_t *shared, void **stream) { *g = grid; *b = block; *shared = lds; *stream = 0; return 0; }
int hipLaunchKernel(const void *f, dims g, dims b, void **args, size_t shared, void *stream) {
    uint64_t *at = recorded[launches++ % 64];
    at[0] = g.x, at[1] = g.y, at[2] = g.z, at[3] = b.x, at[4] = b.y, at[5] = b.z, at[6] = shared;
    return 0;
}
int hipGetLastError(void) { return 0; }
int hipGetDevice(int *device) { *device = 0; return 0; }
int hipFuncSetAttribute(const void *f, int attribute, int value) { return 0; }
"""

CALLS = r"""
import ctypes, json, sys
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from tennis_amd import capi
L = ctypes.CDLL(sys.argv[2])
for name in ("tsx_quantize_tokens", "tsx_gemm_i8_tokens", "tsx_gemm_i8_tokens_workspace_bytes", "tsx_group_norm_nhwc", "tsx_group_norm_tokens_nhwc",
             "tsx_group_norm_workspace_bytes"):
    f = getattr(L, name)
    f.restype, f.argtypes = capi.SIGNATURES[name]
recorded = (ctypes.c_uint64 * 7 * 64).in_dll(recorder, "recorded")
launches = ctypes.c_int.in_dll(recorder, "launches")
at = 1 << 40                      # an address that nothing reads
out = []
for what, *e in json.loads(sys.stdin.read()):
    launches.value = 0
    if what == "quantize":
        rows, cols, kind = e
        rc = L.tsx_quantize_tokens(rows, cols, at, kind, cols, at, cols, at, None)
    elif what == "product":
        m, n, k, kind, to = e
        g = capi.TokenGemm(m, n, k, kind, to, 0, 0.0, at, k, at, at, at, None, at, n)
        rc = L.tsx_gemm_i8_tokens(ctypes.byref(g), at, L.tsx_gemm_i8_tokens_workspace_bytes(ctypes.byref(g)), None)
    else:
        n, pixels, c, groups, kind = e
        g = capi.GroupNorm(n, c, groups, kind, pixels, pixels * c, c, at, None, None, 1e-5, 5, 0.0)
        need = L.tsx_group_norm_workspace_bytes(ctypes.byref(g))
        rc = L.tsx_group_norm_nhwc(ctypes.byref(g), at, at, need, None) if what == "norm" else L.tsx_group_norm_tokens_nhwc(ctypes.byref(g), at, at, at, need, None)
    out.append([rc, [list(r) for r in recorded[:launches.value]]])
print(json.dumps(out))
"""

CASES = ([["quantize", rows, cols, kind] for rows in (1, 511, 512, 1 << 20, (1 << 32) + 1, 1 << 40) for cols in (1, 9, 33, 129, 513, 1025, 2049, 4097, 8193, 1 << 30)
          for kind in (0, 2)] +
         [["product", m, n, k, kind, to] for m in (1, 2, 16, 17, 32, 33, 300, 1 << 14, (1 << 14) + 1, 1 << 20, (1 << 28) - 1)
          for n in (1, 16, 33, 64, 65, 1000, 4096, (1 << 24) - 1) for k, kind in ((1, 2), (64, 3), (1500, 3), (8192, 0), ((1 << 17) - 1, 1)) for to in (0, 2)] +
         [[what, n, pixels, c, groups, kind] for what in ("norm", "tokens") for n in (1, 3, 65535) for pixels in (1, 7, 64, 1000, 16384, 16385, (1 << 30) - 1)
          for c, groups in ((1, 1), (2, 2), (10, 5), (15, 3), (64, 32), (320, 32), (1025, 5), (1280, 32), (4095, 1), (8191, 1), (8192, 8192), (8192, 32)) for kind in (0, 1)])


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    from tennis_amd.build import LIB_PATH
    where = tmp_path_factory.mktemp("recorder")
    source, so = where / "recorder.c", where / "librecorder.so"
    source.write_text(RECORDER)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(so), str(source)])
    run = subprocess.run([sys.executable, "-c", CALLS, str(so), LIB_PATH], input=json.dumps(CASES), capture_output=True, text=True, cwd=ROOT)
    assert run.returncode == 0, run.stderr
    return json.loads(run.stdout)


def too_large(case):
    """Outputs that 288 GB do not hold: a launch may have no room for their tiles, which the call says."""
    return case[0] == "product" and case[1] * case[2] * (2 if case[5] else 4) > 288 << 30


@pytest.mark.parametrize("what", ["quantize", "product", "norm", "tokens"])
def test_launches_hold_their_work_items(recorded, what):
    for case, (rc, launches) in itertools.compress(zip(CASES, recorded), [c[0] == what for c in CASES]):
        assert rc == 0 and launches or rc == -1 and too_large(case), (case, rc)
        for gx, gy, gz, bx, by, bz, lds in launches:
            assert 0 < gx * bx < 1 << 32 and 0 < gy <= 65535 and 0 < gz <= 65535 and bx * by * bz <= 1024 and lds <= 160 << 10, (case, gx, gy, gz, bx, lds)
