"""The launches of the calls on MXFP4 rows and of the root-mean-square norm over their extents, the largest among them: fewer than 2^32
work items along an axis, at most 65535 workgroups along the second and third, at most 160 KiB of LDS.  The library is loaded in a
process where the runtime's launch calls are recorded and not carried out: no device and no memory are needed."""
import itertools
import json
import subprocess
import sys

import pytest

from tests.test_token_launches import RECORDER, ROOT

CALLS = r"""
import ctypes, json, os, sys
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from tennis_amd import capi
L = ctypes.CDLL(sys.argv[2])
for name in ("tsx_quantize_mxfp4", "tsx_dequantize_mxfp4", "tsx_dequantize_tokens", "tsx_gemm_mxfp4", "tsx_gemm_mxfp4_workspace_bytes", "tsx_gemm_mxfp4_pack_weights",
             "tsx_rms_norm_rows", "tsx_rms_norm_tokens", "tsx_rms_norm_mxfp4"):
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
        rc = L.tsx_quantize_mxfp4(rows, cols, at, kind, cols, at, (cols + 1) // 2, at, (cols + 31) // 32, None)
        rc = rc or L.tsx_dequantize_mxfp4(rows, cols, at, (cols + 1) // 2, at, (cols + 31) // 32, at, kind, cols, None)
        rc = rc or L.tsx_dequantize_tokens(rows, cols, at, cols, at, at, kind, cols, None)
    elif what == "product":
        m, n, k, kind, to, kernel = e
        os.environ.pop("TSX_MXFP4_KERNEL", None)
        if kernel is not None:
            os.environ["TSX_MXFP4_KERNEL"] = str(kernel)
        g = capi.Mxfp4Gemm(m, n, k, kind, to, 0, 0.0, at, k, at, k, at, None, at, n)
        rc = L.tsx_gemm_mxfp4(ctypes.byref(g), at, L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(g)), None)
        rc = rc or L.tsx_gemm_mxfp4_pack_weights(k, n, at, k, at, k, at, None)
    else:
        rows, cols, kind = e
        g = capi.RmsNorm(rows, cols, kind, at, cols, at, cols, at, cols, at, 1e-6)
        rc = L.tsx_rms_norm_rows(ctypes.byref(g), at, cols, None) or L.tsx_rms_norm_tokens(ctypes.byref(g), at, at, None) or L.tsx_rms_norm_mxfp4(ctypes.byref(g), at, at, None)
    out.append([rc, [list(r) for r in recorded[:min(launches.value, 64)]]])
print(json.dumps(out))
"""

COLS = (1, 9, 33, 129, 513, 1025, 2049, 4097, 8193, 16385, 1 << 30)
CASES = ([["quantize", rows, cols, kind] for rows in (1, 511, 512, 1 << 20, (1 << 31) + 1) for cols in COLS for kind in (0, 2) if rows * cols <= 1 << 38] +
         [["norm", rows, cols, kind] for rows in (1, 511, 512, 1 << 20, (1 << 32) + 1, 1 << 40) for cols in COLS for kind in (0, 1, 2)] +
         [["product", m, n, k, kind, to, kernel] for m in (1, 2, 16, 17, 32, 33, 300, 1 << 14, (1 << 14) + 1, 1 << 20, (1 << 28) - 1)
          for n in (1, 16, 33, 64, 65, 1000, 4096, (1 << 24) - 1) for k, kind in ((1, 2), (64, 4), (1500, 4), (8192, 0), (8192, 4), ((1 << 21) - 1, 1)) for to in (0, 2)
          for kernel in (None, 0, 1, 2, 3, 4, 5) if m * k <= 1 << 38 and not (kernel == 1 and m * n >= 1 << 34)])      # 1: of few tiles by choice


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


@pytest.mark.parametrize("what", ["quantize", "product", "norm"])
def test_launches_hold_their_work_items(recorded, what):
    for case, (rc, launches) in itertools.compress(zip(CASES, recorded), [c[0] == what for c in CASES]):
        assert rc == 0 and launches or rc == -1 and too_large(case), (case, rc)
        for gx, gy, gz, bx, by, bz, lds in launches:
            assert 0 < gx * bx < 1 << 32 and 0 < gy <= 65535 and 0 < gz <= 65535 and bx * by * bz <= 1024 and lds <= 160 << 10, (case, gx, gy, gz, bx, lds)
