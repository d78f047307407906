"""What the host does for a group norm, whatever the number of groups: the library in a process where launches are recorded and not carried
out, the shortest of many calls."""
import json
import subprocess
import sys

from test_token_launches import RECORDER, ROOT

CALLS = r"""
import ctypes, json, sys, time
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from tennis_amd import capi
L = ctypes.CDLL(sys.argv[2])
for name in ("tsx_group_norm_nhwc", "tsx_group_norm_workspace_bytes"):
    f = getattr(L, name)
    f.restype, f.argtypes = capi.SIGNATURES[name]
at = 1 << 40                      # an address that nothing reads
out = []
for n, pixels, c, groups, kind in json.loads(sys.stdin.read()):
    g = capi.GroupNorm(n, c, groups, kind, pixels, pixels * c, c, at, None, None, 1e-5, 5, 0.0)
    r = ctypes.byref(g)
    need = L.tsx_group_norm_workspace_bytes(r)
    best = 1.0
    for _ in range(2000):
        t = time.perf_counter()
        rc = L.tsx_group_norm_nhwc(r, at, at, need, None)
        best = min(best, time.perf_counter() - t)
        assert rc == 0
    out.append(best)
print(json.dumps(out))
"""

# few groups first; a channel a group, prime numbers of channels among them, where no width of pieces fits
CASES = [[2, 64, 1280, 32, 2]] + [[n, pixels, c, c, kind] for n, pixels in ((2, 64), (1, 1000)) for c in (1280, 7919, 8191, 8192) for kind in (0, 2)]


def test_the_plan_of_many_groups_is_not_slower(tmp_path):
    """A call plans in a few microseconds, 4 more for 8192 groups at the most (a look at every number of groups a workgroup could take
    was 8 to 50 more)."""
    from tennis_amd.build import LIB_PATH
    source, so = tmp_path / "recorder.c", tmp_path / "librecorder.so"
    source.write_text(RECORDER)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(so), str(source)])
    run = subprocess.run([sys.executable, "-c", CALLS, str(so), LIB_PATH], input=json.dumps(CASES), capture_output=True, text=True, cwd=ROOT)
    assert run.returncode == 0, run.stderr
    times = json.loads(run.stdout)
    for case, t in zip(CASES, times):
        print(case, "%.2f us" % (t * 1e6))
    assert max(times[1:]) < times[0] + 4e-6, list(zip(CASES, times))
