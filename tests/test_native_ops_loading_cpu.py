"""The native operators' library (libsfast_torch.so) beside the kernel library: a file that is missing or does not load stops its own operators
and nothing else."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def python(code, **env):
    r = subprocess.run([sys.executable, "-W", "always", "-c", "import sys\nsys.path.insert(0, 'stable-fast_amd')\n" + code], cwd=ROOT, capture_output=True,
                       text=True, timeout=300, env=dict(os.environ, **env))
    assert r.returncode == 0, r.stderr[-3000:]
    return r


USE = """
import sfast
from sfast.hip import functional as F, lib as L
L.load()                                  # every other kernel is there
x = torch.zeros(1, 64, 1, 64, dtype=torch.float16)
try:
    F.block_means(x, 64)
    raise SystemExit("not refused")
except L.SfastHipError as e:
    assert "libsfast_torch.so" in str(e) and "build" in str(e), e
"""


def test_a_library_that_does_not_load(built_lib):
    r = python("""
import torch
load = torch.ops.load_library
def stale(path):
    raise OSError(path + ": undefined symbol: sfast_hip_of_another_build")
torch.ops.load_library = stale
""" + USE + """
torch.ops.load_library = load             # rebuilt meanwhile
assert L.load_torch_ops()
""")
    assert "undefined symbol" in r.stderr and "RuntimeWarning" in r.stderr


def test_a_library_that_is_not_there(built_lib):
    r = python("""
import os, torch
exists = os.path.exists
os.path.exists = lambda p: exists(p) and not str(p).endswith("libsfast_torch.so")
""" + USE)
    assert "libsfast_torch" not in r.stderr


def test_the_probe_build_serves_the_native_operators_too(built_lib, built_probe_lib):
    """SFAST_HIP_PROBES=1: one kernel library in the process, with one state, whichever operator is called."""
    r = python("""
import sfast
from sfast.hip import lib as L
assert L.load().sfast_hip_has_probes() and L.load_torch_ops()
print(*sorted({line.split()[-1].rsplit("/", 1)[1] for line in open("/proc/self/maps") if "libsfast_" in line}))
""", SFAST_HIP_PROBES="1")
    assert r.stdout.split() == ["libsfast_hip_probes.so", "libsfast_torch.so"]
    r = python("""
import sfast
from sfast.hip import lib as L
assert not L.load().sfast_hip_has_probes() and L.load_torch_ops()
assert L.load_probes().sfast_hip_has_probes() and not L.load().sfast_hip_has_probes()
print(*sorted({line.split()[-1].rsplit("/", 1)[1] for line in open("/proc/self/maps") if "libsfast_" in line}))
""")
    assert r.stdout.split() == ["libsfast_hip.so", "libsfast_hip_probes.so", "libsfast_torch.so"]
