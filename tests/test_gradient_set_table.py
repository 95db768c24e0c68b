"""A gradient set's table has arrived on the device when the set is made: clips may follow on any stream.

Without a GPU, against a stand-in for the CUDA runtime whose copies arrive as late as
the real one's may (tests/cpp/late_copy_runtime.c).
"""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes, sys
lib, late = ctypes.CDLL(sys.argv[1]), ctypes.CDLL(None).late_copies
lib.ponni_b200_gradient_set_count.restype = ctypes.c_int64
n = 3
ptrs, counts, kinds = (ctypes.c_void_p * n)(4096, 8192, 12288), (ctypes.c_int64 * n)(100, 5000, 3), (ctypes.c_int32 * n)(0, 0, 0)
handle = ctypes.c_void_p()
assert lib.ponni_b200_gradient_set_create(ptrs, counts, kinds, n, 0, ctypes.byref(handle)) == 0
assert lib.ponni_b200_gradient_set_count(handle) == 5103
print("LATE", late())
'''


def test_table_has_arrived(tmp_path):
    fake = str(tmp_path / "late_copy_runtime.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-Wall", os.path.join(ROOT, "tests", "cpp", "late_copy_runtime.c"),
                    "-o", fake], check=True)
    lib = os.environ.get("PONNI_B200_LIB") or os.path.join(ROOT, "ponni_b200", "libponni_b200.so")
    r = subprocess.run([sys.executable, "-c", CHILD, lib], env=dict(os.environ, LD_PRELOAD=fake), capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["LATE", "0"]
