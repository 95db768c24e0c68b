"""Gradient sets whose tensors share memory, with one another or with the packed vector.

Blocks scale the tensors in no order, so that an element of two tensors would be scaled
once or twice.  Without a GPU: the refusals come before any launch (a launch of the
stand-in runtime, tests/cpp/late_copy_runtime.c, fails with another status).
"""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes, json, sys
lib = ctypes.CDLL(sys.argv[1])
tensors, flat = json.loads(sys.argv[2])
n = len(tensors)
ptrs, counts = (ctypes.c_void_p * n)(*[t[0] for t in tensors]), (ctypes.c_int64 * n)(*[t[1] for t in tensors])
kinds, handle = (ctypes.c_int32 * n)(*[t[2] for t in tensors]), ctypes.c_void_p()
assert lib.ponni_b200_gradient_set_create(ptrs, counts, kinds, n, 0, ctypes.byref(handle)) == 0
lib.ponni_b200_gradient_set_workspace.restype = lib.ponni_b200_gradient_set_count.restype = ctypes.c_int64
need = lib.ponni_b200_gradient_set_workspace(handle)
where, kind = flat or (None, 0)
print("STATUS", lib.ponni_b200_gradient_set_clip(handle, ctypes.c_double(1.0), ctypes.c_void_p(where), kind, ctypes.c_void_p(64),
                                                 ctypes.c_void_p(1 << 40), ctypes.c_int64(need), None))
'''
F32, F16 = 0, 2


@pytest.fixture(scope="module")
def clip(tmp_path_factory):
    fake = str(tmp_path_factory.mktemp("runtime") / "late_copy_runtime.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-Wall", os.path.join(ROOT, "tests", "cpp", "late_copy_runtime.c"),
                    "-o", fake], check=True)
    lib = os.environ.get("PONNI_B200_LIB") or os.path.join(ROOT, "ponni_b200", "libponni_b200.so")

    def status(tensors, flat=None):
        r = subprocess.run([sys.executable, "-c", CHILD, lib, json.dumps([tensors, flat])],
                           env=dict(os.environ, LD_PRELOAD=fake, CUDA_VISIBLE_DEVICES=""), capture_output=True, text=True,
                           timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return int(r.stdout.split()[1])

    return status


@pytest.mark.parametrize("tensors,flat,refused", [
    ([(4096, 100, F32), (4096, 100, F32)], None, True),                        # the same tensor twice, in place
    ([(4096, 100, F32), (8192, 10, F32), (4096 + 396, 1, F32)], None, True),   # the last element of another
    ([(4096, 1000, F32), (4200, 2, F32), (4300, 2, F32)], None, True),         # inside another
    ([(4096, 100, F32), (4496, 100, F32)], None, False),                       # one behind the other
    ([(4096, 100, F32), (4096, 0, F32)], None, False),                         # a tensor without elements
    ([(4096, 100, F32), (4096, 100, F32)], (16384, F32), False),               # the same twice, packed elsewhere
    ([(4096, 100, F32), (4496, 100, F32)], (4096, F32), False),                # views of the packed vector
    ([(4096, 100, F32), (8192, 100, F32)], (4096, F32), False),
    ([(4096, 100, F32), (4496, 100, F32)], (4100, F32), True),                 # one element off
    ([(4496, 100, F32), (4096, 100, F32)], (4096, F32), True),                 # views in another order
    ([(4096, 100, F16), (4296, 100, F16)], (4096, F32), True),                 # of another type
    ([(4096, 1000, F32), (4200, 2, F32), (9000, 2, F32)], (8196, F32), True),  # the packed values reach a tensor
    ([(4096, 1000, F32), (4200, 2, F32), (40000, 2, F32)], (8096, F32), False),
])
def test_overlap(clip, tensors, flat, refused):
    assert (clip(tensors, flat) == 1) == refused
