"""The expert product's bounded waits end with an error status, and the context stays usable.

As tests/test_gpu_wait_bound.py does for the model kernels: the test library
(libponni_b200_waittest.so: waits of 2^20 cycles, a host-settable flag) leaves out
the completion signal of the first tile of a launch; in a child process bound to it
check_operators raises PONNI_B200_ERR_DEVICE, and the next product is right.
"""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "ponni_b200", "libponni_b200_waittest.so")

CHILD = r'''
import json, sys
import torch
import ponni_b200 as pb
from tests import expert_ref as R

rows, experts = int(sys.argv[1]), 2
lib = pb._abi.lib()
skip = lib.ponni_b200_debug_skip_arrive_ge
g = torch.Generator(device="cuda")
g.manual_seed(1)
x = torch.randn(rows, 128, generator=g, device="cuda").to(torch.bfloat16)
w = torch.randn(experts, 128, 256, generator=g, device="cuda").to(torch.bfloat16)
off = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
pb.expert_product(x, w, off)
pb.check_operators()
res = {}
assert skip(1) == 0
pb.expert_product(x, w, off)
try:
    pb.check_operators()
    res["status"] = 0
except pb.PonniError as e:
    res["status"] = e.status
assert skip(0) == 0
pb.check_operators()
y = pb.expert_product(x, w, off)
want, size = R.product(x, w, off)
R.check_sum(y, want, size, 128)
pb.check_operators()
print("RESULT " + json.dumps(res))
'''


@pytest.mark.parametrize("rows", [100, 4096])  # one CTA a tile, a pair of CTAs
def test_wait_runs_out(rows):
    assert os.path.exists(LIB), "build the test library: make -C ponni_b200/csrc"
    env = dict(os.environ, PONNI_B200_LIB=LIB, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CHILD, str(rows)], cwd=ROOT, env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    res = json.loads(next(s for s in r.stdout.splitlines() if s.startswith("RESULT "))[7:])
    assert res["status"] == 7
