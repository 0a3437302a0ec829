"""Calls through the compiled binding while other Python threads have work: a call that
waits for room in the launch queue lets them run, a host callback in that queue among
them."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

# A host callback holds the stream up and needs Python to end, while the launches behind it
# are more than the queue takes. In a process of its own: a binding that keeps Python to
# itself never gets past this.
PROGRAM = r"""
import ctypes, glob, os, sys, time
sys.path[:0] = sys.argv[1:]
import torch, atflash
DEV = "cuda:0"
i = torch.zeros(1, dtype=torch.int32, device=DEV)
indptr = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
cache = torch.zeros((1, 16, 1, 128), dtype=torch.bfloat16, device=DEV)
x = torch.ones((1, 1, 128), dtype=torch.bfloat16, device=DEV)
w, cs = torch.ones(128, device=DEV), torch.ones((4, 64), device=DEV)
out = torch.empty_like(x)
calls = [lambda: atflash.append_paged_kv_cache(x, x, i, i, (cache, cache), i, indptr),
         lambda: atflash.qk_norm_rope(x, None, w, None, cs, cs, q_out=out)]
for f in calls:
    f()
torch.cuda.synchronize()
cudart = [l.split()[-1] for l in open("/proc/self/maps") if "libcudart" in l]
rt = ctypes.CDLL(cudart[0])
done = []

@ctypes.CFUNCTYPE(None, ctypes.c_void_p)
def callback(_):
    time.sleep(0.5)  # (which lets the main thread fill the queue)
    done.append(True)

sys.setswitchinterval(1.0)
for f in calls:
    done.clear()
    rc = rt.cudaLaunchHostFunc(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), callback, None)
    assert rc == 0, rc
    for _ in range(6000):
        f()
    torch.cuda.synchronize()
    assert done
assert atflash.check_device_errors() == 0
print("ran")
"""


def test_a_call_that_waits_for_the_queue_lets_other_threads_run():
    r = subprocess.run([sys.executable, "-c", PROGRAM, *sys.path], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.split() == ["ran"], r.stderr[-2000:]
