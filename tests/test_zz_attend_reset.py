"""The attention after cudaDeviceReset: a new context knows nothing of what an
earlier one was asked, so nothing about its kernels may be taken from there. In a
process of its own, whose context ends with it."""
import glob
import os
import subprocess
import sys

import pytest

import kvmret

pytestmark = pytest.mark.gpu

CHILD = """
import ctypes, sys
import kvmret
rt = ctypes.CDLL(sys.argv[1])

def ok(rc):
    if rc:
        raise SystemExit(f"runtime error {rc}")

def once(kind):
    p = []
    for n, byte in ((512, 0), (32 * 512, 0), (32 * 512, 0x3c), (512, 0), (1 << 22, 0)):
        a = ctypes.c_void_p()
        ok(rt.cudaMalloc(ctypes.byref(a), ctypes.c_size_t(n)))
        ok(rt.cudaMemset(a, byte, ctypes.c_size_t(n)))
        p.append(a.value)
    pages = kvmret.PagesDesc(p[1], p[2], 0, 0, 2, 16, 2, 128, kind, kvmret.TYPE_F16)
    at = kvmret.AttnArgs(q_dev=p[0], out_dev=p[3], n_q=1, n_head=2, scale=0.1, max_prefix=16)
    rc = kvmret.lib.kvmret_prefix_attn(ctypes.byref(pages), None, ctypes.byref(at), p[4], 1 << 22, None)
    if rc:
        raise SystemExit("attention: " + kvmret.lib.kvmret_last_error().decode())
    out = (ctypes.c_uint16 * 256)()
    ok(rt.cudaMemcpy(out, ctypes.c_void_p(p[3]), ctypes.c_size_t(512), 2))
    if any(x != 0x3c3c for x in out):  # equal weights of equal values
        raise SystemExit(f"wrong output {list(out)[:4]}")

for _ in range(3):
    once(kvmret.TYPE_F16)
    once(kvmret.TYPE_Q8_0)
    ok(rt.cudaDeviceReset())
print("fine")
"""


def test_attention_after_a_device_reset():
    import nvidia.cuda_runtime
    found = [p for d in nvidia.cuda_runtime.__path__ for p in glob.glob(os.path.join(d, "lib", "libcudart.so.*"))]
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(kvmret.__file__))))
    r = subprocess.run([sys.executable, "-c", CHILD, found[0]], env=env, capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
