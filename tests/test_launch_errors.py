"""CPU: a launch that fails ends in a status of the call, and leaves no error behind on the thread for the caller's next
check (torch's among them) to find.

The runtime's calls are replaced by fakes in a process of its own: the launch reports an error, nothing runs on a GPU, and
the addresses are never read."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

FAKES = """
static int pending;
static int failed(int e) { pending = e; return e; }
int cudaGetDevice(int* d) { *d = 0; return 0; }
int cudaDeviceGetAttribute(int* v, int what, int d) { *v = what == 16 ? 148 : 232448; return 0; }
int cudaFuncGetAttributes(void* a, const void* f) { for (int i = 0; i < 16; ++i) ((long*)a)[i] = 0; return 0; }
int cudaFuncSetAttribute(const void* f, int what, int v) { return FAIL_LIMIT ? failed(1) : 0; }
int cudaLaunchKernelExC(const void* c, const void* f, void** a) { return failed(1); }
int cudaGetDriverEntryPoint(const char* s, void** p, unsigned long long f, int* q) { *p = 0; return failed(1); }
int cudaGetDriverEntryPointByVersion(const char* s, void** p, unsigned v, unsigned long long f, int* q) { *p = 0; return failed(1); }
int cudaGetLastError(void) { int e = pending; pending = 0; return e; }
int cudaPeekAtLastError(void) { return pending; }
"""

PROGRAM = """
import ctypes as C, sys
lib, fakes = C.CDLL("flashsvd_b200/libflashsvd_b200.so"), C.CDLL(None)
class Kv8(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k8", "v8", "ks", "vs")] + [(n, C.c_int) for n in ("B", "Hk", "S", "Dh", "block")]
p, ll, f = C.c_void_p(1 << 20), C.c_longlong, C.c_float
size = C.c_size_t(1 << 24)
cache = C.byref(Kv8(p, p, p, p, 1, 2, 512, 128, 64))
def sample(V, dtype, B):
    return lib.fsvd_sample(p, ll(V), dtype, p, None, None, None, None, f(1), 0, f(1), f(0), p, p, B, V, None)
calls = {
    "rope": lambda: lib.fsvd_rope_qk(p, ll(128), p, ll(128), p, p, 64, 0, C.c_double(1), p, p, 4, 2, 2, 64, 0, None),
    "append": lambda: lib.fsvd_kv8_append(cache, p, p, ll(16384), ll(256), p, None, p, ll(16384), ll(256), p, p, 128, 0, C.c_double(1), 2, 64, p, size, None),
    "step": lambda: lib.fsvd_kv8_append(cache, p, p, ll(256), ll(256), p, None, None, ll(0), ll(0), None, None, 0, 0, C.c_double(1), 0, 1, p, size, None),
    "load": lambda: lib.fsvd_kv8_load(cache, 0, 8, None, 0, p, p, None),
    "attend": lambda: lib.fsvd_flash_decode_kv8(cache, p, p, 0, p, 2, f(0), p, size, None),
    "sample": lambda: sample(1000, 1, 2),
    "sample_long": lambda: sample(1 << 20, 0, 2),
}
print(calls[sys.argv[1]](), fakes.cudaPeekAtLastError())
"""


@pytest.mark.parametrize("fail_limit", [0, 1])
@pytest.mark.parametrize("call", ["rope", "append", "step", "load", "attend", "sample", "sample_long"])
def test_a_failed_launch_leaves_no_error_on_the_thread(call, fail_limit, tmp_path):
    so = tmp_path / "fakes.so"
    subprocess.run(["gcc", "-shared", "-fPIC", f"-DFAIL_LIMIT={fail_limit}", "-x", "c", "-", "-o", str(so)], input=FAKES, text=True, check=True)
    r = subprocess.run([sys.executable, "-c", PROGRAM, call], cwd=ROOT, env=dict(os.environ, LD_PRELOAD=str(so)),
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-800:]
    status, left = (int(x) for x in r.stdout.split())
    assert status < 0 and left == 0
