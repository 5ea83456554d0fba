"""Contexts of two devices in one process, without a GPU: in a child process a few functions of the HIP runtime stand in
for it and remember which device was current."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = r"""
#include <stdint.h>
#include <stdlib.h>
static int current;
int hipGetDeviceCount(int* n) { *n = 2; return 0; }
int hipSetDevice(int d) { current = d; return 0; }
int hipGetDevicePropertiesR0600(void* p, int d) { return 1; }
int hipStreamCreateWithFlags(void** s, unsigned f) { *s = malloc(1); return 0; }
int hipStreamSynchronize(void* s) { return 0; }
int hipStreamDestroy(void* s) { free(s); return 0; }
int hipGetSymbolAddress(void** p, const void* s) { static char x; *p = &x; return 0; }
int hipMalloc(void** p, size_t n) { int* q = malloc(4); *q = current; *p = q; return 0; }
int hipFree(void* p) { free(p); return 0; }
"""

CHILD = r"""
import ctypes as C, sys
C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)  # found before the runtime's own
from ai_amd import _native as N
a, b = N.Context(0), N.Context(1)
for ctx, device in ((a, 0), (b, 1), (b, 1), (a, 0)):
    p = N.vp()
    N.check(ctx.h, N.lib().fa_device_alloc(ctx.h, 1 << 20, C.byref(p)))
    assert C.cast(p, C.POINTER(C.c_int))[0] == device, (device, C.cast(p, C.POINTER(C.c_int))[0])
    N.check(ctx.h, N.lib().fa_device_free(ctx.h, p))
from ai_amd.kvcache import KVCache
with KVCache(1, 64, 64, ctx=b) as cache, KVCache(1, 64, 64, ctx=a) as other:
    for x, device in ((cache, 1), (other, 0)):
        assert C.cast(x._codes, C.POINTER(C.c_int))[0] == C.cast(x._scales, C.POINTER(C.c_int))[0] == device
b.close()
a.close()
print("done")
"""


def test_device_memory_is_the_contexts(tmp_path):
    src, lib = tmp_path / "hip.c", tmp_path / "libhip_stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(lib), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(lib)], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
