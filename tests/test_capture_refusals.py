"""What calls under capture without work are told, without a GPU: in a child process a few functions of the HIP runtime
stand in for it, with every stream under capture."""
import subprocess
import sys

import test_two_devices as T

STAND_IN = T.STAND_IN + "int hipStreamIsCapturing(void* s, int* status) { *status = 1; return 0; }\n"

CHILD = r"""
import ctypes as C, sys
C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)  # found before the runtime's own
from ai_amd import _native as N
ctx, L = N.Context(0), N.lib()
P = 0x1000  # a buffer that no refused call follows
w = N.F8Matrix(P, P, 64, 128)
cache, batch = N.KvCache(P, P, 64, 8, 64), N.KvBatch(P, 64, P, P, 1, 1)
def attend(work, size):
    return L.fa_kv_attention_dev(ctx.h, C.byref(cache), C.byref(batch), 0, P, 512, 64, 8, 1, 0, 1.0, P, work, size)
def multiply(work, size):
    return L.fa_matmul_f8_dev(ctx.h, 8, 0, P, 128, C.byref(w), None, 0, P, 64, work, size)
def draw(work, size):
    return L.fa_sample_dev(ctx.h, 1, 100000, 0, P, 100000, None, P, P, None, work, size)
for call, size in ((attend, "fa_kv_attention_work"), (multiply, "fa_matmul_f8_work"), (draw, "fa_sample_work")):
    rc, text = call(None, 0), L.fa_last_error(ctx.h).decode()
    assert rc == N.FA_ERR_STATE and "captured" in text, (rc, text)
    assert size in text and "cannot be captured" not in text, text
rc, text = L.fa_matmul_f8(ctx.h, 8, 0, P, 128, C.byref(w), None, 0, P, 64), L.fa_last_error(ctx.h).decode()
assert rc == N.FA_ERR_STATE and "cannot be captured" in text, text
ctx.close()
print("done")
"""


def test_calls_that_need_work_say_so(tmp_path):
    src, lib = tmp_path / "hip.c", tmp_path / "libhip_stand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(lib), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(lib)], cwd=T.ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
