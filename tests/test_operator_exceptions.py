"""No C++ exception leaves the C entries of the feed-forward and optimiser calls: with
every `operator new` failing, a call that needs memory returns an error.  The calls end
before any CUDA call, so no GPU is needed."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

SHIM = r"""
#include <cstdlib>
#include <new>
static bool failing;
extern "C" __attribute__((visibility("default"))) void fail_new(int on) { failing = on; }
void* operator new(std::size_t n) {
    void* p = failing ? nullptr : std::malloc(n ? n : 1);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }
"""

CALLS = """
import ctypes as C
from zengpu_b200 import _lib as L
lib, shim = L.load(), C.CDLL(None)
FAKE = C.c_void_p(0x1000)  # not reached: the calls are refused first

array = L.CDeviceArray()
array.rank = 8  # of long sizes, so that the refusal's text needs memory
for i in range(8):
    array.shape[i] = 1000000000 + i
kernel, ref = L.CGemmKernel(), C.byref(array)
tensor = (L.AdamWTensor * 1)()
for name, _ in L.AdamWTensor._fields_[:-1]:
    setattr(tensor[0], name, None if name == "master" else 0x1000)
tensor[0].n = 8
hyper = L.AdamWHyper(1e-3, 0.9, 0.99, 1e-8, 0.0, 1)
ptrs, sizes = (C.c_void_p * 1)(0x1000), (C.c_uint64 * 1)(8)
out = [C.byref(L.CDeviceArray()) for _ in range(4)]
need = lib.zg_grad_norm_workspace_bytes(1)
calls = {
    "gated_ff": lambda: lib.zg_gemm_gated_ff(C.byref(kernel), FAKE, FAKE, 0, ref, ref, ref, ref,
                                             out[0], None, None),
    "gated_ff_backward": lambda: lib.zg_gemm_gated_ff_backward(
        C.byref(kernel), FAKE, FAKE, 0, *[ref] * 7, *out),
    "adamw": lambda: lib.zg_adamw(0, 0, 32, 1, tensor, C.byref(hyper), None, None, None, None),
    "grad_norm": lambda: lib.zg_grad_norm(0, 1, ptrs, sizes, 1.0, 0x1000, 0x1000, need, None),
}
for name, call in calls.items():
    shim.fail_new(1)
    rc = call()
    text = lib.zg_last_error()
    shim.fail_new(0)
    print(name, rc, text.decode(), flush=True)
"""


def test_no_exception_leaves_a_c_entry(tmp_path):
    source, shim = tmp_path / "shim.cpp", tmp_path / "shim.so"
    source.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(shim), str(source)], check=True)
    r = subprocess.run([sys.executable, "-c", CALLS], cwd=ROOT, capture_output=True, text=True,
                       timeout=120, env=os.environ | {"LD_PRELOAD": str(shim)})
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-2000:])
    lines = r.stdout.splitlines()
    assert len(lines) == 4, lines
    for line, name in zip(lines, ("gated_ff", "gated_ff_backward", "adamw", "grad_norm")):
        assert line.startswith(f"{name} ") and int(line.split()[1]) != 0, line
        assert line.split(" ", 2)[2] == f"{name}: std::bad_alloc", line
