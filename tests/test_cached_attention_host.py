"""How cached_attention's rows and keys are shared out, on the CPU."""
import ctypes
import json
import shutil
import subprocess
import sys

import pytest

from cache_cases import SHAPES
from test_kv_cache_host import c_arg
from titans_core.kernels import _lib


@pytest.mark.parametrize("window", [(1 << 30) + 1, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 63) - 8, (1 << 63) - 1])
def test_no_window(lib, window):
    """A window that is wider than any text is none, whatever its number."""
    n = ctypes.c_size_t(0)

    def size(w, **kw):
        arg = c_arg(**{"max_pages": 4096, "table_stride": 4096, **kw})
        assert lib.tmac_cached_attn_workspace(arg, 2, 1, 6, w, 2, ctypes.byref(n)) == 0
        return n.value

    for kw in ({}, {"format": 0}, {"max_pages": 1 << 20, "table_stride": 1 << 20}):
        assert size(window, **kw) == size(1 << 30, **kw) > 0


SHIM = r"""
#include <cstddef>
#include <cstdint>
#include <cstring>
struct dim3 { uint32_t x, y, z; };
static const void* host[8192];
static char names[8192][256], started[1 << 16];
static int n_names = 0;
static dim3 grid, block;
static size_t lds;
static void* on;
extern "C" void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*,
                                      int*) {
  if (n_names < 8192) host[n_names] = f, strncpy(names[n_names++], name, 255);
}
extern "C" int __hipPushCallConfiguration(dim3 g, dim3 b, size_t s, void* st) {
  grid = g, block = b, lds = s, on = st;
  return 0;
}
extern "C" int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* s, void** st) {
  *g = grid, *b = block, *s = lds, *st = on;
  return 0;
}
extern "C" int hipLaunchKernel(const void* f, dim3, dim3, void**, size_t, void*) {
  for (int i = 0; i < n_names; ++i)
    if (host[i] == f) strcat(started, names[i]), strcat(started, " ");
  return 0;
}
extern "C" int hipGetLastError() { return 0; }
extern "C" const char* registered(int i) { return i < n_names ? names[i] : nullptr; }
extern "C" const char* launched() { return started; }
extern "C" void forget() { started[0] = 0; }
"""

CHILD = r"""
import ctypes, json, struct, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
shim.registered.restype = shim.launched.restype = ctypes.c_char_p
P, L, A = ctypes.c_void_p, ctypes.c_int64, 1 << 20
names, i = [], 0
while shim.registered(i):
    names.append(shim.registered(i).decode())
    i += 1
calls = []
for B, T, H, heads, d, n, page in json.loads(sys.argv[3]):
    per = -(-n // page)
    for dtype in (0, 1, 2):
        for fmt in (0, 1, 2):
            cache = struct.pack("7Q2q7i4x", A, A, A, A, A, A, 0, B * per, per, heads, page, -(-d // 16) * 16, d, per, fmt, dtype)
            shim.forget()
            rc = lib.tmac_cached_attn(cache, P(A), (L * 3)(8, 8, 8), P(0), L(0), P(A), P(A), ctypes.c_size_t(1 << 60), B, T, H,
                                      L(1 << 30), 4, ctypes.c_float(1), P(0))
            calls.append([rc, shim.launched().decode().split()])
print(json.dumps([names, calls]))
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_kernel_has_a_shape(tmp_path):
    """The shapes that the GPU tests run (test_gpu_cached_attention_variants.py) reach every kernel in the library, in a
    process of its own whose launches only write their kernel's name down."""
    src, so = tmp_path / "shim.cpp", tmp_path / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(so), str(_lib.lib_path()), json.dumps(SHAPES)], capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    names, calls = json.loads(r.stdout)
    there = {n for n in names if "cached_attn" in n}
    assert len(there) > 50 and all(rc == 0 and started for rc, started in calls)
    assert there == {n for _, started in calls for n in started}
