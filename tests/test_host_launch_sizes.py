"""Grids at the largest sizes that the token operators' entry points accept: a launch takes fewer than 2^32 threads. On the CPU, in a
process of its own whose launches only write their grid down; and refusals."""
import json
import shutil
import subprocess
import sys

import pytest

from titans_core.kernels import _lib

SHIM = r"""
#include <cstddef>
#include <cstdint>
struct dim3 { uint32_t x, y, z; };
static uint64_t threads[256];
static int n = 0;
extern "C" int __hipPushCallConfiguration(dim3 g, dim3 b, size_t, void*) {
  if (n < 256) threads[n++] = uint64_t(g.x) * b.x * (uint64_t(g.y) * b.y) * (uint64_t(g.z) * b.z);
  return 1;  // the launch itself is left out
}
extern "C" int hipGetLastError() { return 0; }
extern "C" int launches(uint64_t* out) {
  const int had = n;
  for (int i = 0; i < n; ++i) out[i] = threads[i];
  n = 0;
  return had;
}
"""

CHILD = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
P, I, L, Z, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
A, BIG, WS = P(1 << 20), 1 << 30, Z(1 << 62)
out = []
def call(name, *args):
    rc = getattr(lib, name)(*args)
    got = (ctypes.c_uint64 * 256)()
    n = shim.launches(got)
    out.append([name, rc, list(got[:n])])
for V in (1, 50000, BIG):
    for d in (1, 8, 640):
        for B, T, Np in ((1, BIG, 0), (BIG, 1, 0), (BIG // 2, 1, 1), (1, 1, BIG - 1)):
            n_pos = max(T, 1)
            call("tmac_embed_fwd", A, P(0), A, L(d), A, L(d), A, L(d), A, A, WS, I(B), I(T), I(Np), I(d), L(V), L(n_pos),
                 F(1), I(1), P(0))
            call("tmac_embed_fwd", A, P(0), A, L(d), P(0), L(0), A, L(d), A, P(0), Z(0), I(B), I(T), I(Np), I(d), L(V),
                 L(0), F(1), I(1), P(0))
            for pos in (P(0), A):
                for lists in (P(0), A):
                    call("tmac_embed_bwd", A, pos, lists, A, L(d), A, A, A if Np else P(0), A, WS, I(B), I(T), I(Np), I(d),
                         L(V), L(BIG), F(1), I(1), P(0))
for V in (1, 129, 128000, 1 << 28):
    for top in (0, min(V, 64)):
        for B, T in ((1, BIG), (BIG, 1), (1, 1), (2, 100)):
            call("tmac_logprob_fwd", A, L(V), L(V), A, L(-100), A, A, I(top), A, A, A, A, WS, I(B), I(T), L(V), I(1), P(0))
            call("tmac_logprob_bwd", A, L(V), L(V), A, L(-100), A, A, A, L(1), A, L(1), A, I(B), I(T), L(V), I(1), P(0))
            call("tmac_logprob_mean_bwd", A, L(V), L(V), A, L(-100), A, A, A, I(1), A, I(B), I(T), L(V), I(1), P(0))
    for M in (1, 64, 65, 8192, 1 << 26, (1 << 26) + 1, BIG):
        for K in (64, 640, 1024):
            call("tmac_head_logprob", A, L(K), A, L(K), A, L(-100), A, A, I(M), L(V), I(K), A, WS, I(1), P(0))
call("tmac_logprob_mean", A, A, L(-100), I(BIG), A, I(1), A, P(0))
print(json.dumps(out))
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_launch_of_2_to_the_32_threads(tmp_path):
    src, so = tmp_path / "shim.cpp", tmp_path / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(so), str(_lib.lib_path())], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stderr
    calls = json.loads(r.stdout)
    assert len(calls) > 300
    for i, (name, rc, threads) in enumerate(calls):
        assert rc == 0 and threads, (i, name, rc)
        assert all(0 < t < 1 << 32 for t in threads), (i, name, threads)


def test_prefix_rows_are_counted_without_sequences():
    """More prefix rows than the kernels count in 32 bits are refused for an empty batch too, whose gradient writes
    them."""
    import torch

    import titans_core as tc
    w = torch.zeros(5, 8)
    with pytest.raises(ValueError, match="rows"):
        tc.token_embedding(torch.zeros(0, 3, dtype=torch.long), w, prefix=w[:1].expand((1 << 32) + 3, 8))


def test_loss_gradient_argument_errors(lib):
    fake = 1 << 20
    # z, stride_b, stride_t, targets, ignore, stats, neg_inv, g_loss, g_dtype, dz, B, T, V, dtype, stream
    ok = [fake, 0, 100, fake, -100, fake, fake, fake, 1, fake, 1, 4, 100, 0, None]
    for at, value, want in ((0, None, -1), (3, None, -1), (5, None, -1), (6, None, -1), (7, None, -1), (9, None, -1),
                            (8, 3, -4), (0, fake + 2, -5), (9, fake + 1, -5), (2, -1, -2), (10, -1, -2), (12, 0, -2),
                            (13, 3, -4)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_logprob_mean_bwd(*bad) == want, (at, value)
    empty = list(ok)
    empty[10] = 0
    assert lib.tmac_logprob_mean_bwd(*empty) == 0
    assert lib.tmac_logprob_mean(fake, fake, -100, (1 << 30) + 1, fake, 1, fake, None) == -2
