"""The first products of a process, made by several host threads at once."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

FIRST = """
import threading
import torch
from pegainfer_b200 import ffi
from tests import fp8_ref as R
lib = ffi.lib()
lib.cuda_set_device(0)
lib.cublas_init()
M, K, N = 900, 700, 8
tokens = [3, 500] * (N // 2)
ops = []
for T in tokens:
    xc, xs = R.quant_rows(torch.randn(T, K, device="cuda"))
    wc, ws = R.quant_weights(torch.randn(M, K, device="cuda"))
    ops.append((xc, xs, wc, ws, torch.zeros(T, M, device="cuda"), torch.zeros(T, R.up(M, 16), dtype=torch.uint8, device="cuda"), torch.zeros(R.blocks(M), R.up(T, 4), device="cuda")))
streams = [torch.cuda.Stream() for _ in range(N)]
torch.cuda.synchronize()
gate, codes = threading.Barrier(N), [None] * N

def work(i):
    lib.cuda_set_device(0)
    xc, xs, wc, ws, y, c, s = ops[i]
    st = streams[i].cuda_stream
    w, x = (wc.data_ptr(), wc.shape[1], ws.data_ptr()), (xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1])
    gate.wait()
    codes[i] = (lib.pk_fp8_gemm(*w, *x, y.data_ptr(), 0, 1, M, tokens[i], K, st),
                lib.pk_fp8_gemm_gated(w[0], w[2], w[0], w[2], w[1], *x, c.data_ptr(), c.shape[1], s.data_ptr(), s.shape[1], M, tokens[i], K, 1, st))

threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
for t in threads:
    t.start()
for t in threads:
    t.join()
torch.cuda.synchronize()
assert codes == [(0, 0)] * N, codes
for i, T in enumerate(tokens):
    xc, xs, wc, ws, y, c, s = ops[i]
    want, size = R.product(xc, xs, wc, ws, T, M, K)
    assert ((y.double() - want).abs() <= size * R.SUM).all()
    off = want.abs() * size * R.SUM * 2 + (size * R.SUM) ** 2
    R.hold_rows(c, s, R.act(2, want, want), off)
print("all of them")
"""


@pytest.mark.parametrize("time", range(3))
def test_threads_that_make_their_first_product_together(time):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all of them" in run.stdout, run.stdout[-2000:] + run.stderr[-4000:]
