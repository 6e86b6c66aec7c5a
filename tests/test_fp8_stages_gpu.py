"""The 8-bit products for few tokens give a stage of their ring back while the next block's copies wait for it: many calls over long reductions, each of whose blocks has a scale that tells it
from those that the same stage holds later.  (Given back before its scales were in registers, a block took the later one's in 8 of 60000 calls.)"""
import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
U8 = torch.uint8
CALLS = 15000  # of each: with one call in 7500 wrong, 60000 of a kernel would all be right once in 3000 times


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    return l


def operands(T, M, K, period):
    """one product of 1 a block, block b times 2^(b mod period): every sum is a whole number below 2^24 (a ring has twelve stages at most, and no multiple of the period)"""
    kb = R.blocks(K)
    xc, wc = torch.full((T, R.up(K, 16)), 0x38, dtype=U8, device="cuda"), torch.zeros(M, R.up(K, 16), dtype=U8, device="cuda")
    wc[:, 0:K:128] = 0x38
    power = 2.0 ** (torch.arange(kb, device="cuda") % period).float()
    return xc, power[:, None].repeat(1, R.up(T, 4)).contiguous(), wc, torch.ones(R.blocks(M), kb, device="cuda"), power.sum().item()


@pytest.mark.parametrize("T,M,K", [(28, 19000, 6000), (1, 9000, 6000), (48, 4096, 12288), (100, 2560, 9000)])
def test_products(lib, T, M, K):
    xc, xs, wc, ws, want = operands(T, M, K, 17)
    y, wrong = torch.zeros(T, M, device="cuda"), torch.zeros((), device="cuda", dtype=torch.int64)
    st = torch.cuda.current_stream().cuda_stream
    for _ in range(CALLS):
        assert lib.pk_fp8_gemm(wc.data_ptr(), wc.shape[1], ws.data_ptr(), xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], y.data_ptr(), 0, 1, M, T, K, st) == 0
        wrong += (y != want).sum()
    assert wrong.item() == 0 and lib.pk_b200_wait_errors() == 0


@pytest.mark.parametrize("T,M,K", [(28, 9728, 6000), (16, 2500, 9000), (60, 5000, 6000), (1, 12288, 4000)])
def test_gated_products(lib, T, M, K):
    xc, xs, wc, ws, each = operands(T, M, K, 13)
    value = (torch.tensor(each) * torch.tensor(each)).item()  # of fp32 numbers
    want = (torch.tensor(value, dtype=torch.float64) / 448).float().item()
    codes, scales = torch.zeros(T, R.up(M, 16), dtype=U8, device="cuda"), torch.zeros(R.blocks(M), R.up(T, 4), device="cuda")
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    st = torch.cuda.current_stream().cuda_stream
    for _ in range(CALLS):
        assert lib.pk_fp8_gemm_gated(wc.data_ptr(), ws.data_ptr(), wc.data_ptr(), ws.data_ptr(), wc.shape[1], xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], codes.data_ptr(),
                                     codes.shape[1], scales.data_ptr(), scales.shape[1], M, T, K, 1, st) == 0
        wrong += (scales[:, :T] != want).sum()
    assert wrong.item() == 0 and (codes[:, :M] == 0x7E).all() and lib.pk_b200_wait_errors() == 0
