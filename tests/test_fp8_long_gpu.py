"""The 8-bit linear layers on arrays whose offsets pass 32 bits: rows at the far end are those of the formulas, and rows of all zeros before them stay zeros."""
import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
LAST = 5  # rows that hold something


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    yield l
    torch.cuda.empty_cache()


def rn(seed, *n):
    return torch.randn(*n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def st():
    return torch.cuda.current_stream().cuda_stream


def out_rows(T, W):
    return torch.empty(T, R.up(W, 16), dtype=U8, device="cuda"), torch.empty(R.blocks(W), R.up(T, 4), device="cuda")


def hold(codes, scales, v, T, rel):
    R.hold_rows(codes[-LAST:], scales[:, T - LAST:T], v, rel=rel)
    assert (codes[-LAST - 3:-LAST] == 0).all() and (scales[:, :T - LAST] * 448 == R.LEAST).all()


def test_norm(lib):
    T, W = 270000, 16000
    assert T * W > 2 ** 32
    x, w = torch.zeros(T, W, dtype=BF16, device="cuda"), (1 + 0.3 * rn(1, W)).to(BF16)
    x[-LAST:] = rn(2, LAST, W).to(BF16)
    codes, scales = out_rows(T, W)
    assert lib.pk_fp8_add_norm(None, x.data_ptr(), 0, w.data_ptr(), 0.0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], W, T, 1e-6, st()) == 0
    v = x[-LAST:].double()
    hold(codes, scales, v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w.double(), T, 2.0 ** -17)


def test_act(lib):
    T, F = 440000, 9999
    assert T * F > 2 ** 32
    x = torch.zeros(T, 2 * F, dtype=BF16, device="cuda")
    x[-LAST:] = rn(3, LAST, 2 * F).to(BF16)
    codes, scales = out_rows(T, F)
    assert lib.pk_fp8_act(x.data_ptr(), 0, 0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], F, T, st()) == 0
    hold(codes[:, :F], scales, R.act(0, x[-LAST:, :F].double(), x[-LAST:, F:].double()), T, 2.0 ** -16)


def test_weights(lib):
    M, W = 270001, 16000
    w = torch.zeros(M, W, dtype=BF16, device="cuda")
    w[-LAST:] = rn(4, LAST, W).to(BF16)
    codes, scales = torch.empty(M, W, dtype=U8, device="cuda"), torch.empty(R.blocks(M), R.blocks(W), device="cuda")
    assert lib.pk_fp8_weights(w.data_ptr(), 0, 0, codes.data_ptr(), W, scales.data_ptr(), M, W, st()) == 0
    R.hold_weights(codes[-(M % 128):], scales[-1:], w[-(M % 128):].double())
    assert (codes[M // 2] == 0).all() and (scales[:-1] * 448 == R.LEAST).all()


@pytest.mark.parametrize("T,M,K", [(31000, 151936, 130), (900, 5000000, 16)])
def test_product(lib, T, M, K):
    """rows of the output beyond 2^32 entries"""
    assert T * M > 2 ** 32
    xc, xs = R.quant_rows(rn(5, T, K))
    wc, ws = R.quant_weights(rn(6, M, K))
    y = torch.empty(T, M, dtype=BF16, device="cuda")
    assert lib.pk_fp8_gemm(wc.data_ptr(), wc.shape[1], ws.data_ptr(), xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], y.data_ptr(), 0, 0, M, T, K, st()) == 0
    for rows in (slice(0, 2), slice(T - LAST, T)):
        n = len(range(T)[rows])
        R.hold_product(y[rows], *R.product(xc[rows], xs[:, rows], wc, ws, n, M, K))


def test_product_of_weights_beyond_32_bits(lib):
    T, M, K = 3, 300000, 16000
    xc, xs = R.quant_rows(rn(7, T, K))
    wc, ws = torch.zeros(M, K, dtype=U8, device="cuda"), torch.ones(R.blocks(M), R.blocks(K), device="cuda")
    last = R.quant_weights(rn(8, 96, K))
    wc[-96:], ws[-1] = last[0], last[1][0]  # (the last block of 300000 rows has 96)
    y = torch.empty(T, M, device="cuda")
    assert lib.pk_fp8_gemm(wc.data_ptr(), K, ws.data_ptr(), xc.data_ptr(), K, xs.data_ptr(), xs.shape[1], y.data_ptr(), 0, 1, M, T, K, st()) == 0
    R.hold_product(y[:, -96:], *R.product(xc, xs, *last, T, 96, K))
    assert (y[:, :-96] == 0).all()


def test_gated_product(lib):
    T, M, K = 40000, 110000, 128
    assert T * M > 2 ** 32
    xc, xs = R.quant_rows(rn(9, T, K))
    (wc, ws), (uc, us) = R.quant_weights(rn(10, M, K)), R.quant_weights(rn(11, M, K))
    codes, scales = out_rows(T, M)
    assert lib.pk_fp8_gemm_gated(wc.data_ptr(), ws.data_ptr(), uc.data_ptr(), us.data_ptr(), K, xc.data_ptr(), K, xs.data_ptr(), xs.shape[1], codes.data_ptr(), codes.shape[1],
                                 scales.data_ptr(), scales.shape[1], M, T, K, 1, st()) == 0
    for rows in (slice(0, 2), slice(T - LAST, T)):
        n = len(range(T)[rows])
        (a, sa), (b, sb) = R.product(xc[rows], xs[:, rows], wc, ws, n, M, K), R.product(xc[rows], xs[:, rows], uc, us, n, M, K)
        off = sa * R.SUM * (b.abs() + sb * R.SUM) + a.abs() * sb * R.SUM
        R.hold_rows(codes[rows], scales[:, rows], R.act(2, a, b), off)
