"""The 8-bit norm over the whole range of its entries: blocks whose largest entry lies below the least scale's before the root is applied and above it afterwards, and products with
the weight that pass fp32 although the normalised value does not."""
import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    return l


def rn(seed, *n):
    return torch.randn(*n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def hold(lib, x, w, eps, y=None, offset=0.0):
    T, W = x.shape
    codes, scales = torch.full((T, R.up(W, 16) + 16), 0x55, dtype=torch.uint8, device="cuda"), torch.full((R.blocks(W), R.up(T, 4) + 4), 7.0, device="cuda")
    s = x.double() + (0 if y is None else y.double())
    assert lib.pk_fp8_add_norm(None if y is None else y.data_ptr(), x.data_ptr(), int(x.dtype == F32), w.data_ptr(), offset, codes.data_ptr(), codes.shape[1], scales.data_ptr(),
                               scales.shape[1], W, T, eps, torch.cuda.current_stream().cuda_stream) == 0
    # less than 100 roundings of 2^-24, as for rows of ordinary entries; squares that leave fp32 below (each by 2^-150 at most) are nothing beside eps
    R.hold_rows(codes, scales, s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * (offset + w.double()), rel=2.0 ** -17)
    assert (codes[:, W:] == 0x55).all() and (scales[:, T:] == 7).all()


@pytest.mark.parametrize("W", [100, 1000, 2560, 2563, 9000])  # one piece a thread and two, in vectors and entry by entry
@pytest.mark.parametrize("x_f32", [False, True])
@pytest.mark.parametrize("eps", [1e-6, 1e-12])
def test_rows_of_tiny_entries(lib, W, x_f32, eps):
    """the root multiplies by up to 1 / sqrt(eps): rows from 2^-60 to 2^-125, in steps that pass 2^-100 before and after it"""
    steps = torch.arange(60, 126, device="cuda")
    x = (rn(W, len(steps), W) * 2.0 ** -steps.float()[:, None]).to(F32 if x_f32 else BF16)
    hold(lib, x, (1 + 0.3 * rn(1, W)).to(BF16), eps)


@pytest.mark.parametrize("W", [1000, 2560, 2563, 9000])
@pytest.mark.parametrize("x_f32", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_blocks_of_any_size_in_one_row(lib, W, x_f32, add):
    """every block has a size of its own, from 2^10 to 2^-130; the row's root lies anywhere between"""
    T = 40
    power = torch.randint(-130, 11, (T, R.blocks(W)), generator=torch.Generator().manual_seed(W)).cuda()
    power[:20] = power[:20].clamp(max=-12)  # (a row without a large block: the root multiplies)
    size = (2.0 ** power.float()).repeat_interleave(128, 1)[:, :W]
    x = (rn(2, T, W) * size).to(F32 if x_f32 else BF16)
    hold(lib, x, (0.2 * rn(3, W)).to(BF16), 1e-6, y=(rn(4, T, W) * size).to(BF16) if add else None, offset=1.0)


@pytest.mark.parametrize("W", [1000, 2563, 9000])
@pytest.mark.parametrize("x_f32", [False, True])
def test_weights_that_take_an_entry_past_fp32_before_the_root(lib, W, x_f32):
    """entries of 2^50, weights of 2^90 (their product is no fp32 number, the normalised one is), and weights of 2^-110"""
    x = (rn(5, 9, W) * 2.0 ** 50).to(F32 if x_f32 else BF16)
    w = rn(6, W)
    w[:128] *= 2.0 ** 90
    w[128:256] *= 2.0 ** -110
    w[256:384] *= 2.0 ** -128  # most of them bf16 numbers below 2^-126
    hold(lib, x, w.to(BF16), 1e-6)


@pytest.mark.parametrize("W", [300, 2560, 9000])
@pytest.mark.parametrize("x_f32", [False, True])
def test_rows_whose_squares_pass_fp32(lib, W, x_f32):
    """as the header has it: entries of 2^56 are held, a row whose sum of squares is no fp32 number has codes of zero, and its neighbours their own"""
    x = rn(7, 4, W).sign()
    x *= torch.tensor([1.0, 2.0 ** 56, 2.0 ** 66, 2.0 ** -20], device="cuda")[:, None]
    x = x.to(F32 if x_f32 else BF16)
    w = (1 + 0.3 * rn(8, W)).to(BF16)
    codes, scales = torch.zeros(4, R.up(W, 16), dtype=torch.uint8, device="cuda"), torch.zeros(R.blocks(W), 4, device="cuda")
    assert lib.pk_fp8_add_norm(None, x.data_ptr(), int(x_f32), w.data_ptr(), 0.0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), 4, W, 4, 1e-6,
                               torch.cuda.current_stream().cuda_stream) == 0
    assert (codes[2, :W] & 127 == 0).all() and (scales[:, 2] * 448 == R.LEAST).all()
    held = [0, 1, 3]
    v = x[held].double()
    R.hold_rows(codes[held], scales[:, held], v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w.double(), rel=2.0 ** -17)
