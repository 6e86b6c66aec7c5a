"""Gates far below zero in the 8-bit activations and gated products: SiLU and GELU are next to nothing there, but times a large factor they are numbers like any others."""
import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, U8, E4M3 = torch.bfloat16, torch.uint8, torch.float8_e4m3fn
#: The exponential's argument x (SiLU: z log2(e); GELU: 2 sqrt(2 / pi) (z + 0.044715 z^3) log2(e)) is taken in four roundings at most and matters up to 256, beyond which every result is
#: below half a step of the least scale: 256 ln(2) 4 2^-24 < 2^-14.4.  The special-function unit's results, 2^-22 each, and the products around them are nothing beside that.
REL = 2.0 ** -14


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    return l


def st():
    return torch.cuda.current_stream().cuda_stream


def every_bf16(lo, hi):
    """the negative bf16 numbers with magnitudes from lo to hi"""
    bits = [torch.tensor(v, dtype=BF16).view(torch.int16).item() for v in (lo, hi)]
    return -torch.arange(bits[0], bits[1] + 1, dtype=torch.int32).to(torch.int16).view(BF16).cuda()


def activate(lib, x, F, kind):
    T = len(x)
    codes, scales = torch.full((T, R.up(F, 16)), 0x55, dtype=U8, device="cuda"), torch.full((R.blocks(F), R.up(T, 4)), 7.0, device="cuda")
    assert lib.pk_fp8_act(x.data_ptr(), 0, kind, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], F, T, st()) == 0
    return codes, scales


def hold(codes, scales, v):
    """blocks with an entry past fp32 (no other lies near its end): NaN for scale and codes; the others as everywhere"""
    T, W = v.shape
    past = R.amax_rows(v) > 2.0 ** 128
    assert torch.equal(torch.isnan(scales[:, :T]).T, past)
    entries = past.repeat_interleave(128, 1)[:, :W]
    assert (codes[:, :W][entries] & 127 == 127).all()
    codes, scales = codes.clone(), scales.clone()
    codes[:, :W][entries] = 0
    scales[:, :T][past.T] = R.LEAST / R.LARGEST
    R.hold_rows(codes, scales, torch.where(entries, 0.0, v), rel=REL)


@pytest.mark.parametrize("kind,lo,hi", [(0, 60.0, 400.0), (3, 7.0, 30.0)])
@pytest.mark.parametrize("power", [0, 14, 20, 40, 64, 90, 110, 120, 127])
def test_act_of_far_gates_and_large_factors(lib, kind, lo, hi, power):
    """an entry a block, so that its scale tells the value"""
    a = every_bf16(lo, hi)
    b = torch.where(torch.arange(len(a), device="cuda") % 2 == 0, 1.99, -1.0) * 2.0 ** power
    x = torch.stack([a, b.to(BF16)], 1).contiguous()
    codes, scales = activate(lib, x, 1, kind)
    R.hold_rows(codes, scales, R.act(kind, x[:, :1].double(), x[:, 1:].double()), rel=REL)


@pytest.mark.parametrize("kind", [0, 3])
@pytest.mark.parametrize("sign", [1, -1])
def test_act_is_as_exact_as_the_header_says(lib, kind, sign):
    """SiLU: x is z times a constant, each within 2^-24 and 2^-26 of itself, so 2^x is off by 1.25 |z| 2^-24 of itself at most.  GELU: a square, two constants, a fused sum and a product make x,
    each within 2^-24 at most and on one side of zero: 4 |x| ln(2) 2^-24 <= 4 * 1.5958 |z + 0.044715 z^3| 2^-24.  Then the exponential and the quotient by the special-function unit
    (4 + 2), a sum, two products and the scale's product and rounding (1 + 2 + 3), in 2^-24."""
    z = -sign * every_bf16(2.0 ** -7, 80.0 if kind == 0 else 9.5)
    z = z[(z > 0) | (R.act(kind, z.double(), torch.ones_like(z).double()).abs() > 2.0 ** -99)]
    x = torch.stack([z, torch.ones_like(z)], 1).contiguous()
    codes, scales = activate(lib, x, 1, kind)
    want = R.act(kind, z.double(), torch.ones_like(z).double())
    got = R.values(codes[:, 0]) * scales[0, :len(z)].double()
    a = z.double().abs()
    size = 1.25 * a if kind == 0 else 4 * 1.5958 * (a + 0.044715 * a ** 3)
    assert ((got - want).abs() <= want.abs() * (size + 12) * 2.0 ** -24).all()


@pytest.mark.parametrize("kind,far", [(0, 90.0), (3, 10.5)])
@pytest.mark.parametrize("F", [128, 256, 1000, 333])
def test_act_of_far_gates_beside_others(lib, kind, far, F):
    """ordinary gates with small factors, far ones with large factors, in one block; and far ones alone"""
    T = 60
    g = torch.Generator(device="cuda").manual_seed(F + kind)
    rn = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    a, b = 2 * rn(T, F), rn(T, F)
    apart = torch.rand(T, F, generator=g, device="cuda") < 0.2
    apart[40:] = True
    a = torch.where(apart, -far * (1 + 0.3 * rn(T, F).abs()), a)
    b = torch.where(apart, b * 2.0 ** 125, b * 1e-3)
    x = torch.cat([a, b], 1).to(BF16).contiguous()
    codes, scales = activate(lib, x, F, kind)
    R.hold_rows(codes, scales, R.act(kind, x[:, :F].double(), x[:, F:].double()), rel=REL)


@pytest.mark.parametrize("T", [1, 20, 60, 300, 1100])
@pytest.mark.parametrize("act,lo,hi", [(0, 60.0, 240.0), (2, 7.0, 15.0)])
@pytest.mark.parametrize("power", [0, 20, 60, 100, 118])
def test_gated_products_of_far_gates_and_large_factors(lib, T, act, lo, hi, power):
    """one product a sum, of numbers that e4m3 has, so that gate and factor are known: z = token's 1 or 1.125 times the feature's number, u the same times 2^power"""
    M, K = 300, 16
    g = torch.Generator(device="cuda").manual_seed(T + power)
    number = lambda *n: lo + (hi - lo) * torch.rand(*n, generator=g, device="cuda")  # noqa: E731
    xc, w, u = (torch.zeros(n, K, dtype=U8, device="cuda") for n in (T, M, M))
    xc[:, 0] = torch.where(torch.arange(T, device="cuda") % 2 == 0, 1.0, 1.125).to(E4M3).view(U8)
    w[:, 0] = (-number(M)).to(E4M3).view(U8)
    w[::3, 0] = (number(len(w[::3])) / 20).to(E4M3).view(U8)  # (some ordinary gates, with the same factor in the first block, so that the others are below its least codes)
    w[128:, 0] = (-number(M - 128)).to(E4M3).view(U8)
    u[:, 0] = (1 + 200 * torch.rand(M, generator=g, device="cuda")).to(E4M3).view(U8)
    xs, ws, us = torch.ones(1, R.up(T, 4), device="cuda"), torch.ones(R.blocks(M), 1, device="cuda"), torch.full((R.blocks(M), 1), 2.0 ** power, device="cuda")
    codes, scales = torch.full((T, R.up(M, 16)), 0x55, dtype=U8, device="cuda"), torch.full((R.blocks(M), R.up(T, 4)), 7.0, device="cuda")
    assert lib.pk_fp8_gemm_gated(w.data_ptr(), ws.data_ptr(), u.data_ptr(), us.data_ptr(), K, xc.data_ptr(), K, xs.data_ptr(), xs.shape[1], codes.data_ptr(), codes.shape[1],
                                 scales.data_ptr(), scales.shape[1], M, T, K, act, st()) == 0
    (a, _), (b, _) = R.product(xc, xs, w, ws, T, M, K), R.product(xc, xs, u, us, T, M, K)
    hold(codes, scales, R.act((0, 2, 3)[act], a, b))  # (gates up to 12 * 1.125 times factors up to 201 * 1.125 * 2^118 pass 2^128)
