"""Linear layers in 8 bits in plain 64-bit arithmetic, and the bounds that the kernels' results are held to (both test files of the 8-bit linear layers)."""
import math

import torch

F64, U8, E4M3 = torch.float64, torch.uint8, torch.float8_e4m3fn
BLOCK, LARGEST, LEAST = 128, 448.0, 2.0 ** -100
#: an fp32 sum of products by the tensor core: the 33 numbers of a step (32 products, which are exact, and the sum so far) lose at most 2^-23 of the largest of them each, and a block has
#: four steps; then two scales and an addition a block in fp32.  Relative to the sum of the products' magnitudes: 4 * 33 * 2^-23 < 2^-15.
SUM = 2.0 ** -15


def blocks(n):
    return -(-n // BLOCK)


def up(n, to):
    return -(-n // to) * to


def numbers(device="cpu"):
    """what each code stands for"""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = math.nan if e == 15 and m == 7 else math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=F64, device=device)


def values(codes):
    return numbers(codes.device)[codes.long()]


def half_step(q):
    """half the distance of the codes around q (|q| <= 448)"""
    e = torch.frexp(q.abs().clamp(max=LARGEST)).exponent.clamp(min=-5)
    return torch.ldexp(torch.ones_like(q), e - 5)


def row_scales(scales, T, W):
    """[blocks, ld_s] -> [T, W]"""
    return scales[:, :T].double().T.repeat_interleave(BLOCK, 1)[:, :W]


def weight_scales(scales, M, W):
    return scales.double().repeat_interleave(BLOCK, 0)[:M].repeat_interleave(BLOCK, 1)[:, :W]


def amax_rows(v):
    T, W = v.shape
    return torch.nn.functional.pad(v.abs(), (0, blocks(W) * BLOCK - W)).view(T, -1, BLOCK).amax(-1)


def amax_weights(w):
    M, W = w.shape
    p = torch.nn.functional.pad(w.abs(), (0, blocks(W) * BLOCK - W, 0, blocks(M) * BLOCK - M))
    return p.view(blocks(M), BLOCK, blocks(W), BLOCK).amax((1, 3))


def hold_rows(codes, scales, v, off=None, rel=2.0 ** -20):
    """codes [T, ld >= W] and scales [blocks, ld_s >= T] of the rows v [T, W] (64 bits), computed to within `off` (same shape, absolute) and `rel` of themselves: the scale
    is the largest magnitude's within that and fp32's own two roundings, a code is nearest to its entry within it"""
    T, W = v.shape
    off = (torch.zeros_like(v) if off is None else off) + v.abs() * rel
    am, worst = amax_rows(v), amax_rows(off)
    s = scales[:, :T].double().T
    assert ((s * LARGEST - am.clamp(min=LEAST)).abs() <= worst + am.clamp(min=LEAST) * 2.0 ** -22).all()
    _hold(codes[:, :W], s.repeat_interleave(BLOCK, 1)[:, :W], v, off)


def hold_weights(codes, scales, w):
    M, W = w.shape
    am = amax_weights(w).clamp(min=LEAST)
    assert ((scales.double() * LARGEST - am).abs() <= am * 2.0 ** -23).all()
    _hold(codes[:, :W], weight_scales(scales, M, W), w, torch.zeros_like(w))


def _hold(codes, s, v, off):
    got = values(codes)
    assert torch.isfinite(got).all()
    q = v / s
    assert ((got - q).abs() <= half_step(q) * (1 + 2.0 ** -20) + off / s + q.abs() * 2.0 ** -23).all()


def quant_rows(v, ld=None, ld_s=None):
    """operands of a product: any codes and scales do, these are the format's own"""
    T, W = v.shape
    ld, ld_s = ld or up(W, 16), ld_s or up(T, 4)
    s = amax_rows(v.double()).clamp(min=LEAST) / LARGEST
    codes, scales = torch.full((T, ld), 0x7F, dtype=U8, device=v.device), torch.full((blocks(W), ld_s), math.nan, device=v.device)  # NaN wherever nothing may be read
    scales[:, :T] = s.T.float()
    codes[:, :W] = (v.double() / row_scales(scales, T, W)).float().to(E4M3).view(U8)
    return codes, scales


def quant_weights(w, ld=None):
    M, W = w.shape
    ld = ld or up(W, 16)
    scales = (amax_weights(w.double()).clamp(min=LEAST) / LARGEST).float()
    codes = torch.full((M, ld), 0x7F, dtype=U8, device=w.device)
    codes[:, :W] = (w.double() / weight_scales(scales, M, W)).float().to(E4M3).view(U8)
    return codes, scales


def product(xc, xs, wc, ws, T, M, K):
    """x w^T in 64 bits and the sum of its products' magnitudes"""
    x, w = values(xc[:, :K]) * row_scales(xs, T, K), values(wc[:, :K]) * weight_scales(ws, M, K)
    return x @ w.T, x.abs() @ w.abs().T


def hold_product(y, want, size):
    """y within one rounding of the result and the sum's bound (`size`: of its products' magnitudes); NaN is within nothing"""
    ok = (y.double() - want).abs() <= want.abs() * (torch.finfo(y.dtype).eps / 2) + size * SUM
    assert ok.all(), ((~ok).sum().item(), (~ok).nonzero()[:4].tolist(), y[~ok][:4].tolist(), want[~ok][:4].tolist())


def act(kind, a, b=None):
    """pk_fp8_act's kinds (GELU by the logistic function: 1 + tanh of a large negative number loses its bits in 64 of them too)"""
    f = torch.nn.functional
    return {0: lambda: f.silu(a) * b, 1: lambda: f.relu(a) ** 2, 2: lambda: f.relu(a) * b, 3: lambda: a * torch.sigmoid(math.sqrt(8 / math.pi) * (a + 0.044715 * a ** 3)) * b,
            4: lambda: a}[kind]()
