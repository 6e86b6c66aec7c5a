"""The 8-bit linear layers on a GPU against their definition in 64 bits (tests/fp8_ref.py): sizes around the blocks and the kernels' tiles, strides and addresses off their boundaries, entries
that are not finite, and the operators one behind the other as a feed-forward uses them."""
import math

import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, F64, U8 = torch.bfloat16, torch.float32, torch.float64, torch.uint8


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    return l


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum(int(k) * p for k, p in zip(key, (1, 1009, 10007, 100003, 7))))


def rn(g, *n):
    return torch.randn(*n, generator=g, device="cuda")


def st():
    return torch.cuda.current_stream().cuda_stream


def at(t, off):
    """the same numbers `off` elements behind an aligned address"""
    room = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
    room[off:] = t.reshape(-1)
    return room[off:].view(t.shape)


def out_rows(T, W, more=0):
    """codes and scales with room behind the width and the tokens, filled with what must stay"""
    return torch.full((T, R.up(W, 16) + 16 * more), 0x55, dtype=U8, device="cuda"), torch.full((R.blocks(W), R.up(T, 4) + 4 * more), 7.0, device="cuda")


def untouched(codes, scales, T, W):
    assert (codes[:, W:] == 0x55).all() and (scales[:, T:] == 7).all()


# ------------------------------------------------------------------ norm
NORM_SIZES = [(1, 1), (3, 5), (2, 128), (1, 130), (5, 1000), (9, 2048), (7, 2056), (300, 2560), (3, 4097), (2, 8200), (2, 16384)]


@pytest.mark.parametrize("T,W", NORM_SIZES)
@pytest.mark.parametrize("x_f32", [False, True])
@pytest.mark.parametrize("add", [True, False])
def test_norm(lib, T, W, x_f32, add):
    g = gen(T, W, x_f32, add)
    off = 1 if W == 1000 else 0  # (addresses that no vector starts at)
    x = at((3 * rn(g, T, W) * torch.exp(rn(g, W))).to(F32 if x_f32 else BF16), off)
    y, w = at(rn(g, T, W).to(BF16), off), at((1 + 0.3 * rn(g, W)).to(BF16), off)
    offset = float(W % 2)
    codes, scales = out_rows(T, W, more=W % 3)
    want = x.double() + y.double() if add else x.double()
    kept = x.clone()
    assert lib.pk_fp8_add_norm(y.data_ptr() if add else None, x.data_ptr(), int(x_f32), w.data_ptr(), offset, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1],
                               W, T, 1e-6, st()) == 0
    # one fp32 addition, one rounding when stored
    assert torch.equal(x, (kept.float() + y.float()).to(x.dtype) if add else kept)
    v = want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-6) * (offset + w.double())
    # the sum x + y is rounded by 2^-24 of itself; the mean of up to 16384 squares, added in chains of 64 and then pairwise, its root and its quotient, two products: less than 100 roundings
    # of 2^-24
    R.hold_rows(codes, scales, v, rel=2.0 ** -17)
    untouched(codes, scales, T, W)


@pytest.mark.parametrize("T,W", [(800, 333), (1500, 2049), (2000, 128), (900, 520)])
@pytest.mark.parametrize("x_f32", [False, True])
def test_norm_of_many_rows(lib, T, W, x_f32):
    g = gen(T, W, x_f32, 3)
    x, y, w = (2 * rn(g, T, W)).to(F32 if x_f32 else BF16), rn(g, T, W).to(BF16), (1 + 0.3 * rn(g, W)).to(BF16)
    codes, scales = out_rows(T, W, more=1)
    want = x.double() + y.double()
    stored = (x.float() + y.float()).to(x.dtype)
    assert lib.pk_fp8_add_norm(y.data_ptr(), x.data_ptr(), int(x_f32), w.data_ptr(), 0.0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], W, T, 1e-6, st()) == 0
    assert torch.equal(x, stored)
    R.hold_rows(codes, scales, want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-6) * w.double(), rel=2.0 ** -17)  # as in test_norm
    untouched(codes, scales, T, W)


def norm_of(lib, x, w=None):
    T, W = x.shape
    w = torch.ones(W, device="cuda").to(BF16) if w is None else w
    codes, scales = out_rows(T, W)
    assert lib.pk_fp8_add_norm(None, x.data_ptr(), int(x.dtype == F32), w.data_ptr(), 0.0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], W, T, 1e-6, st()) == 0
    return codes, scales


def test_norm_of_rows_that_are_not_finite(lib):
    x = rn(gen(1), 6, 300).to(BF16)
    x[1] = 0
    x[2, 200] = math.nan
    x[4, 5] = math.inf
    x[5, 128:256] = 0
    codes, scales = norm_of(lib, x)
    v = x[[0, 1, 3, 5]].double()
    R.hold_rows(codes[[0, 1, 3, 5]], scales[:, [0, 1, 3, 5]], v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6), rel=2.0 ** -18)
    assert (codes[1, :300] == 0).all() and (scales[:, 1] * 448 == R.LEAST).all()
    # a NaN is in every entry of its row; an infinity leaves NaN where it stands and zeros elsewhere
    assert torch.isnan(scales[:, 2]).all() and (codes[2, :300] & 127 == 127).all()
    assert torch.isnan(scales[0, 4]) and (codes[4, :128] & 127 == 127).all() and (codes[4, 128:300] & 127 == 0).all()


# ------------------------------------------------------------------ activations
@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("T,F,pad", [(1, 1, 0), (5, 127, 1), (3, 128, 0), (33, 136, 8), (2, 9728, 0), (7, 1000, 4), (300, 520, 0)])
def test_act(lib, kind, T, F, pad):
    g = gen(kind, T, F)
    n = F * (1 if kind in (1, 4) else 2)
    x = at((3 * rn(g, T, n + pad)).to(BF16), 3 if F == 1000 else 0)
    codes, scales = out_rows(T, F, more=T % 2)
    assert lib.pk_fp8_act(x.data_ptr(), n + pad if pad else 0, kind, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], F, T, st()) == 0
    a, b = x[:, :F].double(), x[:, F:2 * F].double()
    # |x| <= 20 here: the exponential's argument is rounded by 20 * 1.5 * 2^-24 (GELU: 8 times that, its cube), the special-function unit's results by 2^-22
    R.hold_rows(codes, scales, R.act(kind, a, b), rel=2.0 ** -16)
    untouched(codes, scales, T, F)


@pytest.mark.parametrize("kind", range(5))
def test_act_reads_nothing_behind_a_row(lib, kind):
    """rows of an odd width whose strides are whole vectors: NaN wherever nothing may be read"""
    T, F = 5, 125
    n = F * (1 if kind in (1, 4) else 2)
    x = torch.full((T, R.up(n, 8)), math.nan, device="cuda").to(BF16)
    x[:, :n] = rn(gen(kind, 8), T, n).to(BF16)
    codes, scales = out_rows(T, F)
    assert lib.pk_fp8_act(x.data_ptr(), x.shape[1], kind, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], F, T, st()) == 0
    R.hold_rows(codes, scales, R.act(kind, x[:, :F].double(), x[:, F:2 * F].double()), rel=2.0 ** -16)


@pytest.mark.parametrize("f32", [False, True])
def test_weights_read_nothing_behind_a_row(lib, f32):
    w = torch.full((130, 136), math.nan, device="cuda").to(F32 if f32 else BF16)
    w[:, :130] = rn(gen(f32, 9), 130, 130).to(w.dtype)
    codes, scales = torch.zeros(130, 144, dtype=U8, device="cuda"), torch.empty(2, 2, device="cuda")
    assert lib.pk_fp8_weights(w.data_ptr(), int(f32), 136, codes.data_ptr(), 144, scales.data_ptr(), 130, 130, st()) == 0
    R.hold_weights(codes, scales, w[:, :130].double())


def test_act_of_entries_that_are_not_finite(lib):
    F = 400
    x = rn(gen(3), 5, F).to(BF16)
    x[0, 130], x[1, 3], x[2, 399], x[3, 256:384] = math.nan, -math.inf, math.inf, 0
    x[4] *= 1e30
    codes, scales = out_rows(5, F)
    assert lib.pk_fp8_act(x.data_ptr(), 0, 4, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], F, 5, st()) == 0
    bad = torch.zeros(4, 5, dtype=torch.bool)
    bad[1, 0] = bad[0, 1] = bad[3, 2] = True
    assert torch.equal(torch.isnan(scales[:, :5]).cpu(), bad)
    for b in range(4):
        part = slice(b * 128, min(F, b * 128 + 128))
        ok = ~bad[b].cuda()
        R.hold_rows(codes[ok][:, part], scales[b:b + 1, :5][:, ok], x[ok][:, part].double())
        assert (codes[~ok][:, part] & 127 == 127).all()


def test_act_of_every_bf16_gate(lib):
    """gates from the least to the largest number: nothing overflows on the way"""
    a = torch.arange(0, 0x7F80, 1, dtype=torch.int32).to(torch.int16).view(BF16).cuda()
    a = torch.cat([a, -a]).view(-1, 1)
    for kind in (0, 2, 3):
        one = torch.where(a.abs() > 1e20, 1e-30, 1.0).to(BF16)
        x = torch.cat([a, one], 1).contiguous()
        codes, scales = out_rows(len(a), 1)
        assert lib.pk_fp8_act(x.data_ptr(), 0, kind, codes.data_ptr(), 16, scales.data_ptr(), scales.shape[1], 1, len(a), st()) == 0
        v = R.act(kind, a.double(), one.double())
        got = R.values(codes[:, :1]) * scales[:, :len(a)].double().T
        # the argument of the exponential, up to 88, is rounded by 88 * 1.45 * 2^-24 in the worst case (GELU 4 times that); the code by 2^-4; below 2^-100 by the least scale's steps;
        # and results of less than 2^-120 may be zero
        assert ((got - v).abs() <= v.abs() * (2.0 ** -4 + 2.0 ** -14) + R.LEAST / 448 * 2.0 ** -9).all()


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("M,W,pad", [(1, 1, 0), (3, 5, 0), (128, 128, 0), (129, 130, 2), (1000, 264, 8), (5, 1000, 0), (300, 2560, 0)])
@pytest.mark.parametrize("f32", [False, True])
def test_weights(lib, M, W, pad, f32):
    g = gen(M, W, f32)
    w = at((rn(g, M, W + pad) * torch.exp(rn(g, W + pad))).to(F32 if f32 else BF16), 1 if M == 5 else 0)
    codes = torch.full((M, R.up(W, 16) + 16), 0x55, dtype=U8, device="cuda")
    scales = torch.empty(R.blocks(M), R.blocks(W), device="cuda")
    assert lib.pk_fp8_weights(w.data_ptr(), int(f32), W + pad if pad else 0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), M, W, st()) == 0
    R.hold_weights(codes, scales, w[:, :W].double())
    assert (codes[:, W:] == 0x55).all()


def test_weights_of_extreme_blocks(lib):
    w = torch.zeros(384, 256, device="cuda")
    w[0, 0], w[5, 200] = 3e38, 1e-44                       # the largest numbers, the least
    w[128:256, :128], w[200, 130] = 2.0 ** -90, math.nan
    w[256:, 128:] = rn(gen(4), 128, 128)
    codes, scales = torch.zeros(384, 256, dtype=U8, device="cuda"), torch.empty(3, 2, device="cuda")
    assert lib.pk_fp8_weights(w.data_ptr(), 1, 0, codes.data_ptr(), 256, scales.data_ptr(), 384, 256, st()) == 0
    assert torch.isnan(scales).nonzero().tolist() == [[1, 1]] and (codes[128:256, 128:] & 127 == 127).all()
    w[128:256, 128:] = 0
    codes[128:256, 128:], scales[1, 1] = 0, R.LEAST / 448
    R.hold_weights(codes, scales, w.double())


# ------------------------------------------------------------------ products
def operands(T, M, K, g, wild=False, pad=0):
    x, w = rn(g, T, K) * torch.exp(rn(g, K)), rn(g, M, K) / math.sqrt(K)
    xc, xs = R.quant_rows(x, R.up(K, 16) + 16 * pad, R.up(T, 4) + 4 * pad)
    wc, ws = R.quant_weights(w, R.up(K, 16) + 16 * pad)
    if wild:  # scales as they never come from a quantisation: any sign and size, zero among them
        ws = ws * torch.exp(3 * rn(g, *ws.shape)) * torch.sign(rn(g, *ws.shape))
        ws[0, 0] = 0
    return xc, xs, wc, ws


def gemm(lib, ops, T, M, K, f32=False, ld=0, off=0, stream=None, y=None):
    xc, xs, wc, ws = ops
    ld_y = ld or M
    if y is None:
        y = torch.full((T * ld_y + off,), 7.0, dtype=F32 if f32 else BF16, device="cuda")[off:].view(T, ld_y)
    assert lib.pk_fp8_gemm(wc.data_ptr(), wc.shape[1], ws.data_ptr(), xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], y.data_ptr(), ld, int(f32), M, T, K, stream or st()) == 0
    return y


def near(y, want, size):
    """one rounding of the result, and the sum's"""
    eps = torch.finfo(y.dtype).eps / 2
    bad = (y.double() - want).abs() > want.abs() * eps + size * R.SUM
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4].tolist(), y[bad][:4].tolist(), want[bad][:4].tolist())


TOKENS = [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 255, 256, 257, 700]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("M,K", [(1, 16), (100, 128), (129, 1), (257, 1000), (1000, 2560), (2560, 129)])
def test_gemm(lib, T, M, K):
    for f32 in (False, True):
        ops = operands(T, M, K, gen(T, M, K, f32), pad=T % 2)
        near(gemm(lib, ops, T, M, K, f32), *R.product(*ops, T, M, K))


@pytest.mark.parametrize("T,M,K", [(129, 300, 3333), (200, 513, 4096), (300, 500, 8000), (777, 130, 5000), (1000, 64, 2560), (1024, 100, 9000), (1025, 100, 9000), (513, 40, 128), (70, 19000, 200),
                                   (64, 19000, 300), (33, 37889, 128), (16, 20001, 700)])
def test_gemm_of_many_parts_and_tiles(lib, T, M, K):
    """long reductions of few features are cut into parts however many tokens there are; many features go two tiles to a CTA, in waves"""
    for f32 in (False, True):
        ops = operands(T, M, K, gen(T, M, K))
        near(gemm(lib, ops, T, M, K, f32, ld=M + 1), *(torch.nn.functional.pad(v, (0, 1), value=7.0 * i) for i, v in zip((1, 0), R.product(*ops, T, M, K))))


@pytest.mark.parametrize("T", [1, 7, 40, 90, 300])
@pytest.mark.parametrize("M,ld,off", [(256, 264, 0), (512, 515, 0), (300, 300, 1), (64, 0, 3), (640, 641, 2)])
@pytest.mark.parametrize("f32", [False, True])
def test_gemm_rows_of_any_stride(lib, T, M, ld, off, f32):
    K = 400
    ops = operands(T, M, K, gen(T, M, ld, off))
    y = gemm(lib, ops, T, M, K, f32, ld, off)
    near(y[:, :M], *R.product(*ops, T, M, K))
    assert (y[:, M:] == 7).all()


@pytest.mark.parametrize("T,M,K,ld,off", [(257, 4100, 4000, 4104, 0), (300, 4095, 3900, 0, 0), (200, 8100, 1000, 8101, 1),  # as few waves of narrow tiles as of wide ones,
                                          (300, 9610, 300, 9616, 0), (333, 6145, 2560, 0, 1), (520, 9611, 400, 9700, 0), (150, 24500, 130, 0, 0),  # fewer than of the narrowest,
                                          (2100, 24500, 300, 24504, 0), (430, 16383, 520, 0, 0)])  # fewer of the widest than of any
@pytest.mark.parametrize("f32", [False, True])
def test_gemm_of_tiles_of_any_width(lib, T, M, K, ld, off, f32):
    ops = operands(T, M, K, gen(T, M, K), wild=T % 2 == 1)
    y = gemm(lib, ops, T, M, K, f32, ld=ld, off=off)
    near(y[:, :M], *R.product(*ops, T, M, K))
    assert (y[:, M:] == 7).all()


def with_nan_behind(codes, K):
    codes = codes.clone()
    codes[:, K:] = 0x7f
    return codes


@pytest.mark.parametrize("T", [3, 50, 120, 300])
@pytest.mark.parametrize("K", [1, 5, 127, 129, 515])
def test_products_use_nothing_behind_the_width(lib, T, K):
    M = 200
    xc, xs, wc, ws = operands(T, M, K, gen(T, K, 6), pad=1)
    ops = with_nan_behind(xc, K), xs, with_nan_behind(wc, K), ws
    near(gemm(lib, ops, T, M, K), *R.product(*ops, T, M, K))
    hold_gated(*gated(lib, ops, ops[2:], T, M, K, 1), ops, ops[2:], T, M, K, 1)


@pytest.mark.parametrize("T", [3, 50, 120, 400])
def test_gemm_with_scales_of_any_size_and_sign(lib, T):
    M, K = 1200, 1100
    ops = operands(T, M, K, gen(T, 5), wild=True)
    near(gemm(lib, ops, T, M, K, True), *R.product(*ops, T, M, K))


@pytest.mark.parametrize("T,M,K", [(1, 24576, 4096), (32, 2560, 9728), (64, 151936, 256), (512, 6144, 2560), (1111, 9728, 2560), (4096, 2560, 4096)])
def test_gemm_of_model_sizes(lib, T, M, K):
    ops = operands(T, M, K, gen(T, M))
    near(gemm(lib, ops, T, M, K), *R.product(*ops, T, M, K))


@pytest.mark.parametrize("T", [4, 40, 128, 300])
def test_gemm_keeps_what_is_not_finite_apart(lib, T):
    """a token whose scale is NaN, a block of weights, a code: NaN where they are read and nowhere else; the other tokens keep their bits"""
    M, K = 700, 500
    xc, xs, wc, ws = operands(T, M, K, gen(T))
    before = gemm(lib, (xc, xs, wc, ws), T, M, K)
    xs[2, 1], ws[3, 0] = math.nan, math.nan
    xc[3, 444] = 0x7F
    y = gemm(lib, (xc, xs, wc, ws), T, M, K)
    bad = torch.zeros(T, M, dtype=torch.bool, device="cuda")
    bad[1], bad[3], bad[:, 384:512] = True, True, True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], before[~bad])


@pytest.mark.parametrize("T,M,K", [(28, 19000, 3000), (40, 9728, 2500), (100, 2560, 2900), (300, 19000, 2800)])
def test_gemm_takes_every_block_with_its_own_scale(lib, T, M, K):
    """a power of two for a block, so that the sum tells which were taken: exact, every time of many"""
    kb = R.blocks(K)
    xc, wc = torch.full((T, R.up(K, 16)), 0x38, dtype=U8, device="cuda"), torch.zeros(M, R.up(K, 16), dtype=U8, device="cuda")
    wc[:, 0:K:128] = 0x38  # one product of 1 a block
    xs, ws = (2.0 ** torch.arange(kb, device="cuda").float())[:, None].repeat(1, R.up(T, 4)).contiguous(), torch.ones(R.blocks(M), kb, device="cuda")
    y, wrong = torch.zeros(T, M, device="cuda"), torch.zeros((), device="cuda", dtype=torch.int64)
    for _ in range(1500):
        gemm(lib, (xc, xs, wc, ws), T, M, K, True, y=y)
        wrong += (y != 2.0 ** kb - 1).sum()
    assert wrong.item() == 0


@pytest.mark.parametrize("T", [5, 64, 130])
def test_gemm_gives_a_token_its_bits_whatever_the_others_hold(lib, T):
    M, K = 513, 1300
    xc, xs, wc, ws = operands(T, M, K, gen(T, 9))
    a = gemm(lib, (xc, xs, wc, ws), T, M, K, True)
    xs[:, 1:T] *= 3e20
    b = gemm(lib, (xc, xs, wc, ws), T, M, K, True)
    assert torch.equal(a[0], b[0])


# ------------------------------------------------------------------ gated products
def gated(lib, ops, w2, T, M, K, act, more=0):
    xc, xs, wc, ws = ops
    codes, scales = out_rows(T, M, more)
    assert lib.pk_fp8_gemm_gated(wc.data_ptr(), ws.data_ptr(), w2[0].data_ptr(), w2[1].data_ptr(), wc.shape[1], xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], codes.data_ptr(),
                                 codes.shape[1], scales.data_ptr(), scales.shape[1], M, T, K, act, st()) == 0
    return codes, scales


def hold_gated(codes, scales, ops, w2, T, M, K, act):
    (a, sa), (b, sb) = R.product(*ops, T, M, K), R.product(ops[0], ops[1], *w2, T, M, K)
    kind = (0, 2, 3)[act]
    v = R.act(kind, a, b)
    # |act'| <= 1.13; the activation's own error as in test_act (arguments here up to a few hundred: 2^-14)
    ea, eb = sa * R.SUM, sb * R.SUM
    off = 1.13 * ea * (b.abs() + eb) + R.act(kind, a, torch.ones_like(a)).abs() * eb
    R.hold_rows(codes, scales, v, off, rel=2.0 ** -14)


@pytest.mark.parametrize("T", [1, 16, 17, 31, 64, 65, 128, 200, 256, 300])
@pytest.mark.parametrize("M,K", [(1, 16), (100, 300), (128, 128), (129, 700), (1000, 2560)])
def test_gated(lib, T, M, K):
    g = gen(T, M, K)
    ops = operands(T, M, K, g, pad=T % 2)
    w2 = operands(1, M, K, g, pad=T % 2)[2:]
    act = (T + M) % 3
    codes, scales = gated(lib, ops, w2, T, M, K, act, more=T % 2)
    hold_gated(codes, scales, ops, w2, T, M, K, act)
    untouched(codes, scales, T, M)


@pytest.mark.parametrize("T,M,K", [(100, 640, 8192), (130, 128, 4000), (300, 257, 5000), (1000, 128, 3333), (64, 19000, 256)])
def test_gated_of_many_parts_and_tiles(lib, T, M, K):
    g = gen(T, M, K)
    ops = operands(T, M, K, g)
    w2 = operands(1, M, K, g)[2:]
    codes, scales = gated(lib, ops, w2, T, M, K, T % 3, more=1)
    hold_gated(codes, scales, ops, w2, T, M, K, T % 3)
    untouched(codes, scales, T, M)


@pytest.mark.parametrize("T,M,K", [(1, 12288, 4096), (32, 9728, 2560), (700, 9728, 2560)])
@pytest.mark.parametrize("act", [0, 1, 2])
def test_gated_of_model_sizes(lib, T, M, K, act):
    g = gen(T, M, act)
    ops = operands(T, M, K, g)
    w2 = operands(1, M, K, g)[2:]
    hold_gated(*gated(lib, ops, w2, T, M, K, act), ops, w2, T, M, K, act)


@pytest.mark.parametrize("T", [5, 90, 300])
def test_gated_with_one_matrix_for_both(lib, T):
    ops = operands(T, 200, 400, gen(T, 78))
    hold_gated(*gated(lib, ops, ops[2:], T, 200, 400, 1), ops, ops[2:], T, 200, 400, 1)


@pytest.mark.parametrize("T", [7, 300])
def test_gated_halves_of_one_array(lib, T):
    """gate and up quantised as one array of rows, where a half is whole blocks"""
    M, K = 256, 500
    g = gen(T, 79)
    xc, xs, wc, ws = operands(T, 2 * M, K, g)
    ops, w2 = (xc, xs, wc[:M], ws[:M // 128]), (wc[M:], ws[M // 128:])
    hold_gated(*gated(lib, ops, w2, T, M, K, 2), ops, w2, T, M, K, 2)


@pytest.mark.parametrize("T", [6, 100])
def test_gated_keeps_what_is_not_finite_apart(lib, T):
    M, K = 300, 300
    g = gen(T, 77)
    xc, xs, wc, ws = operands(T, M, K, g)
    w2 = operands(1, M, K, g)[2:]
    c0, s0 = gated(lib, (xc, xs, wc, ws), w2, T, M, K, 0)
    xs[1, 2], w2[1][1, 2] = math.nan, math.nan
    c1, s1 = gated(lib, (xc, xs, wc, ws), w2, T, M, K, 0)
    bad = torch.zeros(3, T, dtype=torch.bool, device="cuda")
    bad[:, 2], bad[1] = True, True
    assert torch.equal(torch.isnan(s1[:, :T]), bad) and torch.equal(s1[:, :T][~bad], s0[:, :T][~bad])
    every = bad.T.repeat_interleave(128, 1)[:, :M]
    assert (c1[:, :M][every] & 127 == 127).all() and torch.equal(c1[:, :M][~every], c0[:, :M][~every])


# ------------------------------------------------------------------ together
class FeedForward:
    """norm -> gate and up -> down, with weights quantised once"""

    def __init__(self, lib, H, F, seed):
        g = gen(seed, H, F)
        self.lib, self.H, self.F = lib, H, F
        self.norm = (1 + 0.1 * rn(g, H)).to(BF16)
        self.gate, self.up, self.down = ((rn(g, *n) / math.sqrt(n[1])).to(BF16) for n in ((F, H), (F, H), (H, F)))
        self.q = [self.quantise(w) for w in (self.gate, self.up, self.down)]

    def quantise(self, w):
        M, K = w.shape
        codes, scales = torch.zeros(M, R.up(K, 16), dtype=U8, device="cuda"), torch.zeros(R.blocks(M), R.blocks(K), device="cuda")
        assert self.lib.pk_fp8_weights(w.data_ptr(), 0, 0, codes.data_ptr(), codes.shape[1], scales.data_ptr(), M, K, st()) == 0
        return codes, scales

    def buffers(self, T):
        return dict(T=T, n=out_rows(T, self.H), h=out_rows(T, self.F), y=torch.zeros(T, self.H, device="cuda").to(BF16), both=torch.zeros(T, 2 * self.F, device="cuda").to(BF16))

    def step(self, x, y, b, fused=True, stream=None):
        """x (fp32 residual) += y, then the layer of x into b["y"]"""
        lib, H, F, T, s = self.lib, self.H, self.F, b["T"], stream or st()
        (gc, gs), (uc, us), (dc, ds) = self.q
        (nc, ns), (hc, hs) = b["n"], b["h"]
        rc = lib.pk_fp8_add_norm(y.data_ptr(), x.data_ptr(), 1, self.norm.data_ptr(), 0.0, nc.data_ptr(), nc.shape[1], ns.data_ptr(), ns.shape[1], H, T, 1e-6, s)
        if fused:
            rc |= lib.pk_fp8_gemm_gated(gc.data_ptr(), gs.data_ptr(), uc.data_ptr(), us.data_ptr(), gc.shape[1], nc.data_ptr(), nc.shape[1], ns.data_ptr(), ns.shape[1], hc.data_ptr(),
                                        hc.shape[1], hs.data_ptr(), hs.shape[1], F, T, H, 0, s)
        else:  # the same by two products and the activation; gate and up side by side in one array of rows
            for k, (c, sc) in enumerate(((gc, gs), (uc, us))):
                rc |= lib.pk_fp8_gemm(c.data_ptr(), c.shape[1], sc.data_ptr(), nc.data_ptr(), nc.shape[1], ns.data_ptr(), ns.shape[1], b["both"].data_ptr() + 2 * F * k, 2 * F, 0, F, T, H, s)
            rc |= lib.pk_fp8_act(b["both"].data_ptr(), 0, 0, hc.data_ptr(), hc.shape[1], hs.data_ptr(), hs.shape[1], F, T, s)
        rc |= lib.pk_fp8_gemm(dc.data_ptr(), dc.shape[1], ds.data_ptr(), hc.data_ptr(), hc.shape[1], hs.data_ptr(), hs.shape[1], b["y"].data_ptr(), 0, 0, H, T, F, s)
        assert rc == 0
        return b["y"]

    def plain(self, x, y):
        x = x.double() + y.double()
        n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * self.norm.double()
        return R.act(0, n @ self.gate.double().T, n @ self.up.double().T) @ self.down.double().T


@pytest.mark.parametrize("T", [1, 20, 150, 520])
@pytest.mark.parametrize("fused", [True, False])
def test_feed_forward(lib, T, fused):
    f = FeedForward(lib, 520, 1400, T)
    x, y = rn(gen(T, 1), T, 520), rn(gen(T, 2), T, 520).to(BF16)
    want = f.plain(x, y)
    got = f.step(x, y, f.buffers(T), fused).double()
    # every code is off by at most 2^-4 of its value, by 2^-4 / sqrt(3) at random: rows and weights of both products and the rows between, about sqrt(2 + 2 + 2 + 1) * 0.036 * 0.6 of the result
    # (entries lie anywhere within a step); twice that is a mistake
    assert (got - want).norm() <= 0.12 * want.norm()


def test_feed_forward_captured_and_replayed_on_new_inputs(lib):
    f = FeedForward(lib, 256, 640, 5)
    pairs = []
    for T in (3, 200):  # two graphs, each with buffers of its own
        b, x, y = f.buffers(T), torch.zeros(T, 256, device="cuda"), torch.zeros(T, 256, device="cuda").to(BF16)
        f.step(x, y, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f.step(x, y, b)
        pairs.append((T, b, x, y, graph))
    streams = [torch.cuda.Stream() for _ in pairs]
    for round_ in range(3):
        data = []
        for T, b, x, y, graph in pairs:
            x.copy_(rn(gen(T, round_), T, 256))
            y.copy_(rn(gen(T, round_, 1), T, 256))
            data.append((x.clone(), y.clone()))
        torch.cuda.synchronize()
        for s, (T, b, x, y, graph) in zip(streams, pairs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (x0, y0), (T, b, x, y, graph) in zip(data, pairs):
            got = b["y"].clone()
            assert torch.equal(got, f.step(x0, y0, f.buffers(T)))


def test_calls_on_several_streams_at_once(lib):
    """products of all kernels side by side: nothing is shared"""
    shapes = [(1, 2560, 4096), (40, 1000, 2560), (120, 4096, 640), (300, 2560, 640)]
    ops = [operands(*s, gen(*s)) for s in shapes]
    want = [gemm(lib, o, *s) for o, s in zip(ops, shapes)]
    streams = [torch.cuda.Stream() for _ in range(8)]
    ys = [torch.zeros_like(want[i % 4]) for i in range(40)]
    torch.cuda.synchronize()
    for i, y in enumerate(ys):
        gemm(lib, ops[i % 4], *shapes[i % 4], stream=streams[i % 8].cuda_stream, y=y)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(ys))
    assert lib.pk_b200_wait_errors() == 0


def test_with_dependent_launches(lib):
    """each launch may begin before the one before it has ended: the products wait for their rows"""
    f = FeedForward(lib, 1024, 2560, 8)
    x, y = rn(gen(8, 1), 9, 1024), rn(gen(8, 2), 9, 1024).to(BF16)
    want = f.step(x.clone(), y, f.buffers(9)).clone()
    lib.pk_b200_set_pdl(1)
    try:
        for _ in range(20):
            assert torch.equal(f.step(x.clone(), y, f.buffers(9)), want)
    finally:
        lib.pk_b200_set_pdl(0)


@pytest.mark.parametrize("fused", [True, False])
def test_with_dependent_launches_of_a_prompt(lib, fused):
    """the same through the kernels for many tokens, and for rows of odd widths"""
    f = FeedForward(lib, 999, 1300, 9)
    x, y = rn(gen(9, 1), 300, 999), rn(gen(9, 2), 300, 999).to(BF16)
    want = f.step(x.clone(), y, f.buffers(300), fused).clone()
    lib.pk_b200_set_pdl(1)
    try:
        for _ in range(20):
            assert torch.equal(f.step(x.clone(), y, f.buffers(300), fused), want)
    finally:
        lib.pk_b200_set_pdl(0)


FIRST = """
import torch
from pegainfer_b200 import ffi
from tests import fp8_ref as R
lib = ffi.lib()
lib.cuda_set_device(0)
lib.cublas_init()
cases = []
for T in (4, 500):
    xc, xs = R.quant_rows(torch.randn(T, 700, device="cuda"))
    wc, ws = R.quant_weights(torch.randn(900, 700, device="cuda"))
    y = torch.zeros(T, 900, device="cuda")
    cases.append((T, xc, xs, wc, ws, y))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    s = torch.cuda.current_stream().cuda_stream
    for T, xc, xs, wc, ws, y in cases:
        assert lib.pk_fp8_gemm(wc.data_ptr(), wc.shape[1], ws.data_ptr(), xc.data_ptr(), xc.shape[1], xs.data_ptr(), xs.shape[1], y.data_ptr(), 0, 1, 900, T, 700, s) == 0
graph.replay()
torch.cuda.synchronize()
for T, xc, xs, wc, ws, y in cases:
    want, size = R.product(xc, xs, wc, ws, T, 900, 700)
    assert ((y.double() - want).abs() <= size * R.SUM).all()
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stdout[-2000:] + run.stderr[-4000:]
