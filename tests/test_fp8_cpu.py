"""The entry points of the 8-bit linear layers without a GPU: what they refuse (before anything is launched), and the plain form that the GPU tests compare with."""
import ctypes as C

import pytest
import torch

from pegainfer_b200 import ffi
from tests import fp8_ref as R

ROOM = (C.c_char * 4096)()
P = (C.addressof(ROOM) + 255) // 256 * 256  # an address that no refused call looks at
Q = P + 1024


@pytest.fixture(scope="module")
def lib():
    from pegainfer_b200 import build
    build.build()
    return ffi.lib()


NORM = dict(y=P, x=P + 512, x_f32=0, w=P, offset=0.0, codes=Q, ld=256, scales=P, ld_s=4, width=256, tokens=3, eps=1e-6, st=None)


@pytest.mark.parametrize("change", [dict(x=None), dict(w=None), dict(codes=None), dict(scales=None), dict(y=P + 512), dict(width=0), dict(width=-8), dict(tokens=0), dict(tokens=-1),
                                    dict(ld=240), dict(ld=264), dict(codes=Q + 8), dict(ld_s=0), dict(ld_s=6), dict(tokens=5), dict(scales=P + 4)])
def test_norm_refuses(lib, change):
    assert lib.pk_fp8_add_norm(*{**NORM, **change}.values()) == -1


def test_norm_has_a_widest_row(lib):
    assert lib.pk_fp8_add_norm(*{**NORM, "width": 16385, "ld": 16400}.values()) == -2


ACT = dict(x=P, ld_in=512, kind=0, codes=Q, ld=256, scales=P, ld_s=4, F=256, tokens=3, st=None)


@pytest.mark.parametrize("change", [dict(x=None), dict(codes=None), dict(scales=None), dict(kind=-1), dict(kind=5), dict(F=0), dict(tokens=0), dict(ld_in=511), dict(kind=4, ld_in=255),
                                    dict(ld_in=-512), dict(ld=255), dict(ld=250), dict(codes=Q + 4), dict(ld_s=2), dict(ld_s=5), dict(scales=P + 8), dict(codes=P)])
def test_act_refuses(lib, change):
    assert lib.pk_fp8_act(*{**ACT, **change}.values()) == -1


def test_act_counts_its_blocks(lib):
    assert lib.pk_fp8_act(*{**ACT, "F": 2 ** 30, "ld": 2 ** 30, "ld_in": 0, "tokens": 2 ** 20, "ld_s": 2 ** 20}.values()) == -2


WEIGHTS = dict(w=P, w_f32=0, ld_w=256, codes=Q, ld=256, scales=P, rows=3, width=256, st=None)


@pytest.mark.parametrize("change", [dict(w=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(width=0), dict(ld_w=255), dict(ld_w=-256), dict(ld=255), dict(ld=264),
                                    dict(codes=Q + 1), dict(codes=P)])
def test_weights_refuse(lib, change):
    assert lib.pk_fp8_weights(*{**WEIGHTS, **change}.values()) == -1


def test_weights_count_their_blocks(lib):
    assert lib.pk_fp8_weights(*{**WEIGHTS, "rows": 2 ** 31 - 1, "width": 2 ** 30, "ld_w": 0, "ld": 2 ** 30}.values()) == -2


GEMM = dict(w=P, ld_w=256, w_scales=P, x=P, ld_x=256, x_scales=P, ld_xs=4, y=Q, ld_y=0, y_f32=0, M=64, N=4, K=256, st=None)
OPERANDS = [dict(x=None), dict(x_scales=None), dict(N=0), dict(K=0), dict(N=-1), dict(K=-1), dict(ld_w=255), dict(ld_w=264), dict(ld_x=240), dict(ld_x=257),
            dict(x=P + 8), dict(ld_xs=3), dict(ld_xs=6), dict(N=5), dict(x_scales=P + 4), dict(ld_w=2 ** 39)]


@pytest.mark.parametrize("change", OPERANDS + [dict(w=None), dict(w_scales=None), dict(y=None), dict(M=0), dict(M=-4), dict(w=P + 8), dict(ld_y=63), dict(ld_y=-64)])
def test_gemm_refuses(lib, change):
    assert lib.pk_fp8_gemm(*{**GEMM, **change}.values()) == -1


GATED = dict(w_gate=P, gate_scales=P, w_up=P, up_scales=P, ld_w=256, x=P, ld_x=256, x_scales=P, ld_xs=4, codes=Q, ld=64, scales=P, ld_s=4, F=64, N=4, K=256, act=0, st=None)


@pytest.mark.parametrize("change", OPERANDS + [dict(w_gate=None), dict(gate_scales=None), dict(w_up=None), dict(up_scales=None), dict(w_up=P + 4), dict(codes=None), dict(scales=None), dict(F=0),
                                               dict(codes=Q + 8), dict(ld=48), dict(ld=72), dict(ld_s=0), dict(ld_s=7), dict(scales=P + 4), dict(act=-1), dict(act=3), dict(codes=P)])
def test_gated_refuses(lib, change):
    assert lib.pk_fp8_gemm_gated(*{**GATED, **change}.values()) == -1


def test_products_count_in_31_bits(lib):
    assert lib.pk_fp8_gemm(*{**GEMM, "M": 2 ** 30 + 1}.values()) == -2
    assert lib.pk_fp8_gemm(*{**GEMM, "N": 2 ** 30 + 1, "ld_xs": 2 ** 30 + 4}.values()) == -2
    assert lib.pk_fp8_gemm(*{**GEMM, "K": 2 ** 30 + 1, "ld_w": 2 ** 31, "ld_x": 2 ** 31}.values()) == -2
    assert lib.pk_fp8_gemm_gated(*{**GATED, "F": 2 ** 30 + 1, "ld": 2 ** 31}.values()) == -2


def test_the_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double().nan_to_num(nan=1e9), R.values(codes).nan_to_num(nan=1e9))


def test_the_plain_form_holds_to_its_own_bounds_and_a_mistake_does_not():
    v = torch.randn(5, 300, dtype=torch.float64) * torch.exp(2 * torch.randn(300, dtype=torch.float64))
    v[3, 128:256] = 0
    codes, scales = R.quant_rows(v)
    R.hold_rows(codes, scales, v)
    w = torch.randn(200, 300, dtype=torch.float64)
    wc, ws = R.quant_weights(w)
    R.hold_weights(wc, ws, w)
    for plant in (lambda c, s: c[2].__setitem__(7, c[2, 7] ^ 2), lambda c, s: s[1].__setitem__(4, s[1, 4] * 1.001), lambda c, s: c[0].__setitem__(299, 0x7F)):
        c, s = codes.clone(), scales.clone()
        plant(c, s)
        with pytest.raises(AssertionError):
            R.hold_rows(c, s, v)
