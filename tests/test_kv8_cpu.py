"""The 8-bit K/V cache's entry points without a GPU: what they refuse (before anything is launched), the sizes they give, and the plain form that the GPU tests
compare with."""
import ctypes as C
import math

import pytest
import torch

from pegainfer_b200 import ffi
from tests import kv8_ref as K

ROOM = (C.c_char * 4096)()
P = (C.addressof(ROOM) + 255) // 256 * 256  # an address that no refused call looks at


@pytest.fixture(scope="module")
def lib():
    from pegainfer_b200 import build
    build.build()
    return ffi.lib()


def test_page_bytes(lib):
    assert lib.pk_kv8_page_bytes(16, 8, 128, 128) == 8 * (16 * 256 + 16)
    assert lib.pk_kv8_page_bytes(48, 3, 32, 256) == 3 * 3 * (16 * 288 + 16)
    for bad in ((0, 8, 128, 128), (24, 8, 128, 128), (16, 0, 128, 128), (16, 8, 48, 128), (16, 8, 128, 288), (16, 8, 0, 32), (16, 8, 128, -32)):
        assert lib.pk_kv8_page_bytes(*bad) == -1


APPEND = dict(qkv=P, ld=2 * 64 + 2 * 128, bias=None, positions=P, slots=None, req=P, page_off=P, pages=P, q_out=P, cache=P, page_stride=2 * (16 * 128 + 16), page_size=16,
              heads=2, kv_heads=2, dim=64, vdim=64, dims=64, interleaved=0, freq=P, mag=1.0, tokens=1, f32=0, st=None)


@pytest.mark.parametrize("change", [
    dict(qkv=None), dict(positions=None), dict(req=None), dict(page_off=None), dict(pages=None), dict(q_out=None), dict(cache=None), dict(tokens=0), dict(tokens=-1),
    dict(heads=-1), dict(kv_heads=0), dict(dim=48), dict(vdim=40), dict(dim=288), dict(page_size=8), dict(page_size=0), dict(page_size=24), dict(dims=65), dict(dims=66),
    dict(dims=-2), dict(freq=None), dict(ld=383), dict(cache=P + 8), dict(page_stride=2 * (16 * 128 + 16) - 16), dict(page_stride=2 * (16 * 128 + 16) + 8),
    dict(page_size=32)])
def test_append_refuses(lib, change):
    assert lib.pk_kv8_append(*{**APPEND, **change}.values()) == -1


ATTEND = dict(q=P, cache=P, sink=None, slots=P, req=P, page_off=P, pages=P, out=P, page_stride=2 * (16 * 128 + 16), page_size=16, tokens=1, heads=4, kv_heads=2,
              dim=64, vdim=64, scale=0.125, options={}, workspace=P, workspace_bytes=1 << 40, f32=0, st=None)


def attend(lib, **change):
    a = {**ATTEND, **change}
    if a["options"] is not None:
        a["options"] = C.byref(ffi.Kv8Options(**{**dict(max_kv_len=100), **a["options"]}))
    return lib.pk_kv8_attention(*a.values())


@pytest.mark.parametrize("change", [
    dict(q=None), dict(cache=None), dict(slots=None), dict(req=None), dict(page_off=None), dict(pages=None), dict(out=None), dict(tokens=0), dict(heads=0), dict(heads=3),
    dict(kv_heads=0), dict(dim=16), dict(vdim=320), dict(page_size=40), dict(options=None), dict(options=dict(max_kv_len=0)), dict(options=dict(max_kv_len=2 ** 30 + 1)),
    dict(options=dict(window=-1)),
    dict(options=dict(softcap=-1.0)), dict(options=dict(max_q_len=-1)), dict(options=dict(out_ld=255)), dict(options=dict(mass=P)), dict(cache=P + 4),
    dict(page_stride=16 * 128 + 16), dict(options=dict(mass=P, mass_ld=100), workspace=None), dict(options=dict(mass=P, mass_ld=100), workspace_bytes=8),
    dict(options=dict(mass=P, mass_ld=100), workspace=P + 4), dict(options=dict(max_kv_len=100000), workspace=None)])
def test_attention_refuses(lib, change):
    assert attend(lib, **change) == -1


def test_workspace_bytes(lib):
    ask = lambda T, H=4, G=2, D=64, V=64, f32=0, **o: lib.pk_kv8_attention_workspace_bytes(T, H, G, D, V, C.byref(ffi.Kv8Options(**{**dict(max_kv_len=100), **o})), f32)  # noqa: E731
    assert ask(0) == -1 and ask(1, H=3) == -1 and ask(1, D=40) == -1 and ask(1, max_kv_len=0) == -1
    assert ask(1) >= 0 and ask(7, mass=P, mass_ld=5) >= 7 * 4 * 4 and ask(1, max_kv_len=1 << 20) > 0
    assert ask(256, 32, 8, max_kv_len=1 << 20, max_q_len=1, mass=P, mass_ld=1 << 20) < 1 << 28  # (the scores of all rows would be 34 GB)
    assert lib.pk_kv8_attention_workspace_bytes(1, 4, 2, 64, 64, None, 0) == -1


EVICT = dict(cache=P, page_stride=2 * (16 * 128 + 16), page_size=16, page_off=P, pages=P, lens=P, mass=P, mass_ld=100, new_page_off=P, new_pages=P + 512, new_lens=P + 768,
             new_mass=P + 256, new_mass_ld=50, kept=P, requests=1, kv_heads=2, dim=64, vdim=64, budget=50, keep_first=4, keep_recent=10, max_kv_len=100, st=None)


@pytest.mark.parametrize("change", [
    *(dict([(k, None)]) for k in ("cache", "page_off", "pages", "lens", "mass", "new_page_off", "new_pages", "new_lens", "new_mass", "kept")),
    dict(requests=0), dict(requests=70000), dict(kv_heads=0), dict(dim=8), dict(vdim=33), dict(budget=0), dict(keep_first=-1), dict(keep_recent=-1), dict(keep_first=41),
    dict(keep_first=2 ** 31 - 1, keep_recent=2 ** 31 - 1), dict(max_kv_len=0), dict(max_kv_len=101), dict(new_mass_ld=49), dict(new_mass=P), dict(new_pages=P), dict(new_lens=P),
    dict(max_kv_len=2 ** 30 + 1, mass_ld=2 ** 31),
    dict(page_size=20), dict(cache=P + 1), dict(page_stride=16)])
def test_evict_refuses(lib, change):
    assert lib.pk_kv8_evict(*{**EVICT, **change}.values()) == -1


def test_plain_codes():
    """every code stands for itself, a value is off by at most half a step, and the exponent is the least"""
    x = K.NUMBERS[torch.isfinite(K.NUMBERS)]
    assert torch.equal(K.NUMBERS[K.encode(x, 0).long()], x)
    y = torch.linspace(-448, 448, 20001, dtype=torch.float64)
    d = (K.NUMBERS[K.encode(y, 0).long()] - y).abs()
    assert (d <= torch.maximum(y.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10))).all()
    for a in (448.0, 448.1, 1e-30, 3e38, 1.0, 2.0 ** -133, 0.875, 0.8751):
        e = K.exponent(a)
        assert e == K.LOW or (a <= 448 * 2.0 ** e or e == K.HIGH) and a > 448 * 2.0 ** (e - 1)


def test_plain_record_goes_on():
    """a record filled token by token: the exponent grows, and what a token was rounded to stays within the steps that it met"""
    g = torch.Generator().manual_seed(1)
    c = K.Cache([40], 2, 32, 64, 16)
    k, v = (torch.randn(37, 2, w, generator=g).double() * torch.linspace(1, 30, 37)[:, None, None] for w in (32, 64))
    for t in range(37):
        K.append(c, 0, t, k[t:t + 1], v[t:t + 1])
    gk, gv = c.read(0, 37)
    for got, want in ((gk, k), (gv, v)):
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 0.03 * want.abs().max() / 448).all()
    rest = c.record(0, 2)[:, 5 * 16:8 * 16]  # slots 37 .. 39
    assert (rest == 0).all()
    w = torch.randn(1, 4, 32, generator=g)
    out, lse, weights, _ = K.attention(w, gk[:, :, :32], gv, torch.tensor([36]), 0.2)
    s = torch.einsum("hd,jhd->hj", w[0].double(), gk.repeat_interleave(2, 1)) * 0.2
    assert torch.allclose(weights[0], torch.softmax(s, -1)) and torch.allclose(lse[0], torch.logsumexp(s, -1))
    assert torch.allclose(out[0], torch.einsum("hj,jhd->hd", torch.softmax(s, -1), gv.repeat_interleave(2, 1)))
    assert math.isinf(K.attention(w, gk, gv, torch.tensor([-1]), 0.2)[1][0, 0])


def test_plain_fill_is_the_plain_append():
    g = torch.Generator().manual_seed(2)
    for n, page in ((1, 16), (16, 32), (53, 48)):
        k, v = torch.randn(n, 3, 32, generator=g).double(), torch.randn(n, 3, 64, generator=g).double()
        v[n // 2] = 0
        a, b = K.Cache([n], 3, 32, 64, page, seed=n), K.Cache([n], 3, 32, 64, page, seed=n)
        K.append(a, 0, 0, k, v)
        K.fill(b, 0, k, v)
        assert torch.equal(a.data, b.data)
