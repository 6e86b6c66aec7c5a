"""The 8-bit K/V cache on the GPU (csrc/kv8*.cu) against 64 bits (tests/kv8_ref.py): the append record by record, attention over ragged batches with every option,
the accumulated weights, the eviction, and all of them together as a decoding loop."""
import ctypes as C
import math

import pytest
import torch

from pegainfer_b200 import ffi
from tests import kv8_ref as K

pytestmark = pytest.mark.gpu
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = "cuda"


@pytest.fixture(scope="module")
def lib():
    l = ffi.lib()
    l.cuda_set_device(0)
    l.cublas_init()
    return l


def i32(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ calls
def call_append(lib, c, qkv, positions, req, H, dims=0, interleaved=False, freq=None, mag=1.0, slots=None, bias=None, ld=None):
    T = positions.numel()
    q = torch.full((T + 1, max(1, H * c.D)), 7.0, dtype=qkv.dtype, device=DEV)
    rc = lib.pk_kv8_append(qkv.data_ptr(), ld or qkv.shape[1], ptr(bias), positions.data_ptr(), ptr(slots), req.data_ptr(), c.page_off.data_ptr(), c.pages.data_ptr(),
                           q.data_ptr() if H else None, c.data.data_ptr(), c.stride, c.page, H, c.G, c.D, c.V, dims, int(interleaved), ptr(freq), mag, T,
                           int(qkv.dtype == F32), stream())
    assert rc == 0
    assert (q[T] == 7.0).all()
    return q[:T, :H * c.D].view(T, H, c.D)


def call_attention(lib, c, q, slots, req, scale, sink=None, mass=None, lse=True, out_ld=0, longest=None, max_q=0, out=None, **opts):
    T, H, _ = q.shape
    o = torch.full((T + 1, out_ld or H * c.V), 3.0, dtype=q.dtype, device=DEV) if out is None else out
    z = torch.full((T, H), 5.0, device=DEV) if lse else None
    op = ffi.Kv8Options(max_kv_len=longest, max_q_len=max_q, out_ld=out_ld, lse=ptr(z), mass=ptr(mass), mass_ld=mass.shape[2] if mass is not None else 0, **opts)
    f32 = int(q.dtype == F32)
    need = lib.pk_kv8_attention_workspace_bytes(T, H, c.G, c.D, c.V, C.byref(op), f32)
    ws = torch.full((max(16, need) + 64,), 0xff, dtype=torch.uint8, device=DEV)  # (NaN as floats)
    rc = lib.pk_kv8_attention(q.data_ptr(), c.data.data_ptr(), ptr(sink), slots.data_ptr(), req.data_ptr(), c.page_off.data_ptr(), c.pages.data_ptr(), o.data_ptr(),
                              c.stride, c.page, T, H, c.G, c.D, c.V, scale, C.byref(op), ws.data_ptr(), need, f32, stream())
    assert rc == 0
    assert (ws[max(need, 0):] == 0xff).all()
    if out is None:
        assert (o[T] == 3.0).all() and (o[:, H * c.V:] == 3.0).all()
        o = o[:T, :H * c.V].reshape(T, H, c.V)
    return o, z


def filled(lens, G, D, V, page, seed=0, room=None, **kw):
    """a cache whose requests hold lens[r] tokens of random keys and values, through the append's plain form"""
    c = K.Cache(room or lens, G, D, V, page, seed=seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    for r, n in enumerate(lens):
        if n:
            k = torch.randn(n, G, D, generator=g) * torch.exp(0.5 * torch.randn(1, G, D, generator=g))
            v = torch.randn(n, G, V, generator=g) * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g))
            K.fill(c, r, k.to(BF16).double(), v.to(BF16).double())
    c.data, c.page_off, c.pages = c.data.to(DEV), c.page_off.to(DEV), c.pages.to(DEV)
    return c


# ------------------------------------------------------------------ append
def check_append(lib, steps, G, D, V, page, H, dims, interleaved=False, f32=False, bias=False, shift=0, seed=0, ld_more=0, scale_by=1.0):
    """steps: calls, each a list of (request, tokens); a request's tokens follow those of the calls before.  shift: positions run ahead of slots (as after an eviction)"""
    R = 1 + max(r for call in steps for r, _ in call)
    room = [sum(n for call in steps for q, n in call if q == r) for r in range(R)]
    c = K.Cache(room, G, D, V, page, device=DEV, seed=seed, stride_more=32 if seed % 2 else 0)
    want = K.Cache(room, G, D, V, page, seed=seed, stride_more=32 if seed % 2 else 0)
    g = torch.Generator().manual_seed(seed + 7)
    E = F32 if f32 else BF16
    freq = (1.0 / 10000.0 ** (torch.arange(max(1, dims // 2)) / max(1, dims // 2))).float()
    have = [0] * R
    W = H * D + G * (D + V)
    for call in steps:
        T = sum(n for _, n in call)
        qkv = (torch.randn(T, W + ld_more, generator=g) * torch.exp(torch.randn(T, 1, generator=g)) * scale_by).to(E)
        b = torch.randn(W, generator=g).to(E) if bias else None
        slots = [have[r] + i for r, n in call for i in range(n)]
        req = [r for r, n in call for _ in range(n)]
        pos = torch.tensor([s + shift for s in slots], dtype=I32)
        q = call_append(lib, c, qkv.to(DEV), pos.to(DEV), i32(req), H, dims, interleaved, freq.to(DEV), 1.25 if shift else 1.0, i32(slots) if shift else None,
                        b.to(DEV) if bias else None)
        x = qkv[:, :W].double() + (b.double() if bias else 0.0)
        mag = 1.25 if shift else 1.0
        wq, wk, wv = x[:, :H * D].view(T, H, D), x[:, H * D:H * D + G * D].view(T, G, D), x[:, H * D + G * D:].view(T, G, V)
        wq, wk = K.rotate(wq, pos, freq, dims, interleaved, mag), K.rotate(wk, pos, freq, dims, interleaved, mag)
        if H:
            # one rounding to the element type; the table's sines and cosines, the products and the bias' sum are fp32: five roundings of the two terms
            size = wq.abs() if not dims else torch.sqrt(2 * K.rotate(x[:, :H * D].view(T, H, D) ** 2, pos * 0, freq, dims, interleaved)).abs().amax(-1, keepdim=True) * mag
            bound = (2.0 ** -8 if not f32 else 0) * wq.abs() + 8 * 2.0 ** -24 * (size + wq.abs()) + 1e-38
            assert ((q.cpu().double() - wq).abs() <= bound).all()
        t = 0
        for r, n in call:
            K.append(want, r, have[r], wk[t:t + n], wv[t:t + n])
            have[r] += n
            t += n
    torch.cuda.synchronize()
    got = K.Cache(room, G, D, V, page, seed=seed, stride_more=32 if seed % 2 else 0)
    got.data = c.data.cpu()
    for r in range(R):
        for blk in range(-(-have[r] // 16)):
            a, b = got.record(r, blk), want.record(r, blk)
            if not dims and not bias:
                assert torch.equal(a, b), (r, blk)  # nothing but the rounding to codes happens: the same bytes
            else:
                n = 16 * (D + V)
                assert torch.equal(a[:, n + 2:], b[:, n + 2:])
                assert torch.equal(got.record(r, blk)[:, n + 1], want.record(r, blk)[:, n + 1]) or bias
        (gk, gv), (wk, wv) = got.read(r, -(-have[r] // 16) * 16), want.read(r, -(-have[r] // 16) * 16)
        for x, y in ((gk, wk), (gv, wv)):
            # fp32 noise moves a value over a border between two codes now and then: a whole step there (2^-3 of the value, 2^-9 of the exponent's unit), and few of them
            off = (x - y).abs()
            unit = y.abs().amax((0, 2), keepdim=True) * 2.0 ** -16
            assert (off <= 2.0 ** -3 * y.abs() + unit).all() and (off > 0).double().mean() < 1e-3
    # nothing else was written: bytes behind the records, other pages' bytes
    used = torch.zeros_like(got.data, dtype=torch.bool)
    n = page // 16
    for r in range(R):
        for blk in range(-(-have[r] // 16)):
            pg, sub = got.order[got.off[r] + blk * 16 // page], blk * 16 % page // 16
            used[pg, :G * n * got.rec].view(G, n, got.rec)[:, sub] = True
    fresh = K.Cache(room, G, D, V, page, seed=seed, stride_more=32 if seed % 2 else 0)
    assert torch.equal(got.data[~used], fresh.data[~used])


@pytest.mark.parametrize("steps", [
    [[(0, 1)]], [[(0, 16)]], [[(0, 17), (1, 1), (2, 33)]], [[(0, 40)]] + [[(0, 1)]] * 12, [[(0, 5)], [(0, 30)], [(0, 1)], [(0, 3)]],
    [[(r, 1 + 3 * r) for r in range(20)], [(r, 1) for r in range(20)], [(r, 2) for r in range(19, -1, -1)]], [[(0, 100), (1, 3)], [(1, 61), (0, 7)]]])
@pytest.mark.parametrize("G,D,V,page,H", [(2, 64, 64, 16, 4), (8, 128, 128, 16, 8), (1, 32, 256, 48, 3), (3, 96, 32, 32, 0)])
def test_append_bytes(lib, steps, G, D, V, page, H):
    check_append(lib, steps, G, D, V, page, H, 0)
    check_append(lib, steps, G, D, V, page, H, 0, f32=True, seed=1)


@pytest.mark.parametrize("G,D,V,page,H,dims", [(2, 64, 64, 16, 4, 64), (4, 128, 128, 64, 8, 128), (1, 256, 256, 16, 2, 64), (2, 96, 96, 32, 4, 10), (2, 32, 64, 16, 2, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_append_rotated(lib, G, D, V, page, H, dims, interleaved, f32):
    steps = [[(0, 19), (1, 50)], [(1, 1), (0, 1)], [(0, 14), (1, 2)]]
    check_append(lib, steps, G, D, V, page, H, dims, interleaved, f32)
    check_append(lib, steps, G, D, V, page, H, dims, interleaved, f32, bias=True, shift=100000, seed=1, ld_more=8)
    check_append(lib, steps, G, D, V, page, H, dims, interleaved, f32, seed=2, ld_more=3)  # rows that start anywhere


@pytest.mark.parametrize("scale_by", [1e-36, 1e-20, 1e20, 1e36])
def test_append_far_scales(lib, scale_by):
    check_append(lib, [[(0, 20)], [(0, 5)]], 2, 32, 32, 16, 2, 0, scale_by=scale_by)


def test_append_zeros_and_small_after_large(lib):
    """a record of zeros, one whose values fall below the codes of its exponent, one that begins again (a page used by another request)"""
    c, want = K.Cache([32], 1, 32, 32, 16, device=DEV), K.Cache([32], 1, 32, 32, 16)
    for first, rows in ((0, torch.zeros(3, 64)), (3, torch.full((1, 64), 400.0)), (4, torch.full((4, 64), 1e-3)), (8, torch.full((2, 64), 448.1)), (0, torch.full((2, 64), 0.01))):
        n = rows.shape[0]
        call_append(lib, c, rows.to(BF16).to(DEV), i32([first + i for i in range(n)]), i32([0] * n), 0)
        x = rows.to(BF16).double()
        K.append(want, 0, first, x[:, None, :32], x[:, None, 32:])
        assert torch.equal(c.record(0, 0).cpu(), want.record(0, 0))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_append_of_what_is_not_finite(lib, bad, where):
    """the token's key is NaN in that head, its value's codes are zero, its neighbours are as if it were not there; it stays so when the record goes on"""
    G, D = 2, 64
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(21, 2 * G * D, generator=g).to(BF16)
    rows[5, (0 if where == "k" else G * D) + D + 9] = bad  # head 1
    c, want = K.Cache([21], G, D, D, 16, device=DEV), K.Cache([21], G, D, D, 16)
    for a, b in ((0, 8), (8, 9), (9, 21)):
        call_append(lib, c, rows[a:b].to(DEV).contiguous(), i32(range(a, b)), i32([0] * (b - a)), 0)
        K.append(want, 0, a, rows[a:b, :G * D].double().view(-1, G, D), rows[a:b, G * D:].double().view(-1, G, D))
    for blk in (0, 1):
        assert torch.equal(c.record(0, blk).cpu(), want.record(0, blk))
    k, v = c.read(0, 21)
    assert torch.isnan(k[5, 1]).all() and torch.isfinite(k[torch.arange(21) != 5]).all() and torch.isfinite(k[5, 0]).all() and torch.isfinite(v).all()
    q, slots = torch.randn(21, 4, D, generator=g).to(BF16).to(DEV), i32(range(21))
    out, lse = call_attention(lib, c, q, slots, i32([0] * 21), 0.1, longest=21)
    hit = torch.zeros(21, 4, dtype=torch.bool, device=DEV)
    hit[5:, 2:] = True
    assert torch.equal(torch.isnan(out).all(-1), hit) and torch.equal(torch.isnan(out).any(-1), hit) and torch.equal(torch.isnan(lse), hit)


def test_append_leaves_rows_without_a_slot(lib):
    c = K.Cache([16], 1, 32, 32, 16, device=DEV)
    before = c.data.clone()
    rows = torch.randn(3, 96, device=DEV).to(BF16)
    q = call_append(lib, c, rows, i32([4, 4, 4]), i32([99999, 99999, 99999]), 1, slots=i32([-1, -1, -1]))
    assert torch.equal(c.data, before) and torch.equal(q[:, 0], rows[:, :32])


# ------------------------------------------------------------------ attention
def out_bound(want, size, f32, split=True):
    """bf16: one rounding of the result (2^-8), one of each weight where it goes into the product (f16: 2^-11, taken as 2^-8), fp32 sums and
    exponentials (1e-5 of the weights); fp32: exponentials, sums and scores of about 20 in fp32 (weights and q as two f16: 2^-22)"""
    return (2.0 ** -8 + 2e-5) * size + 2.0 ** -8 * want.abs() + 1e-6 if not f32 else 2e-5 * size + 1e-7


def lse_bound(q, k, scale, f32):
    """scores: D products in fp32 and q as two 8-bit numbers (2^-18 of its largest entry) or one or two f16 (less); the logarithm: a few units of fp32"""
    kk = torch.nan_to_num(k).abs().sum(-1).max() if k.numel() else torch.tensor(0.0)
    qm = q.abs().double().max()
    return float(scale * qm * kk * ((0 if f32 else 2.0 ** -18) + 64 * 2.0 ** -24)) + 2e-6


def check_attention(lib, steps, H, G, D, V=None, page=16, f32=False, sink=False, mass=False, seed=0, out_ld=0, max_q=None, q_scale=1.5, longest=None, **opts):
    """steps: (tokens, already cached) of every request"""
    V = V or D
    lens = [a + b for a, b in steps]
    c = filled(lens, G, D, V, page, seed=seed, stride_more=16 if seed % 2 else 0)
    g = torch.Generator().manual_seed(seed + 5)
    T = sum(a for a, _ in steps)
    E = F32 if f32 else BF16
    q = (q_scale * torch.randn(T, H, D, generator=g)).to(E).to(DEV)
    sk = torch.randn(H, generator=g).to(E).to(DEV) if sink else None
    slots, req = i32([b + j for a, b in steps for j in range(a)]), i32([r for r, (a, _) in enumerate(steps) for _ in range(a)])
    scale = D ** -0.5
    most = longest or max(lens)
    m0 = torch.rand(len(steps), G, most, generator=g).to(DEV) if mass else None
    m = m0.clone() if mass else None
    out, lse = call_attention(lib, c, q, slots, req, scale, sk, m, longest=most, out_ld=out_ld, max_q=max(a for a, _ in steps) if max_q is None else max_q, **opts)
    torch.cuda.synchronize()
    t = 0
    for r, (a, b) in enumerate(steps):
        k, v = c.read(r, a + b)
        want, z, w, size = K.attention(q[t:t + a], k, v, slots[t:t + a], scale, sink=sk, **opts)
        assert ((out[t:t + a].double() - want).abs() <= out_bound(want, size, f32)).all(), (r, a, b, (out[t:t + a].double() - want).abs().max().item())
        e = lse_bound(q[t:t + a], k, scale, f32)
        assert ((lse[t:t + a].double() - z).abs() <= e + 2.0 ** -22 * z.abs()).all(), (r, (lse[t:t + a].double() - z).abs().max().item(), e)
        if mass:
            want = m0[r].double()
            want[:, :a + b] += w.view(a, G, H // G, -1).sum((0, 2))
            # every weight is off by twice the bound of the scores, and a count of a thousand of them by one unit of fp32 each time
            assert ((m[r].double() - want).abs() <= 2 * e * (want - m0[r].double()) + 2.0 ** -23 * (1 + a) * want + 1e-6).all(), (r, (m[r].double() - want).abs().max().item())
        t += a


SIZES = [(8, 2, 64), (32, 8, 128), (3, 3, 32), (14, 2, 128), (16, 1, 96), (6, 3, 256), (40, 2, 64)]
STEPS = [[(1, 0)], [(1, 15)], [(1, 16), (1, 63), (1, 200)], [(1, 2500)], [(3, 0), (5, 17), (4, 300)], [(17, 30), (1, 511), (1, 0), (16, 1)], [(63, 0)], [(1, 9 * i) for i in range(70)],
         [(130, 77), (1, 500), (75, 0)], [(300, 0)]]


@pytest.mark.parametrize("H,G,D", SIZES)
@pytest.mark.parametrize("steps", STEPS, ids=lambda s: "+".join(f"{a}at{b}" for a, b in s[:4]) + f"x{len(s)}")
def test_attention(lib, H, G, D, steps):
    check_attention(lib, steps, H, G, D, mass=True)


@pytest.mark.parametrize("steps", STEPS[2:6] + STEPS[8:9], ids=lambda s: "+".join(f"{a}at{b}" for a, b in s[:4]))
@pytest.mark.parametrize("H,G,D,V,page", [(8, 2, 64, 64, 16), (4, 4, 96, 32, 48), (6, 2, 32, 256, 32), (4, 1, 256, 256, 16)])
def test_attention_f32(lib, steps, H, G, D, V, page):
    check_attention(lib, steps, H, G, D, V, page, f32=True, mass=True, sink=True, seed=1)


@pytest.mark.parametrize("opts", [
    dict(window=1), dict(window=16), dict(window=100, sink=True), dict(softcap=20.0), dict(sink=True), dict(softcap=5.0, window=33, sink=True, out_ld=16 * 128 + 8), dict(page=64),
    dict(page=48, max_q=0), dict(longest=20000), dict(q_scale=20.0), dict(q_scale=1e-3, sink=True)])
@pytest.mark.parametrize("steps", [[(1, 400), (1, 31), (1, 129)], [(6, 130), (1, 64), (9, 0), (20, 250)], [(100, 33), (40, 300)]], ids=["decode", "mixed", "prompts"])
def test_options(lib, steps, opts):
    check_attention(lib, steps, 16, 4, 128, mass=True, **opts)
    o = dict(opts)
    o.update(out_ld=0)
    check_attention(lib, steps, 6, 2, 64, mass=True, seed=1, **o)


@pytest.mark.parametrize("D", [64, 96])
def test_weights_where_the_scores_are_not_kept(lib, D):
    """2 GB of them by what max_kv_len allows"""
    check_attention(lib, [(1, 400), (32, 31), (20, 129)], 32, 8, D, mass=True, longest=300000, window=100)


@pytest.mark.parametrize("f32", [False, True])
def test_weights_of_more_tokens_than_a_launch_looks_at(lib, f32):
    """65536; the portion of one request lies on both sides"""
    check_attention(lib, [(61, 0)] * 1076, 2, 1, 64, f32=f32, mass=True)


@pytest.mark.parametrize("steps", [[(1, 400), (3, 31)], [(100, 33), (40, 300)]], ids=["few", "prompts"])
def test_window_that_hides_nothing(lib, steps):
    """as long as the longest context, one token less than it, the largest number"""
    for window in (433, 432, 2 ** 31 - 1):
        check_attention(lib, steps, 8, 2, 64, mass=True, longest=433, window=window)
        check_attention(lib, steps, 4, 2, 32, f32=True, mass=True, longest=433, window=window, seed=1)


@pytest.mark.parametrize("H,G,D,V", [(4, 2, 128, 64), (3, 3, 32, 256), (14, 2, 64, 96), (70, 1, 64, 32), (130, 2, 32, 32), (6, 2, 256, 160), (5, 1, 96, 96)])
@pytest.mark.parametrize("steps", [[(64, 0)], [(33, 700), (8, 1), (40, 64)], [(9, 5000)], [(100, 13), (1, 0), (1, 90), (63, 65)]], ids=["prompt", "portions", "long", "mixed"])
@pytest.mark.parametrize("f32", [False, True])
def test_tiles(lib, H, G, D, V, steps, f32):
    """fp32 rows, and sizes of keys and values that differ: tiles of rows that cross requests, groups larger than a tile, keys in shares"""
    check_attention(lib, steps, H, G, D, V, f32=f32)
    check_attention(lib, steps, H, G, D, V, page=48, f32=f32, mass=True, sink=True, window=77, softcap=15.0, seed=1, max_q=0, out_ld=H * V + 3)


@pytest.mark.parametrize("V", [32, 64, 192])
def test_values_of_another_width(lib, V):
    check_attention(lib, [(1, 333), (20, 40)], 8, 2, 128, V, mass=True)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [5, 90])
def test_rows_without_a_slot(lib, f32, T):
    """padding: rows that see nothing are zero, whatever their request says, and count nowhere"""
    E = F32 if f32 else BF16
    c = filled([40], 2, 64, 64, 16)
    q = torch.randn(T, 4, 64, device=DEV).to(E)
    slots, req = torch.full((T,), -1, dtype=I32, device=DEV), torch.zeros(T, dtype=I32, device=DEV)
    slots[0] = 39
    req[T // 2:] = 12345678
    sk = torch.randn(4, device=DEV).to(E)
    for sink in (None, sk):
        m = torch.zeros(1, 2, 40, device=DEV)
        out, lse = call_attention(lib, c, q, slots, req, 0.125, sink, m, longest=40, max_q=T if T > 5 else 1)
        assert (out[1:] == 0).all() and (out[0] != 0).any()
        assert (torch.isinf(lse[1:]) & (lse[1:] < 0)).all() if sink is None else torch.allclose(lse[1:], sk.float().expand(T - 1, 4), atol=1e-6)
        assert torch.allclose(m.sum(-1), torch.full((1, 2), 2.0, device=DEV), atol=1e-4) or sink is not None


def test_mass_stops_at_its_row(lib):
    c = filled([100], 2, 64, 64, 16)
    m = torch.zeros(2, 2, 50, device=DEV)
    q = torch.randn(1, 4, 64, device=DEV).to(BF16)
    call_attention(lib, c, q, i32([99]), i32([0]), 0.125, None, m, lse=False, longest=100, max_q=1)
    _, _, w, _ = K.attention(q, *c.read(0, 100), i32([99]), 0.125)
    assert torch.allclose(m[0].double(), w[0].view(2, 2, 100).sum(1)[:, :50], atol=1e-5) and (m[1] == 0).all()


def test_far_into_a_large_pool(lib):
    """pages behind 2^32 bytes"""
    G, D, n = 8, 128, 700
    stride = lib.pk_kv8_page_bytes(16, G, D, D)
    before = (1 << 32) // stride + 3
    c = filled([0], G, D, D, 16, room=[n], pages_before=0)
    big = torch.zeros(before + len(c.order), stride, dtype=torch.uint8, device=DEV)
    c.data = big
    c.order = [p + before for p in c.order]
    c.pages = c.pages + before
    rows = torch.randn(n, 2 * G * D, device=DEV).to(BF16)
    call_append(lib, c, rows, i32(range(n)), i32([0] * n), 0)
    k, v = c.read(0, n)
    assert (k - rows[:, :G * D].double().view(n, G, D)).abs().max() < 0.3 and (big[:before] == 0).all()
    q = torch.randn(1, 16, D, device=DEV).to(BF16)
    out, _ = call_attention(lib, c, q, i32([n - 1]), i32([0]), 0.1, longest=n, max_q=1)
    want, _, _, size = K.attention(q, k, v, i32([n - 1]), 0.1)
    assert ((out.double() - want).abs() <= out_bound(want, size, False)).all()


@pytest.mark.parametrize("T,max_q", [(3, 1), (3, 0), (150, 0)])
def test_captured_and_on_another_stream(lib, T, max_q):
    """a captured call serves later contexts: slots and page tables are read when it runs; two graphs with workspaces of their own side by side"""
    G, H, D = 2, 8, 128
    n = 900
    c = filled([n, n], G, D, D, 16)
    q = torch.randn(T, H, D, device=DEV).to(BF16)
    slots, req = torch.zeros(T, dtype=I32, device=DEV), torch.zeros(T, dtype=I32, device=DEV)
    o = [torch.zeros(T, H, D, dtype=BF16, device=DEV) for _ in range(2)]
    op = ffi.Kv8Options(max_kv_len=n, max_q_len=max_q)
    need = max(16, lib.pk_kv8_attention_workspace_bytes(T, H, G, D, D, C.byref(op), 0))
    ws = [torch.empty(need, dtype=torch.uint8, device=DEV) for _ in range(2)]

    def go(i):
        return lib.pk_kv8_attention(q.data_ptr(), c.data.data_ptr(), None, slots.data_ptr(), req.data_ptr(), c.page_off.data_ptr(), c.pages.data_ptr(), o[i].data_ptr(), c.stride,
                                    c.page, T, H, G, D, D, 0.09, C.byref(op), ws[i].data_ptr(), need, 0, stream())
    assert go(0) == 0
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert go(i) == 0
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for last in (T - 1, 200, n - 1):
        slots.copy_(torch.arange(last - T + 1, last + 1, device=DEV))
        req.fill_(1 if last == 200 else 0)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        want, _, _, size = K.attention(q, *c.read(int(req[0]), n), slots, 0.09)
        for x in o:
            assert ((x.double() - want).abs() <= out_bound(want, size, False)).all()
        assert torch.equal(o[0], o[1])


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [1, 6, 100])
def test_a_row_that_sees_nothing_but_what_is_not_finite(lib, f32, T):
    """no share, warp or piece of the keys may hide a NaN behind its largest score"""
    G, D, n = 2, 64, 2000
    c = filled([n], G, D, D, 16)
    for blk in range(n // 16):  # every key of head 1
        rec = c.record(0, blk)
        rec[1, :16 * D] = 0x7f
    q = torch.randn(T, 4, D, device=DEV).to(F32 if f32 else BF16)
    for window, cap in ((0, 0.0), (1, 0.0), (40, 0.0), (0, 20.0), (1, 20.0)):
        out, lse = call_attention(lib, c, q, i32(range(n - T, n)), i32([0] * T), 0.125, longest=n, max_q=T, window=window, softcap=cap)
        assert torch.isnan(out[:, 2:]).all() and torch.isnan(lse[:, 2:]).all() and torch.isfinite(out[:, :2]).all() and torch.isfinite(lse[:, :2]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [3, 100])
def test_a_query_that_is_not_finite(lib, bad, f32, T):
    """stays in its row and head"""
    G, D, n = 2, 64, 300
    c = filled([n], G, D, D, 16)
    q = torch.randn(T, 4, D, device=DEV).to(F32 if f32 else BF16)
    q[1, 1, 5] = bad
    hit = torch.zeros(T, 4, dtype=torch.bool, device=DEV)
    hit[1, 1] = True
    for cap in (0.0, 20.0):
        if cap and math.isinf(bad):
            continue  # (a capped infinite score is the cap)
        out, lse = call_attention(lib, c, q, i32(range(n - T, n)), i32([0] * T), 0.125, longest=n, max_q=T, softcap=cap)
        assert torch.equal(torch.isnan(out).any(-1), hit) and torch.isfinite(out[~hit]).all() and torch.isnan(out[1, 1]).all()


@pytest.mark.parametrize("D", [64, 128])
def test_one_key_that_is_not_finite(lib, D):
    """whichever column of a block it is in: the rows that see it are NaN, and no others"""
    G, n = 1, 150
    q = torch.randn(n, 2, D, device=DEV).to(BF16)
    for bad in list(range(60, 80)) + [0, 127, 149]:
        c = filled([n], G, D, D, 16)
        rec = c.record(0, bad // 16)
        at = bad % 16
        for ch in range(D // 16):
            rec[0, at // 8 * 8 * D + ch * 128 + at % 8 * 16:][:16] = 0x7f
        out, lse = call_attention(lib, c, q, i32(range(n)), i32([0] * n), 0.125, longest=n, max_q=n)
        hit = (torch.arange(n, device=DEV) >= bad)[:, None].expand(n, 2)
        assert torch.equal(torch.isnan(out).all(-1), hit) and torch.equal(torch.isnan(out).any(-1), hit) and torch.equal(torch.isnan(lse), hit)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [2, 90])
def test_rows_that_start_anywhere(lib, f32, T):
    """queries and results on addresses that only their type aligns"""
    G, H, D, n = 2, 6, 64, 333
    E = F32 if f32 else BF16
    c = filled([n], G, D, D, 16)
    room = torch.randn(T * H * D + 3, device=DEV).to(E)
    q = room[3:].view(T, H, D)
    o = torch.zeros(T * (H * D + 1) + 1, dtype=E, device=DEV)
    slots, req = i32(range(n - T, n)), i32([0] * T)
    call_attention(lib, c, q, slots, req, 0.125, longest=n, max_q=T, out_ld=H * D + 1, out=o[1:])
    want, _, _, size = K.attention(q, *c.read(0, n), slots, 0.125)
    got = o[1:].view(T, H * D + 1)
    assert ((got[:, :H * D].reshape(T, H, D).double() - want).abs() <= out_bound(want, size, f32)).all() and (got[:, H * D] == 0).all()


@pytest.mark.parametrize("steps", [[(1, 40 + 13 * i) for i in range(600)], [(1, 7)] * 513 + [(1, 3000)], [(1 + i % 7, 20 * (i % 9)) for i in range(200)]], ids=["600", "513", "200x4"])
def test_many_requests(lib, steps):
    """more tokens than a launch of the few-row kernel looks at"""
    check_attention(lib, steps, 4, 1, 64, mass=True)


@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (16, 4, 128), (6, 2, 96), (24, 1, 128)])
@pytest.mark.parametrize("steps", [[(70, 5000)], [(64, 2047), (1, 3000), (90, 4100)], [(333, 2500), (100, 0)], [(5, 3000)] * 20], ids=["one", "mixed", "two", "twenty"])
@pytest.mark.parametrize("opts", [dict(), dict(window=1500, softcap=20.0, sink=True), dict(sink=True, longest=9000)], ids=["plain", "window", "sink"])
def test_portions_behind_long_contexts(lib, H, G, D, steps, opts):
    """the keys of a few tiles are dealt out to several CTAs"""
    check_attention(lib, steps, H, G, D, mass=True, max_q=0, **opts)


@pytest.mark.parametrize("big", [1e30, 1e-30])
def test_values_of_very_different_sizes(lib, big):
    """records whose exponents lie far apart, the large ones first, last and in between: the small ones' part of the result is lost only where it is small"""
    G, D, n = 1, 64, 200
    c = K.Cache([n], G, D, D, 16)
    g = torch.Generator().manual_seed(2)
    v = torch.randn(n, G, D, generator=g).double()
    v[64:96] *= big
    K.append(c, 0, 0, torch.randn(n, G, D, generator=g).double(), v)
    c.data, c.page_off, c.pages = c.data.to(DEV), c.page_off.to(DEV), c.pages.to(DEV)
    q = torch.randn(1, 8, D, generator=g).to(BF16).to(DEV)
    for last in (63, 95, 199):
        out, _ = call_attention(lib, c, q, i32([last]), i32([0]), 0.125, longest=n, max_q=1)
        want, _, _, size = K.attention(q, *c.read(0, n), i32([last]), 0.125)
        assert ((out.double() - want).abs() <= out_bound(want, size, False)).all()


# ------------------------------------------------------------------ eviction
def pick(mass, n, budget, first, recent):
    m = [(0, 0.0) if math.isnan(x) else (-1, -min(x, 3.4028234663852886e38)) for x in mass[:n].tolist()]  # smaller is better; NaN is behind every number
    if n <= budget:
        return list(range(n))
    always = [j for j in range(n) if j < first or j >= n - recent]
    others = sorted((j for j in range(n) if not (j < first or j >= n - recent)), key=lambda j: (m[j], j))
    return sorted(always + others[:budget - len(always)])


def check_evict(lib, lens, budget, first, recent, G, D, V, page=16, seed=0, mass=None, poison=False, longest=None):
    R = len(lens)
    need = -(-budget // page)
    c = filled([max(0, n) for n in lens], G, D, V, page, seed=seed, room=[max(1, n) for n in lens], spare=R * need)
    if poison:
        rec = c.record(0, 0)
        rec[0, 3 * 16:4 * 16] = 0x7f  # token 3: piece 0 of its key
        for ch in range(1, D // 16):
            rec[0, ch * 128 + 3 * 16:ch * 128 + 4 * 16] = 0x7f
    longest = longest or max(1, *lens)
    g = torch.Generator().manual_seed(seed + 9)
    if mass is None:
        mass = torch.exp(3 * torch.randn(R, G, longest + 5, generator=g)).float()
    m = mass.to(DEV)
    new_m = torch.full((R, G, budget + 9), 4.0, device=DEV)
    kept = torch.full((R, G, budget), -7, dtype=I32, device=DEV)
    new_lens = torch.full((R,), -7, dtype=I32, device=DEV)
    new_off, new_pages = [r * need for r in range(R)], c.spare
    before = c.data.clone()
    old = [c.read(r, max(0, n)) for r, n in enumerate(lens)]
    no, npg, ln = i32(new_off), i32(new_pages), i32(lens)
    assert lib.pk_kv8_evict(c.data.data_ptr(), c.stride, page, c.page_off.data_ptr(), c.pages.data_ptr(), ln.data_ptr(), m.data_ptr(), m.shape[2], no.data_ptr(), npg.data_ptr(),
                            new_lens.data_ptr(), new_m.data_ptr(), new_m.shape[2], kept.data_ptr(), R, G, D, V, budget, first, recent, longest, stream()) == 0
    torch.cuda.synchronize()
    want = K.Cache([max(1, n) for n in lens], G, D, V, page)
    want.data = before.cpu()
    for r, n in enumerate(lens):
        n = max(0, n)
        b = min(n, budget)
        assert int(new_lens[r]) == b
        K_, V_, bad = torch.zeros(-(-b // 16) * 16, G, D, dtype=F64), torch.zeros(-(-b // 16) * 16, G, V, dtype=F64), torch.zeros(-(-b // 16) * 16, G, dtype=torch.bool)
        for h in range(G):
            w = pick(mass[r, h], n, budget, first, recent)
            assert kept[r, h].tolist() == w + [-1] * (budget - b)
            got = new_m[r, h].cpu()
            assert torch.equal(torch.nan_to_num(got[:b], nan=-1), torch.nan_to_num(mass[r, h, w], nan=-1)) and (got[b:] == 0).all()
            K_[:b, h], V_[:b, h] = old[r][0][w, h].cpu(), old[r][1][w, h].cpu()
        bad = torch.isnan(K_).any(-1)
        K_ = torch.nan_to_num(K_)
        for blk in range(-(-b // 16)):
            s = slice(blk * 16, blk * 16 + 16)
            want.write_record(r, blk, K_[s], V_[s], bad[s], [K.exponent(K_[s, h].abs().max().item()) for h in range(G)],
                              [K.exponent(V_[s, h].abs().max().item()) for h in range(G)], new_off, new_pages)
    assert torch.equal(c.data.cpu(), want.data)  # new records, and every other byte as it was
    return c


@pytest.mark.parametrize("lens,budget,first,recent", [
    ([100], 40, 4, 10), ([5, 16, 17, 33], 16, 0, 0), ([1, 0, 3], 1, 0, 1), ([700, 650, 20], 256, 4, 64), ([64], 64, 10, 20), ([300], 33, 33, 0), ([300], 33, 0, 33),
    ([2000, 1500], 1111, 100, 301), ([-1, 40], 17, 1, 1), ([5000], 2049, 0, 16)])
@pytest.mark.parametrize("G,D,V,page", [(2, 64, 64, 16), (3, 128, 32, 48), (1, 32, 256, 32)])
def test_evict(lib, lens, budget, first, recent, G, D, V, page):
    check_evict(lib, lens, budget, first, recent, G, D, V, page)


@pytest.mark.parametrize("kind", ["zeros", "equal", "two", "special", "negative"])
def test_evict_ties_and_special_masses(lib, kind):
    n, G = 1500, 2
    g = torch.Generator().manual_seed(4)
    m = {"zeros": torch.zeros(1, G, n), "equal": torch.full((1, G, n), 0.3), "two": torch.randint(0, 2, (1, G, n), generator=g).float(),
         "special": torch.rand(1, G, n, generator=g), "negative": torch.randn(1, G, n, generator=g)}[kind]
    if kind == "zeros":
        m[0, 0, ::3] = -0.0
    if kind == "special":
        m[0, 0, 5:900:7] = math.nan
        m[0, 0, 6:900:11] = math.inf
        m[0, 1] = math.nan
        m[0, 0, 1000:1100] = -math.inf
    check_evict(lib, [n], 400, 3, 50, G, 32, 32, mass=m)
    check_evict(lib, [n], 1400, 3, 50, G, 32, 32, mass=m)


def test_evict_keeps_what_is_not_finite(lib):
    check_evict(lib, [50], 30, 8, 5, 2, 64, 64, poison=True)


@pytest.mark.parametrize("n,budget,first,recent", [(33000, 1000, 3, 40), (40001, 40000, 1, 1), (32768, 77, 0, 0)])
def test_evict_from_long_contexts(lib, n, budget, first, recent):
    """around the longest that the keys' registers hold, and behind it"""
    check_evict(lib, [n], budget, first, recent, 1, 32, 32)


def test_evict_of_records_with_far_exponents(lib):
    """tokens whose codes are all zero beside a large neighbour, moved to records of small ones and the other way round"""
    G, D, n = 1, 32, 64
    c = K.Cache([n], G, D, D, 16, spare=4)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(n, G, D, generator=g).double(), torch.randn(n, G, D, generator=g).double()
    for b, (x, y) in enumerate(((1e30, 1e-30), (1e-30, 1e-35), (1.0, 1e30), (1e-12, 3e38))):
        k[b * 16:b * 16 + 5] *= x
        k[b * 16 + 5:b * 16 + 16] *= y if y < 1e31 else 1e-20
        v[b * 16:b * 16 + 9] *= y if y < 1e31 else 1e37
        v[b * 16 + 9:b * 16 + 16] *= x
    v[40:] = 0
    K.fill(c, 0, k, v)
    old_k, old_v = c.read(0, n)
    c.data = c.data.to(DEV)
    for keep in (range(5, 21), range(0, 64, 4), list(range(10, 16)) + list(range(40, 64)), range(16)):
        keep = list(keep)
        m = torch.zeros(1, G, n, device=DEV)
        m[0, 0, keep] = 1.0
        B = len(keep)
        kept, new_lens, new_m = torch.zeros(1, G, B, dtype=I32, device=DEV), torch.zeros(1, dtype=I32, device=DEV), torch.zeros(1, G, B, device=DEV)
        ln, off, pages, no, npg = i32([n]), c.page_off.to(DEV), c.pages.to(DEV), i32([0]), i32(c.spare)
        assert lib.pk_kv8_evict(c.data.data_ptr(), c.stride, 16, off.data_ptr(), pages.data_ptr(), ln.data_ptr(), m.data_ptr(), n, no.data_ptr(), npg.data_ptr(),
                                new_lens.data_ptr(), new_m.data_ptr(), B, kept.data_ptr(), 1, G, D, D, B, 0, 0, n, stream()) == 0
        assert kept[0, 0].tolist() == keep
        want = K.Cache([n], G, D, D, 16, spare=4, fill=0)
        pad = -(-B // 16) * 16 - B
        kk, vv = (torch.cat([x[keep], torch.zeros(pad, G, D, dtype=F64)]) for x in (old_k, old_v))
        for blk in range(-(-B // 16)):
            s = slice(blk * 16, blk * 16 + 16)
            want.write_record(0, blk, kk[s], vv[s], torch.zeros(16, G, dtype=torch.bool), [K.exponent(kk[s].abs().max().item())], [K.exponent(vv[s].abs().max().item())], [0], c.spare)
            assert torch.equal(c.record(0, blk, [0], c.spare).cpu(), want.record(0, blk, [0], c.spare))


def test_evict_longer_than_told(lib):
    """no slot from max_kv_len on is looked at"""
    G, D = 2, 32
    c = filled([100], G, D, D, 16, spare=3)
    m = torch.rand(1, G, 64, device=DEV)
    kept, new_lens, new_m = torch.zeros(1, G, 40, dtype=I32, device=DEV), torch.zeros(1, dtype=I32, device=DEV), torch.zeros(1, G, 40, device=DEV)
    ln, no, npg = i32([100]), i32([0]), i32(c.spare)
    assert lib.pk_kv8_evict(c.data.data_ptr(), c.stride, 16, c.page_off.data_ptr(), c.pages.data_ptr(), ln.data_ptr(), m.data_ptr(), 64, no.data_ptr(), npg.data_ptr(),
                            new_lens.data_ptr(), new_m.data_ptr(), 40, kept.data_ptr(), 1, G, D, D, 40, 1, 5, 64, stream()) == 0
    assert [kept[0, h].tolist() for h in range(G)] == [pick(m[0, h].cpu(), 64, 40, 1, 5) for h in range(G)]


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("f32", [False, True])
def test_a_decoding_loop_with_evictions(lib, f32):
    """prompts, decoded tokens, an eviction whenever a request is full, more tokens: every step's attention and the masses against 64 bits on the same cache"""
    G, H, D, page, R, budget = 2, 8, 64, 16, 3, 40
    E = F32 if f32 else BF16
    g = torch.Generator().manual_seed(11)
    room = 96
    c = K.Cache([room] * R, G, D, D, page, device=DEV, spare=R * room // page)
    other = (i32([r * room // page for r in range(R)]), i32(c.spare))
    names = ([c.off, c.order], [other[0].tolist(), c.spare])
    freq = (1.0 / 10000.0 ** (torch.arange(D // 2) / (D // 2))).float().to(DEV)
    lens, pos = [0] * R, [0] * R
    mass = torch.zeros(R, G, room, device=DEV)
    want_mass = torch.zeros(R, G, room, dtype=F64, device=DEV)
    for step, counts in enumerate([(50, 7, 33), (1, 1, 1), (1, 40, 1), "evict", (1, 1, 1), (20, 1, 3), (1, 1, 1), "evict", (1, 1, 1)]):
        if counts == "evict":
            new_m, kept, new_lens = torch.zeros(R, G, room, device=DEV), torch.zeros(R, G, budget, dtype=I32, device=DEV), torch.zeros(R, dtype=I32, device=DEV)
            ln = i32(lens)
            assert lib.pk_kv8_evict(c.data.data_ptr(), c.stride, page, c.page_off.data_ptr(), c.pages.data_ptr(), ln.data_ptr(), mass.data_ptr(), room, other[0].data_ptr(),
                                    other[1].data_ptr(), new_lens.data_ptr(), new_m.data_ptr(), room, kept.data_ptr(), R, G, D, D, budget, 2, 8, room, stream()) == 0
            moved = torch.zeros_like(want_mass)
            for r in range(R):
                for h in range(G):
                    w = pick(mass[r, h].cpu(), lens[r], budget, 2, 8)
                    assert kept[r, h, :len(w)].tolist() == w
                    moved[r, h, :len(w)] = want_mass[r, h, w]
            lens, want_mass, mass = new_lens.tolist(), moved, new_m
            (c.page_off, c.pages), other = other, (c.page_off, c.pages)
            names = names[::-1]
            c.off, c.order = names[0]
            continue
        T = sum(counts)
        qkv = torch.randn(T, H * D + 2 * G * D, generator=g).to(E).to(DEV)
        slots, req = i32([lens[r] + j for r in range(R) for j in range(counts[r])]), i32([r for r in range(R) for _ in range(counts[r])])
        positions = i32([pos[r] + j for r in range(R) for j in range(counts[r])])
        q = call_append(lib, c, qkv, positions, req, H, D, False, freq, slots=slots).contiguous()
        lens, pos = [a + b for a, b in zip(lens, counts)], [a + b for a, b in zip(pos, counts)]
        out, lse = call_attention(lib, c, q, slots, req, D ** -0.5, None, mass, longest=room, max_q=max(counts))
        t = 0
        for r in range(R):
            k, v = c.read(r, lens[r])
            want, z, w, size = K.attention(q[t:t + counts[r]], k, v, slots[t:t + counts[r]], D ** -0.5)
            assert ((out[t:t + counts[r]].double() - want).abs() <= out_bound(want, size, f32)).all(), (step, r)
            want_mass[r, :, :lens[r]] += w.view(counts[r], G, H // G, -1).sum((0, 2))
            t += counts[r]
        assert torch.allclose(mass.double(), want_mass, rtol=2e-4, atol=1e-5)
