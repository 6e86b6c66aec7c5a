"""The 8-bit K/V cache's attention where a kernel's shortcuts could show: large groups of heads, padding inside a request, records of very different sizes beside one
another, negative scales, queries that are not finite.  Everything against 64 bits (tests/kv8_ref.py), results, lse and weights."""
import math

import pytest
import torch

from tests import kv8_ref as K
from tests.test_kv8_gpu import BF16, DEV, F32, F64, call_attention, filled, i32, lib, lse_bound  # noqa: F401

pytestmark = pytest.mark.gpu


def record_sizes(c, r, n):
    """[n, G]: the largest value that a slot's record can hold"""
    out = []
    for b in range(-(-n // 16)):
        rec = c.record(r, b)
        e = rec[:, 16 * (c.D + c.V) + 1].contiguous().view(torch.int8).double()
        out.append((448.0 * torch.exp2(e))[None].expand(16, -1))
    return torch.cat(out)[:n]


def check(lib, c, q, slots, req, lens, scale, sink=None, mass=True, max_q=None, longest=None, skip=(), **opts):
    """slots, req: lists; lens[r]: slots that request r has.  skip: (row, head) pairs whose results have to be NaN"""
    T, H, _ = q.shape
    f32, most = q.dtype == F32, longest or max(lens)
    g = torch.Generator().manual_seed(T)
    m0 = torch.rand(len(lens), c.G, most, generator=g).to(DEV)
    m = m0.clone() if mass else None
    counts = {r: sum(1 for x in req if x == r) for r in range(len(lens))}
    out, lse = call_attention(lib, c, q, i32(slots), i32(req), scale, sink, m, longest=most, max_q=max(counts.values()) if max_q is None else max_q, **opts)
    torch.cuda.synchronize()
    hit = torch.zeros(T, H, dtype=torch.bool, device=DEV)
    for t, h in skip:
        hit[t, h] = True
    assert torch.equal(torch.isnan(out).any(-1), hit) and torch.equal(torch.isnan(out).all(-1), hit) and torch.equal(torch.isnan(lse), hit)
    sl = torch.tensor(slots, device=DEV)
    for r, n in enumerate(lens):
        at = torch.tensor([t for t in range(T) if req[t] == r], device=DEV, dtype=torch.long)
        if not len(at) or not n:
            continue
        k, v = c.read(r, n)
        qq = torch.nan_to_num(q[at], nan=0.0, posinf=0.0, neginf=0.0)
        want, z, w, size = K.attention(qq, k, v, sl[at], scale, sink=sink, **{x: y for x, y in opts.items() if x != "out_ld"})
        fine = ~hit[at]
        e = lse_bound(qq, k, abs(scale), f32)
        # the result's own rounding; a weight's where it goes into the product (f16: 2^-11, fp32 as two of them) and its exponential's; below f16's normal numbers 2^-25 of a
        # weight that is held at least 2^7 times too large, where the row's largest (weight times a record's largest value) is 1: 2^-32, twice that for a maximum of before
        least = n * 2.0 ** -31 * (w * record_sizes(c, r, n).repeat_interleave(H // c.G, 1).T[None]).amax(-1)
        if f32:
            bound = (2.0 ** -20 + 2 * e) * size + 2.0 ** -23 * want.abs() + least[..., None] + 1e-30
        else:
            bound = (2.0 ** -11 + 2.0 ** -18 + 2 * e) * size + 2.0 ** -8 * want.abs() + least[..., None] + 1e-30
        off = (out[at].double() - want).abs()
        assert (off <= bound)[fine].all(), (r, (off - bound)[fine].max().item(), off[fine].max().item())
        seen = torch.isfinite(z)
        assert torch.equal(torch.isfinite(lse[at])[fine], seen[fine]) and (lse[at][fine & ~seen] == -math.inf).all()
        assert ((lse[at].double() - z).abs() <= e + 2.0 ** -22 * z.abs())[fine & seen].all()
        if mass and not skip:
            total = m0[r].double()
            total[:, :n] += w.view(len(at), c.G, H // c.G, n).sum((0, 2))
            more = total - m0[r].double()
            assert ((m[r].double() - total).abs() <= 2 * (e + 2.0 ** -20) * more + 2.0 ** -23 * (1 + len(at)) * total + 1e-6).all(), (r, (m[r].double() - total).abs().max().item())
    return out, lse


def rows(T, H, D, E, seed=0, size=1.5):
    return (size * torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed))).to(E).to(DEV)


# ------------------------------------------------------------------ large groups
@pytest.mark.parametrize("R", [256, 257, 500, 640, 1000])
def test_groups_of_many_heads(lib, R):
    """more query heads to a kv head than fit a byte: every head has its result"""
    c = filled([41, 7, 300], 1, 32, 32, 16)
    check(lib, c, rows(3, R, 32, BF16), [40, 6, 299], [0, 1, 2], [41, 7, 300], 0.2)
    check(lib, c, rows(5, R, 32, BF16), [38, 39, 40, 6, 299], [0, 0, 0, 1, 2], [41, 7, 300], 0.2, sink=rows(1, R, 1, BF16).view(R), max_q=0)


@pytest.mark.parametrize("D", [64, 96])
def test_weights_of_more_rows_than_a_launch_counts(lib, D):
    """255 tokens of 4096 heads are a launch's; the request lies on both sides"""
    c = filled([300], 1, D, D, 16)
    check(lib, c, rows(300, 4096, D, BF16, size=0.5), list(range(300)), [0] * 300, [300], 0.1)


# ------------------------------------------------------------------ padding
def holes(n, pattern):
    """slots 0 .. n - 1 with rows of no slot in between: (valid, padding) by turns"""
    out, s, i = [], 0, 0
    while s < n:
        a, b = pattern[i % len(pattern)]
        out += list(range(s, min(n, s + a))) + [-1] * b
        s, i = s + a, i + 1
    return out


@pytest.mark.parametrize("H,G,D,V,f32", [(8, 2, 64, 64, False), (4, 1, 128, 128, False), (8, 2, 96, 96, False), (6, 2, 32, 32, False), (6, 2, 192, 192, False), (4, 2, 64, 32, False),
                                         (4, 2, 64, 64, True), (3, 1, 96, 160, True)])
@pytest.mark.parametrize("pattern", [[(1, 1)], [(30, 100), (7, 1)], [(1, 300), (150, 2)]], ids=["each", "some", "many"])
@pytest.mark.parametrize("window", [0, 40])
def test_padding_inside_a_request(lib, H, G, D, V, f32, pattern, window):
    """rows without a slot between the others: every key has the weights of all rows that see it"""
    n = 200
    slots = [-1, -1] + holes(n, pattern) + [-1]
    T = len(slots)
    c = filled([n, 17], G, D, V, 16)
    check(lib, c, rows(T + 1, H, D, F32 if f32 else BF16), slots + [16], [0] * T + [1], [n, 17], D ** -0.5, window=window)


@pytest.mark.parametrize("f32", [False, True])
def test_padding_between_three_tokens(lib, f32):
    c = filled([34], 2, 64, 64, 16)
    check(lib, c, rows(3, 4, 64, F32 if f32 else BF16), [32, -1, 33], [0, 0, 0], [34], 0.125)


@pytest.mark.parametrize("H,G,D,V,f32", [(8, 2, 64, 64, False), (4, 1, 128, 128, False), (8, 2, 96, 96, False), (4, 2, 64, 32, False), (4, 2, 64, 64, True), (3, 1, 96, 160, True)])
@pytest.mark.parametrize("T", [4, 100])
@pytest.mark.parametrize("softcap", [0.0, 15.0])
def test_padding_of_any_contents(lib, H, G, D, V, f32, T, softcap):
    """rows without a slot hold NaN and name requests that there are not: zeros, the sink's lse, no weight"""
    E = F32 if f32 else BF16
    c = filled([130, 60], G, D, V, 16)
    slots = [-1] + list(range(130 - T, 130)) + [-1, 59, -1, -1]
    req = [77] + [0] * T + [0, 1, 1, 99999]
    q = rows(len(slots), H, D, E)
    for t, s in enumerate(slots):
        if s < 0:
            q[t] = math.nan
    sink = rows(1, H, 1, E).view(H)
    out, lse = check(lib, c, q, slots, req, [130, 60], 0.2, sink=sink, softcap=softcap)
    pad = torch.tensor([s < 0 for s in slots], device=DEV)
    assert (out[pad] == 0).all() and torch.allclose(lse[pad], sink.float().expand(int(pad.sum()), H), atol=1e-6)


# ------------------------------------------------------------------ records of different sizes
def sized(lens, G, D, V, factors, seed=0, page=16, push=0.0):
    """factors: (request, first record, last record, factor of the values, push of the keys' first entry)"""
    c = K.Cache(lens, G, D, V, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    for r, n in enumerate(lens):
        k, v = torch.randn(n, G, D, generator=g).to(BF16).double(), torch.randn(n, G, V, generator=g).to(BF16).double()
        for q, a, b, f, x in factors:
            if q == r:
                v[a * 16:b * 16 + 16] *= f
                k[a * 16:b * 16 + 16, :, 0] += x
        K.fill(c, r, k, v)
    c.data, c.page_off, c.pages = c.data.to(DEV), c.page_off.to(DEV), c.pages.to(DEV)
    return c


FORMS = [(8, 2, 64, 64, False), (16, 4, 128, 128, False), (3, 1, 96, 96, False), (6, 2, 32, 32, False), (4, 1, 192, 192, False), (4, 2, 64, 96, False), (8, 2, 64, 64, True), (3, 3, 128, 32, True)]


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("big", [1e12, 1e-12, 1e30])
@pytest.mark.parametrize("which", [0, 1])
def test_large_values_of_another_request(lib, H, G, D, V, f32, big, which):
    """rows of several requests in one tile, one of them with far larger values: the others are as if it were not there"""
    lens = [70, 75, 71, 33]
    c = sized(lens, G, D, V, [(which, 0, 4, big, 0.0)])
    for steps in ((40, 45, 40, 3), (3, 5, 2, 1), (1, 1, 1, 1)):
        slots = [n - s + i for n, s in zip(lens, steps) for i in range(s)]
        req = [r for r, s in enumerate(steps) for _ in range(s)]
        check(lib, c, rows(len(slots), H, D, F32 if f32 else BF16), slots, req, lens, D ** -0.5)


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("big", [1e12, 1e30])
def test_large_values_behind_the_query(lib, H, G, D, V, f32, big):
    """tokens that come later in the same portion: rows before them do not know of them"""
    lens = [200]
    c = sized(lens, G, D, V, [(0, 3, 3, big, 0.0), (0, 9, 9, big ** 1.2, 0.0)])
    check(lib, c, rows(200, H, D, F32 if f32 else BF16), list(range(200)), [0] * 200, lens, D ** -0.5)
    for first, T in ((42, 12), (46, 4), (141, 6)):
        check(lib, c, rows(T, H, D, F32 if f32 else BF16), list(range(first, first + T)), [0] * T, lens, D ** -0.5)


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("big", [1e12, 1e30])
def test_large_values_outside_the_window(lib, H, G, D, V, f32, big):
    lens = [200]
    c = sized(lens, G, D, V, [(0, 1, 1, big, 0.0), (0, 6, 6, big, 0.0)])
    check(lib, c, rows(200, H, D, F32 if f32 else BF16), list(range(200)), [0] * 200, lens, D ** -0.5, window=20)
    for first, T in ((42, 12), (49, 4), (128, 6), (131, 1)):
        check(lib, c, rows(T, H, D, F32 if f32 else BF16), list(range(first, first + T)), [0] * T, lens, D ** -0.5, window=20)


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("n,T", [(200, 200), (200, 12), (200, 1), (3000, 70), (3000, 1)])
@pytest.mark.parametrize("where", ["first", "inside", "next"])
def test_large_values_of_no_weight(lib, H, G, D, V, f32, n, T, where):
    """keys that a row sees and gives next to no weight: 1e12 times e^-60"""
    rec = {"first": 0, "inside": 5, "next": 8}[where]
    c = sized([n], G, D, V, [(0, rec, rec, 1e12, -10.0)])
    q = rows(T, H, D, F32 if f32 else BF16)
    q[..., 0] = 6.0
    check(lib, c, q, list(range(n - T, n)), [0] * T, [n], 1.0 if D == 32 else 0.9, mass=False)


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("T", [1, 6, 150])
def test_values_of_all_sizes(lib, H, G, D, V, f32, T):
    """every record of a size of its own, growing, falling and by turns; several requests"""
    lens = [190, 175, 160, 48]
    f = [(0, b, b, 10.0 ** (b - 6), 0.0) for b in range(12)] + [(1, b, b, 10.0 ** (6 - b), 0.0) for b in range(11)] + [(2, b, b, 1e8 if b & 1 else 1e-8, 0.0) for b in range(10)]
    f += [(3, 1, 1, 0.0, 0.0)]  # a record of zeros
    c = sized(lens, G, D, V, f)
    E = F32 if f32 else BF16
    for window, sink in ((0, None), (37, rows(1, H, 1, E).view(H))):
        each = [min(T, n) for n in lens]
        slots = [n - s + i for n, s in zip(lens, each) for i in range(s)]
        check(lib, c, rows(len(slots), H, D, E), slots, [r for r, s in enumerate(each) for _ in range(s)], lens, D ** -0.5, window=window, sink=sink)


@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
def test_scores_that_rise_all_the_way(lib, H, G, D, V, f32):
    """every block of keys is far above the one before: a reference of before is left behind again and again"""
    n = 1500
    c = K.Cache([n], G, D, V, 16)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(n, G, D, generator=g).to(BF16).double(), torch.randn(n, G, V, generator=g).to(BF16).double()
    k[..., 0] = (torch.arange(n) / 4.0).to(BF16).double()[:, None]
    v[:16] *= 1e15
    K.fill(c, 0, k, v)
    c.data, c.page_off, c.pages = c.data.to(DEV), c.page_off.to(DEV), c.pages.to(DEV)
    for T in (1, 10, 100):
        q = rows(T, H, D, F32 if f32 else BF16)
        for sign in (1.0, -1.0):
            q[..., 0] = 3.0 * sign
            check(lib, c, q, list(range(n - T, n)), [0] * T, [n], 0.25, mass=False)


# ------------------------------------------------------------------ scales
@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("T", [1, 20, 150])
@pytest.mark.parametrize("scale,softcap", [(-0.125, 0.0), (-0.2, 10.0), (0.0, 0.0), (0.0, 5.0)])
def test_scales_of_any_sign(lib, H, G, D, V, f32, T, scale, softcap):
    c = filled([160, 31], G, D, V, 16)
    slots, req = list(range(160 - T, 160)) + [30], [0] * T + [1]
    check(lib, c, rows(T + 1, H, D, F32 if f32 else BF16), slots, req, [160, 31], scale, softcap=softcap)


# ------------------------------------------------------------------ queries that are not finite
@pytest.mark.parametrize("H,G,D,V,f32", FORMS)
@pytest.mark.parametrize("T", [1, 3, 150])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_a_query_that_is_not_finite_whatever_the_cap(lib, H, G, D, V, f32, T, bad, softcap):
    """its row is NaN in that head, in every kernel alike, and no other"""
    n = 300
    c = filled([n], G, D, V, 16)
    q = rows(T, H, D, F32 if f32 else BF16)
    q[T // 2, H - 1, D - 3] = bad
    check(lib, c, q, list(range(n - T, n)), [0] * T, [n], D ** -0.5, softcap=softcap, mass=False, skip=[(T // 2, H - 1)])
