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
