"""The 8-bit K/V cache in plain 64-bit torch: its format, the append, the attention and the eviction, token by token and head by head."""
import math

import torch

BLOCK, LARGEST, LOW, HIGH = 16, 448.0, -110, 120
F64, U8, I8, E4M3 = torch.float64, torch.uint8, torch.int8, torch.float8_e4m3fn


def number(code):
    sign, x, m = -1.0 if code & 128 else 1.0, code >> 3 & 15, code & 7
    if x == 15 and m == 7:
        return math.nan
    return sign * (m / 8 * 2.0 ** -6 if x == 0 else (1 + m / 8) * 2.0 ** (x - 7))


NUMBERS = torch.tensor([number(i) for i in range(256)], dtype=F64)


def exponent(amax):
    """the least e with amax <= 448 * 2^e"""
    if amax == 0:
        return LOW
    m, x = math.frexp(amax)
    return min(max(x - 9 if m <= 0.875 else x - 8, LOW), HIGH)


def encode(values, e):
    """[..] finite values -> codes (fp64 / 2^e is exact; from there to fp32 nothing is lost that a test here uses)"""
    return (values * 2.0 ** -e).float().clamp(-LARGEST, LARGEST).to(E4M3).view(U8)


class Cache:
    """A pool of pages and the tables of some requests; `codes` / `tails` are read back from its bytes."""

    def __init__(self, lens_room, G, D, V, page, device="cpu", seed=0, fill=None, spare=0, stride_more=0, pages_before=0):
        self.G, self.D, self.V, self.page = G, D, V, page
        self.rec = BLOCK * (D + V) + 16
        self.stride = G * (page // BLOCK) * self.rec + stride_more
        need = [max(1, -(-n // page)) for n in lens_room]
        gen = torch.Generator().manual_seed(seed)
        order = torch.randperm(sum(need) + spare, generator=gen) + pages_before
        self.off, at = [], 0
        for n in need:
            self.off.append(at)
            at += n
        self.order = order.tolist()
        total = sum(need) + spare + pages_before
        if fill is None:
            self.data = torch.randint(0, 256, (total, self.stride), dtype=U8, generator=gen).to(device)  # what earlier requests left, NaN codes among it
        else:
            self.data = torch.full((total, self.stride), fill, dtype=U8, device=device)
        self.page_off = torch.tensor(self.off, dtype=torch.int32, device=device)
        self.pages = torch.tensor(self.order[:at], dtype=torch.int32, device=device)
        self.spare = self.order[at:]

    def record(self, r, b, off=None, order=None):
        """bytes of the b-th record of a request, [G, record]"""
        off, order = off or self.off, order or self.order
        page, sub = order[off[r] + b * BLOCK // self.page], b * BLOCK % self.page // BLOCK
        n = self.page // BLOCK
        return self.data[page, :self.G * n * self.rec].view(self.G, n, self.rec)[:, sub]

    def values(self, rec):
        """records [n, G, bytes] -> K [16 n, G, D] and V [16 n, G, V] in 64 bits"""
        n, num = rec.shape[0], NUMBERS.to(rec.device)
        e = rec[..., BLOCK * (self.D + self.V):BLOCK * (self.D + self.V) + 2].contiguous().view(I8).double()
        kc = rec[..., :BLOCK * self.D].reshape(n, self.G, 2, self.D // 16, 8, 16).transpose(3, 4).reshape(n, self.G, BLOCK, self.D)
        vc = rec[..., BLOCK * self.D:BLOCK * (self.D + self.V)].reshape(n, self.G, self.V, BLOCK).transpose(2, 3)
        k, v = num[kc.long()] * torch.exp2(e[..., 0])[..., None, None], num[vc.long()] * torch.exp2(e[..., 1])[..., None, None]
        return k.transpose(1, 2).reshape(n * BLOCK, self.G, self.D), v.transpose(1, 2).reshape(n * BLOCK, self.G, self.V)

    def read(self, r, n, off=None, order=None):
        """K [n, G, D] and V [n, G, V] of a request's first n slots, in 64 bits"""
        off, order = off or self.off, order or self.order
        per, b = self.page // BLOCK, torch.arange(-(-n // BLOCK))
        page = torch.tensor(order, dtype=torch.long)[off[r] + b // per].to(self.data.device)
        rec = self.data[:, :self.G * per * self.rec].view(-1, self.G, per, self.rec)[page, :, (b % per).to(page.device)]
        k, v = self.values(rec)
        return k[:n], v[:n]

    def write_record(self, r, b, k, v, bad, ek, ev, off=None, order=None):
        """k [16, G, D], v [16, G, V] values; bad [16, G]: tokens whose key is NaN; ek, ev [G]"""
        rec = self.record(r, b, off, order)
        for g in range(self.G):
            kc, vc = encode(k[:, g], ek[g]), encode(v[:, g], ev[g])
            kc[bad[:, g]] = 0x7f
            rec[g, :BLOCK * self.D] = kc.reshape(2, 8, self.D // 16, 16).transpose(1, 2).reshape(-1)
            rec[g, BLOCK * self.D:BLOCK * (self.D + self.V)] = vc.T.reshape(-1)
            tail = torch.zeros(16, dtype=torch.int16)
            tail[0], tail[1] = ek[g] & 255, ev[g] & 255
            rec[g, BLOCK * (self.D + self.V):] = tail.to(U8).to(rec.device)

    def tail(self, r, b):
        rec = self.record(r, b)
        return rec[:, BLOCK * (self.D + self.V):BLOCK * (self.D + self.V) + 2].contiguous().view(I8).long().tolist()


def rotate(x, positions, freq, dims, interleaved, mag=1.0):
    """x [T, heads, D] in 64 bits"""
    x = x.clone()
    if not dims:
        return x
    i = torch.arange(dims // 2, device=x.device)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)
    a = positions.double()[:, None] * freq.double()
    c, s = torch.cos(a)[:, None] * mag, torch.sin(a)[:, None] * mag
    p, q = x[..., one], x[..., two]
    y = x.clone()
    y[..., one], y[..., two] = p * c - q * s, p * s + q * c
    return y


def append(cache, r, first, k, v):
    """k [n, G, D] (rotated), v [n, G, V] in 64 bits become slots first .. first + n - 1 of request r"""
    n = k.shape[0]
    for b in range(first // BLOCK, (first + n - 1) // BLOCK + 1):
        lo, hi = max(first, b * BLOCK), min(first + n, b * BLOCK + BLOCK)
        goes_on = lo > b * BLOCK
        ok, ov = cache.values(cache.record(r, b)[None])
        K, V = torch.zeros_like(ok), torch.zeros_like(ov)
        old = lo - b * BLOCK
        K[:old], V[:old] = ok[:old], ov[:old]
        K[old:old + hi - lo], V[old:old + hi - lo] = k[lo - first:hi - first], v[lo - first:hi - first]
        bad_v = ~torch.isfinite(V).all(-1)
        bad = ~torch.isfinite(K).all(-1) | bad_v
        V = torch.where(bad_v[..., None], 0.0, V)
        K = torch.where(bad[..., None], 0.0, K)
        tails, new = cache.tail(r, b), slice(old, old + hi - lo)
        ek, ev = ([exponent(x[new, g].abs().max().item()) for g in range(cache.G)] for x in (K, V))
        if goes_on:
            ek, ev = [max(e, t[0]) for e, t in zip(ek, tails)], [max(e, t[1]) for e, t in zip(ev, tails)]
        cache.write_record(r, b, K, V, bad, ek, ev)


def fill(cache, r, k, v):
    """append of finite tokens to an empty request, all records at once"""
    n, nb, per, G = k.shape[0], -(-k.shape[0] // BLOCK), cache.page // BLOCK, cache.G
    out = []
    for x in (k, v):
        y = torch.zeros(nb * BLOCK, G, x.shape[2], dtype=F64)
        y[:n] = x
        y = y.view(nb, BLOCK, G, -1).transpose(1, 2)
        m, e = torch.frexp(y.abs().amax((2, 3)))
        e = torch.where(m == 0, LOW, torch.where(m <= 0.875, e - 9, e - 8).clamp(LOW, HIGH))
        out.append((encode(y * torch.exp2(-e.double())[..., None, None], 0), e))
    (kc, ek), (vc, ev) = out
    rec = torch.zeros(nb, G, cache.rec, dtype=U8)
    rec[..., :BLOCK * cache.D] = kc.reshape(nb, G, 2, 8, cache.D // 16, 16).transpose(3, 4).reshape(nb, G, -1)
    rec[..., BLOCK * cache.D:BLOCK * (cache.D + cache.V)] = vc.transpose(2, 3).reshape(nb, G, -1)
    rec[..., -16], rec[..., -15] = ek.to(I8).view(U8), ev.to(I8).view(U8)
    b = torch.arange(nb)
    page = torch.tensor(cache.order, dtype=torch.long)[cache.off[r] + b // per]
    cache.data[:, :G * per * cache.rec].view(-1, G, per, cache.rec)[page, :, b % per] = rec


def attention(q, k, v, slots, scale, window=0, softcap=0.0, sink=None):
    """One request.  q [T, H, D], k [n, G, D], v [n, G, V], slots [T], sink [H] -> out, lse, weights [T, H, n], and sum of w |v| (all 64 bits)"""
    T, H, _ = q.shape
    n, G, V = v.shape
    out, lse = torch.zeros(T, H, V, dtype=F64, device=q.device), torch.full((T, H), -math.inf, dtype=F64, device=q.device)
    size, weights = torch.zeros_like(out), torch.zeros(T, H, n, dtype=F64, device=q.device)
    j = torch.arange(n, device=q.device)
    seen = j <= slots[:, None]
    if window:
        seen &= j > slots[:, None] - window
    for h in range(H):
        g = h // (H // G)
        s = q[:, h].double() @ k[:, g].T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s = torch.where(seen, s, -math.inf)
        every = s if sink is None else torch.cat([s, sink[h].double().expand(T, 1)], 1)
        z = torch.logsumexp(every, 1) if every.shape[1] else lse[:, h]
        w = torch.where(seen, torch.exp(s - z[:, None]), 0.0)
        lse[:, h], weights[:, h] = z, w
        vv = torch.nan_to_num(v[:, g])
        out[:, h], size[:, h] = w @ vv, w @ vv.abs()
    return out, lse, weights, size
