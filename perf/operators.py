"""Operators over a paged K/V cache held in 8 bits: the append that rotates, quantises and stores, the attention that reads it (decoded tokens and
prompts, optionally adding up every cached token's attention weight) and the eviction that keeps the tokens with the most weight.

A case is a dict of plain values.  ``prepare`` makes what a program has in hand before the call, ``run`` is one pass through one operator,
``exact`` the same from the definition in 64 bits, ``work`` what a pass has to read, write and compute at least.

The cache: 16 consecutive tokens of a kv head are one record, 16 * (dim + vdim) codes (e4m3) and two exponents; a value is its code times two to the
power of its record's exponent, one for K and one for V.
"""
import ctypes as C
import math

import torch

own = False

BF16, F32, F64, I32, I8, U8, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int8, torch.uint8, torch.float8_e4m3fn
BLOCK = 16               # tokens of a record
LARGEST = 448.0          # of e4m3
LOW, HIGH = -110, 120    # exponents of a record


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoded token of eight chat requests: latency
        dict(name="append_decode", op="append", requests=8, cached=1000, spread=300, new=1, heads=32, kv_heads=8, dim=128, vdim=128, dims=128, interleaved=False, page=16, f32=False),
        # a long prompt from its first token
        dict(name="append_prompt", op="append", requests=1, cached=0, spread=0, new=4096, heads=32, kv_heads=8, dim=128, vdim=128, dims=128, interleaved=False, page=64, f32=False),
        # one user, a short context: the smallest call
        dict(name="decode_one", op="attention", requests=1, cached=300, spread=0, new=1, heads=16, kv_heads=8, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=False, page=16, f32=False),
        # a full decoding batch with contexts of different lengths
        dict(name="decode_batch", op="attention", requests=32, cached=4095, spread=1500, new=1, heads=32, kv_heads=8, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=False, page=16, f32=False),
        # one user behind a very long document
        dict(name="decode_long", op="attention", requests=1, cached=131071, spread=0, new=1, heads=32, kv_heads=8, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=False, page=64, f32=False),
        # a layer with a sliding window, a sink and capped scores, heads of 64
        dict(name="decode_window", op="attention", requests=48, cached=2500, spread=1900, new=1, heads=64, kv_heads=8, dim=64, vdim=64, window=1024, softcap=30.0, sink=True, mass=False, page=16, f32=False),
        # the all-float32 build of a small model
        dict(name="decode_f32", op="attention", requests=4, cached=1001, spread=400, new=1, heads=8, kv_heads=2, dim=96, vdim=96, window=0, softcap=0.0, sink=True, mass=False, page=32, f32=True),
        # a decoding batch that keeps account of the weights, for the eviction
        dict(name="decode_mass", op="attention", requests=16, cached=8190, spread=77, new=1, heads=32, kv_heads=8, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=True, page=16, f32=False),
        # a long prompt
        dict(name="prompt", op="attention", requests=1, cached=0, spread=0, new=4096, heads=32, kv_heads=8, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=False, page=16, f32=False),
        # two prompt portions of odd length behind a context, with the weights of their tokens
        dict(name="portion_mass", op="attention", requests=2, cached=5003, spread=3000, new=333, heads=16, kv_heads=4, dim=128, vdim=128, window=0, softcap=0.0, sink=False, mass=True, page=16, f32=False),
        # a few requests that reach a small budget
        dict(name="evict_few", op="evict", requests=4, cached=700, spread=150, budget=256, first=4, recent=64, kv_heads=8, dim=128, vdim=128, page=16),
        # a batch of long contexts cut to a quarter
        dict(name="evict_batch", op="evict", requests=16, cached=16384, spread=1000, budget=4096, first=16, recent=512, kv_heads=8, dim=128, vdim=128, page=16),
    ]


def _log(rng, lo, hi):
    """a whole number between lo and hi, spread over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "attention", "attention", "attention", "evict"])
        kv_heads, group = rng.choice([(8, 4), (8, 2), (4, 4), (2, 4), (8, 8), (4, 7), (1, 16), (2, 1), (3, 5)])
        dim = rng.choice([128, 128, 128, 64, 96, 32, 256])
        vdim = dim if rng.random() < 0.85 else rng.choice([32, 64, 128])
        c = dict(op=op, requests=_log(rng, 1, 64), cached=_log(rng, 1, 20000), spread=0, kv_heads=kv_heads, dim=dim, vdim=vdim, page=rng.choice([16, 16, 32, 48, 64]))
        c["spread"] = rng.randrange(c["cached"])
        if op == "evict":
            c["requests"] = min(c["requests"], 16)
            c["budget"] = max(1, int(c["cached"] * rng.uniform(0.1, 0.9)))
            c["first"] = rng.randrange(c["budget"] // 4 + 1)
            c["recent"] = rng.randrange(c["budget"] // 2 + 1)
        else:
            c.update(heads=kv_heads * group, f32=rng.random() < 0.15)
            if rng.random() < 0.4:  # prompts
                c.update(new=_log(rng, 2, 4096), requests=_log(rng, 1, 8))
                if rng.random() < 0.5:
                    c.update(cached=0, spread=0)
            else:
                c["new"] = 1
        if op == "append":
            c.update(dims=rng.choice([0, dim // 2, dim]), interleaved=rng.random() < 0.3)
        if op == "attention":
            c.update(window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), sink=rng.random() < 0.3, mass=rng.random() < 0.3)
        w, most = work(c), [work(x) for x in listed() if x["op"] == op]
        span = c["requests"] * (c["cached"] + c.get("new", 0)) * kv_heads * max(dim, vdim)  # what the plain form has in 32 bits at once
        scores = c["requests"] * c.get("new", 0) * (c["cached"] + c.get("new", 0)) * c.get("heads", 0)
        f32_cost = 8 if c.get("f32") else 1
        if w["bytes"] <= max(m["bytes"] for m in most) and f32_cost * w["flops"] <= max(m["flops"] for m in most) and span <= 1 << 28 and scores <= 1 << 29:
            return c


def _before(c):
    """tokens that every request has in the cache before the call"""
    return [c["cached"] - i * 61 % (c["spread"] + 1) for i in range(c["requests"])]


def _after(c):
    return [n + c.get("new", 0) for n in _before(c)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    G, D, Dv = c["kv_heads"], c["dim"], c["vdim"]
    rec = BLOCK * (D + Dv) + 2
    if c["op"] == "evict":
        lens, B = _before(c), c["budget"]
        kept = sum(min(n, B) for n in lens)
        return {"bytes": G * (4 * sum(lens) + kept * (D + Dv) + kept // BLOCK * rec + 4 * kept + 4 * kept), "flops": 0}
    es, T, H = 4 if c["f32"] else 2, c["requests"] * c["new"], c["heads"]
    if c["op"] == "append":
        return {"bytes": T * (2 * H * D + G * (D + Dv)) * es + T * G * (D + Dv), "flops": 6 * T * (H + G) * c["dims"]}
    pairs = seen = 0
    for n in _before(c):
        for lo, hi in ((n, n + c["new"]),):
            w = c["window"]
            full = sum(min(p + 1, w) for p in range(lo, hi)) if w else (hi * (hi + 1) - lo * (lo + 1)) // 2
            pairs += full
            seen += min(hi, c["new"] - 1 + w) if w else hi
    return {"bytes": seen * G * (D + Dv) + T * H * (D + Dv) * es + T * H * 4 + (8 * seen * G if c["mass"] else 0), "flops": 2 * pairs * H * (D + Dv)}


# ------------------------------------------------------------------ the cache in plain torch
def _exponent(amax):
    """the least e with amax <= 448 * 2^e, within its limits"""
    m, x = torch.frexp(amax.float())
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, LOW)).clamp(LOW, HIGH)


def _two_to(e):
    return torch.exp2(e.double())


def _codes(values, e):
    """[..., 16, D] values and [...] exponents -> codes"""
    return (values.double() * _two_to(-e)[..., None, None]).float().to(E4M3)


def _pack(k, v, ek, ev):
    """codes [..., 16, D] and [..., 16, Dv] and exponents -> records [..., bytes]"""
    lead, D = k.shape[:-2], k.shape[-1]
    kb = k.view(U8).reshape(*lead, 2, 8, D // 16, 16).transpose(-3, -2).reshape(*lead, BLOCK * D)
    vb = v.view(U8).transpose(-1, -2).reshape(*lead, -1)
    tail = torch.zeros(*lead, 16, dtype=U8, device=k.device)
    tail[..., 0], tail[..., 1] = ek.to(I8).view(U8), ev.to(I8).view(U8)
    return torch.cat([kb, vb, tail], -1)


def _unpack(rec, D, Dv):
    """records -> codes [..., 16, D], codes [..., 16, Dv], exponents"""
    lead = rec.shape[:-1]
    k = rec[..., :BLOCK * D].reshape(*lead, 2, D // 16, 8, 16).transpose(-3, -2).reshape(*lead, BLOCK, D).contiguous().view(E4M3)
    v = rec[..., BLOCK * D:BLOCK * (D + Dv)].reshape(*lead, Dv, BLOCK).transpose(-1, -2).contiguous().view(E4M3)
    e = rec[..., BLOCK * (D + Dv):BLOCK * (D + Dv) + 2].contiguous().view(I8).int()
    return k, v, e[..., 0], e[..., 1]


def _values(codes, e):
    return codes.float() * torch.exp2(e.float())[..., None, None]


def _records(s):
    """the cache as [pages, kv heads, records of a page, bytes]"""
    return s["cache"].view(s["cache"].shape[0], s["G"], s["page"] // BLOCK, s["rec"])


def _tables(c, lens, gen, spare=0):
    """pages of every request in no order: (page_off, pages, number of pages); `spare` more pages of a table of its own behind them"""
    need = [-(-max(1, n) // c["page"]) for n in lens]
    more = c["requests"] * spare
    order = torch.randperm(sum(need) + more, generator=gen, device="cuda").to(I32)
    off, at = [], 0
    for n in need:
        off.append(at)
        at += n
    return torch.tensor(off, dtype=I32, device="cuda"), order[:at].contiguous(), order[at:].contiguous(), sum(need) + more


def _fill(s, lens, gen):
    """keys with some large channels and values whose first token is small, quantised record by record, request by request"""
    D, Dv, G = s["D"], s["Dv"], s["G"]
    cache, off, pages = _records(s), s["off_list"], s["pages"].long()
    chan = torch.exp(0.5 * torch.randn(G, 1, D, generator=gen, device="cuda"))
    for r, n in enumerate(lens):
        if n == 0:
            continue
        nb = -(-n // BLOCK)
        k = (torch.randn(G, nb * BLOCK, D, generator=gen, device="cuda") * chan).to(BF16).float()
        v = torch.randn(G, nb * BLOCK, Dv, generator=gen, device="cuda").to(BF16).float()
        v[:, 0] *= 0.0625
        k[:, n:], v[:, n:] = 0, 0
        k, v = k.view(G, nb, BLOCK, D), v.view(G, nb, BLOCK, Dv)
        ek, ev = _exponent(k.abs().amax((-1, -2))), _exponent(v.abs().amax((-1, -2)))
        rec = _pack(_codes(k, ek), _codes(v, ev), ek, ev).transpose(0, 1)  # [blocks, heads, bytes]
        b = torch.arange(nb, device="cuda")
        cache[pages[off[r] + b // (s["page"] // BLOCK)], :, b % (s["page"] // BLOCK)] = rec


# ------------------------------------------------------------------ what a program has before the call
def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *n: torch.randn(*n, generator=gen, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=I32, device="cuda")  # noqa: E731
    G, D, Dv, R, P = c["kv_heads"], c["dim"], c["vdim"], c["requests"], c["page"]
    rec = BLOCK * (D + Dv) + 16
    lens, after = _before(c), _after(c)
    s = dict(c, G=G, D=D, Dv=Dv, R=R, rec=rec, lens=i32(lens), longest=max(after))
    spare = -(-c["budget"] // P) if c["op"] == "evict" else 0
    s["page_off"], s["pages"], s["new_pages"], total = _tables(c, after, gen, spare)
    s["off_list"] = s["page_off"].tolist()
    s["stride"] = G * (P // BLOCK) * rec
    s["cache"] = torch.zeros(total, s["stride"], dtype=U8, device="cuda")
    _fill(s, lens if c["op"] != "attention" else after, gen)
    if c["op"] == "evict":
        s["new_off"] = i32([r * spare for r in range(R)])
        s["ld"], s["new_ld"] = max(lens), c["budget"] + 128
        # few tokens have most of the weight
        s["mass"] = torch.exp(2.0 * rn(R, G, s["ld"]))
        s["new_mass"] = torch.zeros(R, G, s["new_ld"], device="cuda")
        s["new_lens"] = torch.zeros(R, dtype=I32, device="cuda")
        s["kept"] = torch.zeros(R, G, c["budget"], dtype=I32, device="cuda")
        return s
    H, n, E = c["heads"], c["new"], F32 if c["f32"] else BF16
    T = R * n
    s.update(H=H, T=T, E=E)
    s["req"] = torch.arange(R, device="cuda", dtype=I32).repeat_interleave(n)
    s["slots"] = (s["lens"].view(R, 1) + torch.arange(n, device="cuda", dtype=I32)).view(-1).contiguous()
    if c["op"] == "append":
        s["qkv"] = rn(T, H * D + G * (D + Dv)).to(E)
        s["freq"] = 1.0 / (500000.0 ** (torch.arange(0, max(c["dims"], 2), 2, device="cuda", dtype=F64) / max(c["dims"], 2))).to(F32)
        s["q_out"] = torch.zeros(T, H * D, dtype=E, device="cuda")
        # the blocks that the tokens fall into, of every request
        at = [(r, b) for r in range(R) for b in range(lens[r] // BLOCK, (after[r] - 1) // BLOCK + 1)]
        s["at_req"], s["at_block"] = (torch.tensor(x, device="cuda") for x in zip(*at))
        return s
    s["q"] = (1.2 * rn(T, H, D)).to(E)
    s["sinks"] = rn(H).to(E) if c["sink"] else None
    s["scale"] = D ** -0.5
    s["out"] = torch.zeros(T, H, Dv, dtype=E, device="cuda")
    s["lse"] = torch.zeros(T, H, device="cuda")
    s["totals"] = torch.rand(R, G, s["longest"], generator=gen, device="cuda") if c["mass"] else None
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return {"append": _own_append, "attention": _own_attention, "evict": _own_evict}[s["op"]](s)
    return {"append": _append, "attention": _attention, "evict": _evict}[s["op"]](s)


def _cache_outputs(s, rows=slice(None)):
    """the cache as the numbers that its codes stand for, in units of their records' scales, and the scales' exponents (views: nothing is copied)"""
    rec, n = _records(s), BLOCK * (s["D"] + s["Dv"])
    return rec.view(E4M3)[..., :n], rec.view(I8)[..., n:n + 2]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ok(rc):
    if rc != 0:
        raise RuntimeError("the call returned %d" % rc)


def _lib():
    from pegainfer_b200 import ffi
    return ffi.lib(), torch.cuda.current_stream().cuda_stream


def _own_append(s):
    lib, st = _lib()
    _ok(lib.pk_kv8_append(s["qkv"].data_ptr(), s["qkv"].shape[1], None, s["slots"].data_ptr(), None, s["req"].data_ptr(), s["page_off"].data_ptr(),
                          s["pages"].data_ptr(), s["q_out"].data_ptr(), s["cache"].data_ptr(), s["stride"], s["page"], s["H"], s["G"], s["D"], s["Dv"], s["dims"],
                          int(s["interleaved"]), s["freq"].data_ptr(), 1.0, s["T"], int(s["f32"]), st))
    codes, scales = _cache_outputs(s)
    return {"q": s["q_out"], "codes": codes, "scales": scales}


def _own_attention(s):
    lib, st = _lib()
    if "options" not in s:
        from pegainfer_b200 import ffi
        s["options"] = ffi.Kv8Options(window=s["window"], softcap=s["softcap"], max_kv_len=s["longest"], max_q_len=s["new"], lse=s["lse"].data_ptr(),
                                      mass=_ptr(s["totals"]), mass_ld=s["longest"])
        need = lib.pk_kv8_attention_workspace_bytes(s["T"], s["H"], s["G"], s["D"], s["Dv"], C.byref(s["options"]), int(s["f32"]))
        s["workspace"] = torch.empty(max(16, need), dtype=U8, device="cuda")
    _ok(lib.pk_kv8_attention(s["q"].data_ptr(), s["cache"].data_ptr(), _ptr(s["sinks"]), s["slots"].data_ptr(), s["req"].data_ptr(), s["page_off"].data_ptr(),
                             s["pages"].data_ptr(), s["out"].data_ptr(), s["stride"], s["page"], s["T"], s["H"], s["G"], s["D"], s["Dv"], s["scale"],
                             C.byref(s["options"]), s["workspace"].data_ptr(), s["workspace"].numel(), int(s["f32"]), st))
    return {"out": s["out"], "lse": s["lse"], **({"mass": s["totals"]} if s["mass"] else {})}


def _own_evict(s):
    lib, st = _lib()
    _ok(lib.pk_kv8_evict(s["cache"].data_ptr(), s["stride"], s["page"], s["page_off"].data_ptr(), s["pages"].data_ptr(), s["lens"].data_ptr(), s["mass"].data_ptr(),
                         s["ld"], s["new_off"].data_ptr(), s["new_pages"].data_ptr(), s["new_lens"].data_ptr(), s["new_mass"].data_ptr(), s["new_ld"],
                         s["kept"].data_ptr(), s["R"], s["G"], s["D"], s["Dv"], s["budget"], s["first"], s["recent"], s["longest"], st))
    codes, scales = _cache_outputs(s)
    return {"kept": s["kept"], "lens": s["new_lens"], "mass": s["new_mass"], "codes": codes, "scales": scales}


def _append(s):
    T, H, G, D, Dv, R, n = s["T"], s["H"], s["G"], s["D"], s["Dv"], s["R"], s["new"]
    x = s["qkv"].double()
    q, k, v = x[:, :H * D].view(T, H, D), x[:, H * D:(H + G) * D].view(T, G, D), x[:, (H + G) * D:].view(T, G, Dv)
    if s["dims"]:
        half = s["dims"] // 2
        a = s["slots"].double()[:, None] * s["freq"].double()  # far positions: angles in 64 bits
        cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]

        def turn(y):
            y1, y2 = (y[..., 0:s["dims"]:2], y[..., 1:s["dims"]:2]) if s["interleaved"] else (y[..., :half], y[..., half:s["dims"]])
            z1, z2 = y1 * cos - y2 * sin, y1 * sin + y2 * cos
            z = torch.stack([z1, z2], -1).flatten(-2) if s["interleaved"] else torch.cat([z1, z2], -1)
            return torch.cat([z, y[..., s["dims"]:]], -1)
        q, k = turn(q), turn(k)
    s["q_out"] = q.reshape(T, H * D).to(s["E"])
    # the records that the tokens fall into, as values: what the cache has of them, and the new tokens in their places
    cache, per = _records(s), s["page"] // BLOCK
    r, b = s["at_req"], s["at_block"]
    page, sub = s["pages"][s["page_off"][r] + b // per].long(), b % per
    ck, cv, ek, ev = _unpack(cache[page, :, sub], D, Dv)  # [records, heads, ..]
    first = s["lens"][r]
    slot = b[:, None] * BLOCK + torch.arange(BLOCK, device=x.device)
    old = (slot < first[:, None])[:, None, :, None]
    token = slot - first[:, None]
    new = ((token >= 0) & (token < n))[:, None, :, None]
    row = (r[:, None] * n + token.clamp(0, n - 1)).long()
    fresh_k, fresh_v = (torch.where(new, y[row].transpose(1, 2), 0.0) for y in (k, v))
    goes_on = (b * BLOCK < first)[:, None]
    stored = []
    for codes, e, fresh in ((ck, ek, fresh_k), (cv, ev, fresh_v)):
        need = _exponent(fresh.abs().amax((-1, -2)))
        e_new = torch.where(goes_on, torch.maximum(e, need), need)
        stored.append((_codes(torch.where(old, _values(codes, e).double(), fresh), e_new), e_new))
    (ck, ek), (cv, ev) = stored
    cache[page, :, sub] = _pack(ck, cv, ek, ev)
    codes, scales = _cache_outputs(s)
    return {"q": s["q_out"], "codes": codes, "scales": scales}


def _gather(s, longest):
    """records of all requests: codes [R, G, tokens, D], codes [R, G, tokens, Dv], exponents [R, G, blocks] each"""
    per, nb = s["page"] // BLOCK, -(-longest // BLOCK)
    b = torch.arange(nb, device=s["cache"].device)
    at = s["page_off"].long()[:, None] + b // per
    page = s["pages"][at.clamp(max=s["pages"].numel() - 1)].long()  # a shorter request's rows behind its last are masked
    k, v, ek, ev = _unpack(_records(s)[page, :, b % per].transpose(1, 2), s["D"], s["Dv"])  # [R, G, blocks, 16, ..]
    return k, v, ek, ev


def _attention(s):
    T, H, G, D, Dv, R, n = s["T"], s["H"], s["G"], s["D"], s["Dv"], s["R"], s["new"]
    k, v, ek, ev = _gather(s, s["longest"])
    k, v = _values(k, ek).flatten(2, 3), _values(v, ev).flatten(2, 3)  # [R, G, tokens, ..]
    L = k.shape[2]
    p = s["slots"].view(R, 1, n, 1)
    j = torch.arange(L, device=p.device)
    seen = j <= p
    if s["window"]:
        seen = seen & (j > p - s["window"])
    q = s["q"].float().view(R, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(R, G, H // G * n, D)
    x = torch.matmul(q, k.transpose(-1, -2)).view(R, G, H // G, n, L) * s["scale"]
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    x = x.masked_fill(~seen[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    sink = None
    if s["sinks"] is not None:
        sink = s["sinks"].float().view(1, G, H // G, 1, 1)
        top = torch.maximum(top, sink)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    x = x / total
    out = torch.matmul(x.view(R, G, -1, L), v).view(R, G, H // G, n, Dv).permute(0, 3, 1, 2, 4).reshape(T, H, Dv).to(s["E"])
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(T, H).contiguous()
    if s["totals"] is None:
        return {"out": out, "lse": lse}
    s["totals"] += x.sum((2, 3))[..., :s["longest"]]
    return {"out": out, "lse": lse, "mass": s["totals"]}


def _evict(s):
    R, G, D, Dv, B, L = s["R"], s["G"], s["D"], s["Dv"], s["budget"], s["ld"]
    j = torch.arange(L, device="cuda")
    n = s["lens"].long().view(R, 1, 1)
    rank = torch.where((j < s["first"]) | (j >= n - s["recent"]), math.inf, torch.nan_to_num(s["mass"], nan=-math.inf, posinf=torch.finfo(F32).max, neginf=-math.inf))
    rank = torch.where(j < n, rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :B]
    if best.shape[-1] < B:
        best = torch.cat([best, best.new_full((R, G, B - best.shape[-1]), L)], -1)
    kept = torch.sort(best, dim=-1).values
    have = kept < n
    s["kept"] = torch.where(have, kept, -1).to(I32)
    s["new_lens"] = torch.minimum(s["lens"], torch.full_like(s["lens"], B))
    at = kept.clamp(max=L - 1)
    s["new_mass"] = torch.zeros_like(s["new_mass"])
    s["new_mass"][..., :B] = torch.where(have, s["mass"].gather(-1, at), 0.0)
    nb = -(-B // BLOCK)
    k, v, ek, ev = _gather(s, L)
    at, have = torch.nn.functional.pad(at, (0, nb * BLOCK - B)), torch.nn.functional.pad(have, (0, nb * BLOCK - B))[..., None]

    def moved(codes, e):
        W = codes.shape[-1]
        rows = codes.view(U8).flatten(2, 3).gather(2, at[..., None].expand(-1, -1, -1, W)).view(E4M3).float()
        y = torch.where(have, rows * torch.exp2(e.float()).gather(2, at // BLOCK)[..., None], 0.0).view(R, G, nb, BLOCK, W)
        e_new = _exponent(y.abs().amax((-1, -2)))
        return _codes(y, e_new), e_new
    (ck, nk), (cv, nv) = moved(k, ek), moved(v, ev)
    rec = _pack(ck, cv, nk, nv).transpose(1, 2)  # [R, blocks, G, bytes]
    per = s["page"] // BLOCK
    b = torch.arange(nb, device="cuda")
    page = s["new_pages"][s["new_off"].long()[:, None] + b // per].long()
    sub = (b % per).expand_as(page)
    used = (b * BLOCK).view(1, -1) < s["new_lens"].view(-1, 1)  # records behind a short request's last stay as they were
    cache = _records(s)
    cache[page, :, sub] = torch.where(used[..., None, None], rec, cache[page, :, sub])
    codes, scales = _cache_outputs(s)
    return {"kept": s["kept"], "lens": s["new_lens"], "mass": s["new_mass"], "codes": codes, "scales": scales}


# ------------------------------------------------------------------ the definition in 64 bits
def _number(code):
    """what an e4m3 code stands for"""
    sign, x, m = -1.0 if code & 128 else 1.0, code >> 3 & 15, code & 7
    if x == 15 and m == 7:
        return math.nan
    return sign * (m / 8 * 2.0 ** -6 if x == 0 else (1 + m / 8) * 2.0 ** (x - 7))


def _rows(s, r, n, numbers):
    """K and V of the first n tokens of request r: [n, G, D], [n, G, Dv]"""
    D, Dv, P = s["D"], s["Dv"], s["page"]
    t = torch.arange(n, device="cuda")
    page, rec, i = s["pages"].long()[s["off_list"][r] + t // P], t % P // BLOCK, t % BLOCK
    raw = s["cache"].view(s["cache"].shape[0], s["G"], P // BLOCK, s["rec"])
    g = torch.arange(s["G"], device="cuda")[None, :, None]
    d, dv = torch.arange(D, device="cuda"), torch.arange(Dv, device="cuda")
    i3, page3, rec3 = i[:, None, None], page[:, None, None], rec[:, None, None]
    kc = raw[page3, g, rec3, i3 // 8 * (8 * D) + d // 16 * 128 + i3 % 8 * 16 + d % 16]
    vc = raw[page3, g, rec3, BLOCK * D + dv * 16 + i3]
    e = raw[page3, g, rec3, BLOCK * (D + Dv) + torch.arange(2, device="cuda")].view(I8).double()
    return numbers[kc.long()] * 2.0 ** e[..., :1], numbers[vc.long()] * 2.0 ** e[..., 1:]


def exact(c, seed):
    s = prepare(c, seed)
    numbers = torch.tensor([_number(i) for i in range(256)], dtype=F64, device="cuda")
    if c["op"] == "attention":
        return _exact_attention(s, numbers)
    if c["op"] == "append":
        return _exact_append(s, numbers)
    return _exact_evict(s, numbers)


def _exact_attention(s, numbers):
    n, H, G = s["new"], s["H"], s["G"]
    out, lse = torch.zeros(s["T"], H, s["Dv"], dtype=F64, device="cuda"), torch.zeros(s["T"], H, dtype=F64, device="cuda")
    mass = s["totals"].double() if s["mass"] else None
    for r, before in enumerate(s["lens"].tolist()):
        k, v = _rows(s, r, before + n, numbers)
        p, j = torch.arange(before, before + n, device="cuda")[:, None], torch.arange(before + n, device="cuda")
        hidden = j > p
        if s["window"]:
            hidden |= j <= p - s["window"]
        for h in range(H):
            g = h // (H // G)
            x = s["q"][r * n:r * n + n, h].double() @ k[:, g].T * s["scale"]
            if s["softcap"]:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            x[hidden] = -math.inf
            every = x if s["sinks"] is None else torch.cat([x, s["sinks"][h].double().expand(n, 1)], 1)
            z = torch.logsumexp(every, 1)
            w = torch.exp(x - z[:, None])
            out[r * n:r * n + n, h], lse[r * n:r * n + n, h] = w @ v[:, g], z
            if mass is not None:
                mass[r, g, :before + n] += w.sum(0)
    return {"out": out, "lse": lse, "mass": mass}


def _least(amax):
    """exponents of [...] largest magnitudes, in 64 bits"""
    e = torch.ceil(torch.log2((amax / LARGEST).clamp(min=1e-300)))
    for d in (-1, 1):  # the logarithm may be off at a power of two
        e = torch.where((amax <= LARGEST * 2.0 ** (e + d)) if d < 0 else (amax > LARGEST * 2.0 ** e), e + d, e)
    return e.clamp(LOW, HIGH)


def _nearest(x, numbers):
    """the e4m3 numbers nearest to x (|x| <= 448), ties to the even code"""
    a = x.abs()
    step = 2.0 ** (torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    step = torch.where(a >= 16 * step, 2 * step, torch.where(a < 8 * step, torch.where(step > 2.0 ** -9, step / 2, step), step))
    return torch.sign(x) * torch.round(a / step) * step


def _exact_append(s, numbers):
    T, H, G, D, Dv, n, dims = s["T"], s["H"], s["G"], s["D"], s["Dv"], s["new"], s["dims"]
    x = s["qkv"].double()
    qk, v = x[:, :(H + G) * D].reshape(T, H + G, D).clone(), x[:, (H + G) * D:].reshape(T, G, Dv)
    i = torch.arange(dims // 2, device="cuda")
    one, two = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + dims // 2)
    if dims:
        z = torch.polar(torch.ones(T, dims // 2, dtype=F64, device="cuda"), s["slots"].double()[:, None] * s["freq"].double())
        y = torch.complex(qk[..., one], qk[..., two]) * z[:, None]
        qk[..., one], qk[..., two] = y.real, y.imag
    q, k = qk[:, :H].reshape(T, H * D), qk[:, H:]
    P, G_ = s["page"], s["G"]
    rec = _records(s)
    codes = numbers[rec[..., :BLOCK * (D + Dv)].long()]
    scales = rec.view(I8)[..., BLOCK * (D + Dv):BLOCK * (D + Dv) + 2].clone()
    for r, before in enumerate(s["lens"].tolist()):
        old_k, old_v = _rows(s, r, before, numbers) if before else (x.new_zeros(0, G_, D), x.new_zeros(0, G_, Dv))
        for b in range(before // BLOCK, (before + n - 1) // BLOCK + 1):
            page, sub = int(s["pages"][s["off_list"][r] + b * BLOCK // P]), b * BLOCK % P // BLOCK
            lo, hi = max(b * BLOCK, before), min((b + 1) * BLOCK, before + n)
            for which, old, new, W in ((0, old_k, k, D), (1, old_v, v, Dv)):
                rows = x.new_zeros(BLOCK, G_, W)
                fresh = new[r * n + lo - before:r * n + hi - before]
                rows[lo % BLOCK:lo % BLOCK + hi - lo] = fresh
                rows[:lo - b * BLOCK] = old[b * BLOCK:lo]
                e = _least(fresh.abs().amax((0, 2)))
                if lo > b * BLOCK:
                    e = torch.maximum(e, rec[page, :, sub, BLOCK * (D + Dv) + which].view(I8).double())
                y = _nearest(rows * 2.0 ** -e[:, None], numbers)
                scales[page, :, sub, which] = e.to(I8)
                y = y.permute(1, 0, 2)
                if which == 0:
                    codes[page, :, sub, :BLOCK * D] = y.reshape(G_, 2, 8, D // 16, 16).permute(0, 1, 3, 2, 4).reshape(G_, -1)
                else:
                    codes[page, :, sub, BLOCK * D:] = y.permute(0, 2, 1).reshape(G_, -1)
    return {"q": q, "codes": codes, "scales": None}


def _exact_evict(s, numbers):
    R, G, D, Dv, B, P = s["R"], s["G"], s["D"], s["Dv"], s["budget"], s["page"]
    if R * G * B * (D + Dv) > 1 << 24:
        return None  # too long in this form
    mass = torch.zeros(R, G, s["new_ld"], dtype=F64, device="cuda")
    rec = _records(s)
    codes = numbers[rec[..., :BLOCK * (D + Dv)].long()]
    for r, n in enumerate(s["lens"].tolist()):
        k, v = _rows(s, r, n, numbers)
        for g in range(G):
            m = s["mass"][r, g, :n].tolist()
            always = [j for j in range(n) if j < s["first"] or j >= n - s["recent"]]
            others = sorted((j for j in range(s["first"], n - s["recent"])), key=lambda j: (-m[j], j))
            kept = list(range(n)) if n <= B else sorted(always[:B] + others[:max(0, B - len(always))])
            at = torch.tensor(kept, device="cuda")
            mass[r, g, :len(kept)] = s["mass"][r, g, at].double()
            for b in range(-(-len(kept) // BLOCK)):
                page, sub = int(s["new_pages"][int(s["new_off"][r]) + b * BLOCK // P]), b * BLOCK % P // BLOCK
                for which, rows in ((0, k), (1, v)):
                    y = rows[at[b * BLOCK:(b + 1) * BLOCK], g]
                    e = _least(y.abs().amax())
                    y = torch.nn.functional.pad(_nearest(y * 2.0 ** -e, numbers), (0, 0, 0, BLOCK - y.shape[0]))
                    if which == 0:
                        codes[page, g, sub, :BLOCK * D] = y.reshape(2, 8, D // 16, 16).permute(0, 2, 1, 3).reshape(-1)
                    else:
                        codes[page, g, sub, BLOCK * D:] = y.T.reshape(-1)
    return {"kept": None, "lens": None, "mass": mass, "codes": codes, "scales": None}
