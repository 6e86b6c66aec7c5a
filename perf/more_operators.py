"""Operators of linear layers in 8 bits: the norm that adds a residual and quantises, the gated activation that quantises, the quantisation of weights, the
product of quantised rows and weights, and the product of a feed-forward's gate and up weights whose activated result is quantised again.

A case is a dict of plain values.  ``prepare`` makes what a program has in hand before the call, ``run`` is one pass through one operator, ``exact`` the same
from the definition in 64 bits, ``work`` what a pass has to read, write and compute at least.

A value is its code (e4m3) times its block's scale (float): 128 consecutive entries of a row of activations, 128 rows x 128 entries of weights.  A row's
scales lie block by block, [blocks][tokens].
"""
import math

import torch

own = False

BF16, F32, F64, U8, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.uint8, torch.float8_e4m3fn
BLOCK = 128
LARGEST = 448.0        # of e4m3
LEAST = 2.0 ** -100    # a block's largest magnitude counts as this at least
EPS = 1e-6
ACTS = ("silu", "relu2", "relu_gate", "gelu_gate", "none")  # "silu", "relu_gate" and "gelu_gate" take a gate and a factor beside it


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decoded token of eight requests before the attention's projections: latency
        dict(name="norm_decode", op="norm", tokens=8, width=2560, x_f32=False, offset=0.0, add=True),
        # a prompt behind an fp32 residual stream
        dict(name="norm_prompt", op="norm", tokens=4096, width=4096, x_f32=True, offset=1.0, add=True),
        # a decoding batch between the two products of a feed-forward
        dict(name="act_decode", op="act", tokens=32, width=9728, kind="silu", strided=False),
        # the same for a prompt
        dict(name="act_prompt", op="act", tokens=4096, width=12288, kind="silu", strided=False),
        # a small projection of an fp32 checkpoint, neither side a multiple of a block
        dict(name="weights_small", op="weights", rows=1000, width=2500, f32=True),
        # gate and up of a feed-forward
        dict(name="weights_large", op="weights", rows=24576, width=4096, f32=False),
        # one user's decoded token: latency
        dict(name="gemm_one", op="gemm", tokens=1, rows=2560, width=4096, y_f32=False),
        # a decoding batch through a feed-forward's last product
        dict(name="gemm_batch", op="gemm", tokens=48, rows=4096, width=12288, y_f32=True),
        # a prompt portion of odd length
        dict(name="gemm_portion", op="gemm", tokens=333, rows=6144, width=2560, y_f32=False),
        # a long prompt
        dict(name="gemm_prompt", op="gemm", tokens=4096, rows=24576, width=4096, y_f32=False),
        # a decoding batch through a feed-forward's first product
        dict(name="gated_batch", op="gated", tokens=32, rows=9728, width=2560, kind="silu"),
        # a prompt through it
        dict(name="gated_prompt", op="gated", tokens=2048, rows=12288, width=4096, kind="silu"),
    ]


def _log(rng, lo, hi):
    """a whole number between lo and hi, spread over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """of rows: mostly what models have, now and then odd"""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(lo, n // 64 * 64)


def draw(rng):
    while True:
        op = rng.choice(["norm", "act", "weights", "gemm", "gemm", "gemm", "gated", "gated"])
        tokens = _log(rng, 1, 4096)
        if op == "norm":
            c = dict(op=op, tokens=tokens, width=_width(rng, 64, 8192), x_f32=rng.random() < 0.5, offset=rng.choice([0.0, 1.0]), add=rng.random() < 0.8)
        elif op == "act":
            c = dict(op=op, tokens=tokens, width=_width(rng, 64, 12288), kind=rng.choice(ACTS), strided=rng.random() < 0.3)
        elif op == "weights":
            c = dict(op=op, rows=_width(rng, 64, 24576), width=_width(rng, 64, 12288), f32=rng.random() < 0.3)
        elif op == "gemm":
            c = dict(op=op, tokens=tokens, rows=_width(rng, 16, 24576), width=_width(rng, 64, 12288), y_f32=rng.random() < 0.3)
        else:
            c = dict(op=op, tokens=tokens, rows=_width(rng, 64, 12288), width=_width(rng, 64, 8192), kind=rng.choice(["silu", "relu_gate", "gelu_gate"]))
        w, most = work(c), [work(x) for x in listed() if x["op"] == op]
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return c


def _blocks(n):
    return -(-n // BLOCK)


def _up(n, to):
    return -(-n // to) * to


def _gated(kind):
    return kind in ("silu", "relu_gate", "gelu_gate")


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    T, W = c.get("tokens", 0), c["width"]
    if c["op"] == "norm":
        x = T * W * (4 if c["x_f32"] else 2)
        return {"bytes": x * (2 if c["add"] else 1) + (2 * T * W if c["add"] else 0) + 2 * W + T * (W + 4 * _blocks(W)), "flops": 6 * T * W}
    if c["op"] == "act":
        return {"bytes": T * ((4 if _gated(c["kind"]) else 2) * W + W + 4 * _blocks(W)), "flops": 6 * T * W}
    M = c["rows"]
    if c["op"] == "weights":
        return {"bytes": M * W * ((4 if c["f32"] else 2) + 1) + 4 * _blocks(M) * _blocks(W), "flops": 2 * M * W}
    n = 2 if c["op"] == "gated" else 1
    inputs = n * (M * W + 4 * _blocks(M) * _blocks(W)) + T * (W + 4 * _blocks(W))
    outputs = T * (M + 4 * _blocks(M)) if c["op"] == "gated" else T * M * (4 if c["y_f32"] else 2)
    return {"bytes": inputs + outputs, "flops": 2 * n * T * M * W}


# ------------------------------------------------------------------ the format in plain torch
def _scale(amax):
    return torch.clamp(amax, min=LEAST) / LARGEST


def _quant_rows(v, ld, ld_s):
    """float rows [T, W] -> codes [T, ld], scales [blocks, ld_s]"""
    T, W = v.shape
    nb = _blocks(W)
    b = torch.nn.functional.pad(v, (0, nb * BLOCK - W)).view(T, nb, BLOCK)
    s = _scale(b.abs().amax(-1))
    codes, scales = v.new_zeros(T, ld, dtype=U8), v.new_zeros(nb, ld_s)
    codes[:, :W] = (b / s[..., None]).view(T, -1)[:, :W].to(E4M3).view(U8)
    scales[:, :T] = s.T
    return codes, scales


def _quant_weights(w, ld):
    """[M, W] -> codes [M, ld], scales [blocks of rows, blocks]"""
    M, W = w.shape
    mb, nb = _blocks(M), _blocks(W)
    b = torch.nn.functional.pad(w.float(), (0, nb * BLOCK - W, 0, mb * BLOCK - M)).view(mb, BLOCK, nb, BLOCK)
    s = _scale(b.abs().amax((1, 3)))
    codes = torch.zeros(M, ld, dtype=U8, device=w.device)
    codes[:, :W] = (b / s[:, None, :, None]).reshape(mb * BLOCK, nb * BLOCK)[:M, :W].to(E4M3).view(U8)
    return codes, s


def _rows_values(codes, scales, T, W):
    s = scales[:, :T].T.repeat_interleave(BLOCK, 1)[:, :W]
    return codes[:, :W].view(E4M3).float() * s


def _weights_values(codes, scales, M, W):
    s = scales.repeat_interleave(BLOCK, 0)[:M].repeat_interleave(BLOCK, 1)[:, :W]
    return codes[:, :W].view(E4M3).float() * s


def _act(kind, a, b):
    if kind == "silu":
        return a / (1 + torch.exp(-a)) * b
    if kind == "relu2":
        return torch.clamp(a, min=0) ** 2
    if kind == "relu_gate":
        return torch.clamp(a, min=0) * b
    if kind == "gelu_gate":
        return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))) * b
    return a


# ------------------------------------------------------------------ what a program has before the call
def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *n: torch.randn(*n, generator=gen, device="cuda")  # noqa: E731
    T, W = c.get("tokens", 0), c["width"]
    s = dict(c, T=T, W=W)

    def out_rows(width):
        s["ld"], s["ld_s"] = _up(width, 16), _up(T, 4)
        s["codes"], s["scales"] = torch.zeros(T, s["ld"], dtype=U8, device="cuda"), torch.zeros(_blocks(width), s["ld_s"], device="cuda")

    # a few channels are much larger than the others, as activations have them
    channels = lambda n: torch.exp(0.7 * rn(n)) * torch.where(torch.rand(n, generator=gen, device="cuda") < 0.005, 30.0, 1.0)  # noqa: E731
    if c["op"] == "norm":
        chan = channels(W)
        s["x"] = (rn(T, W) * chan).to(F32 if c["x_f32"] else BF16)
        s["y"] = (0.3 * rn(T, W) * chan).to(BF16) if c["add"] else None
        s["w"] = (1 - c["offset"] + 0.2 * rn(W)).to(BF16)
        out_rows(W)
        return s
    if c["op"] == "act":
        n = (2 if _gated(c["kind"]) else 1) * W
        s["ld_in"] = n + (24 if c["strided"] else 0)
        s["in"] = (1.5 * rn(T, s["ld_in"])).to(BF16)
        out_rows(W)
        return s
    M = c["rows"]
    if c["op"] == "weights":
        s["w"] = (0.02 * rn(M, W) * channels(W)).to(F32 if c["f32"] else BF16)
        s["ld"] = _up(W, 16)
        s["codes"], s["scales"] = torch.zeros(M, s["ld"], dtype=U8, device="cuda"), torch.zeros(_blocks(M), _blocks(W), device="cuda")
        return s
    # weights as a checkpoint has them, rows as the norm or the activation leaves them
    s["ld_w"], s["ld_x"], s["ld_xs"] = _up(W, 16), _up(W, 16), _up(T, 4)
    for name in ("w", "w2") if c["op"] == "gated" else ("w",):
        s[name], s[name + "_scales"] = _quant_weights(rn(M, W).mul_(1 / math.sqrt(W)), s["ld_w"])
    s["xc"], s["x_scales"] = _quant_rows(rn(T, W) * channels(W), s["ld_x"], s["ld_xs"])
    if c["op"] == "gated":
        out_rows(M)
    else:
        s["out"] = torch.zeros(T, M, dtype=F32 if c["y_f32"] else BF16, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return {"norm": _own_norm, "act": _own_act, "weights": _own_weights, "gemm": _own_gemm, "gated": _own_gated}[s["op"]](s)
    return {"norm": _norm, "act": _activate, "weights": _weights, "gemm": _gemm, "gated": _gated_product}[s["op"]](s)


def _ok(rc):
    if rc != 0:
        raise RuntimeError("the call returned %d" % rc)


def _lib():
    from pegainfer_b200 import ffi
    return ffi.lib(), torch.cuda.current_stream().cuda_stream


def _own_norm(s):
    lib, st = _lib()
    y = s["y"].data_ptr() if s["add"] else None
    _ok(lib.pk_fp8_add_norm(y, s["x"].data_ptr(), int(s["x_f32"]), s["w"].data_ptr(), s["offset"], s["codes"].data_ptr(), s["ld"], s["scales"].data_ptr(), s["ld_s"],
                            s["W"], s["T"], EPS, st))
    return {"x": s["x"], "codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _own_act(s):
    lib, st = _lib()
    _ok(lib.pk_fp8_act(s["in"].data_ptr(), s["ld_in"], ACTS.index(s["kind"]), s["codes"].data_ptr(), s["ld"], s["scales"].data_ptr(),
                       s["ld_s"], s["W"], s["T"], st))
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _own_weights(s):
    lib, st = _lib()
    _ok(lib.pk_fp8_weights(s["w"].data_ptr(), int(s["f32"]), s["W"], s["codes"].data_ptr(), s["ld"], s["scales"].data_ptr(), s["rows"], s["W"], st))
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _own_gemm(s):
    lib, st = _lib()
    _ok(lib.pk_fp8_gemm(s["w"].data_ptr(), s["ld_w"], s["w_scales"].data_ptr(), s["xc"].data_ptr(), s["ld_x"], s["x_scales"].data_ptr(), s["ld_xs"],
                        s["out"].data_ptr(), s["rows"], int(s["y_f32"]), s["rows"], s["T"], s["W"], st))
    return {"y": s["out"]}


def _own_gated(s):
    lib, st = _lib()
    _ok(lib.pk_fp8_gemm_gated(s["w"].data_ptr(), s["w_scales"].data_ptr(), s["w2"].data_ptr(), s["w2_scales"].data_ptr(), s["ld_w"], s["xc"].data_ptr(), s["ld_x"],
                              s["x_scales"].data_ptr(), s["ld_xs"], s["codes"].data_ptr(), s["ld"], s["scales"].data_ptr(), s["ld_s"], s["rows"], s["T"], s["W"],
                              ("silu", "relu_gate", "gelu_gate").index(s["kind"]), st))
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _norm(s):
    v = s["x"].float()
    if s["add"]:
        v = v + s["y"].float()
        s["x"].copy_(v)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * (s["offset"] + s["w"].float())
    s["codes"], s["scales"] = _quant_rows(v, s["ld"], s["ld_s"])
    return {"x": s["x"], "codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _activate(s):
    W = s["W"]
    a = s["in"][:, :W].float()
    b = s["in"][:, W:2 * W].float() if _gated(s["kind"]) else None
    s["codes"], s["scales"] = _quant_rows(_act(s["kind"], a, b), s["ld"], s["ld_s"])
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _weights(s):
    s["codes"], s["scales"] = _quant_weights(s["w"], s["ld"])
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


def _product(s, name):
    x = _rows_values(s["xc"], s["x_scales"], s["T"], s["W"])
    return torch.matmul(x, _weights_values(s[name], s[name + "_scales"], s["rows"], s["W"]).T)


def _gemm(s):
    return {"y": _product(s, "w").to(s["out"].dtype)}


def _gated_product(s):
    s["codes"], s["scales"] = _quant_rows(_act(s["kind"], _product(s, "w"), _product(s, "w2")), s["ld"], s["ld_s"])
    return {"codes": s["codes"].view(E4M3), "scales": s["scales"]}


# ------------------------------------------------------------------ the definition in 64 bits
def _numbers():
    """what each of the 256 codes stands for"""
    out = []
    for code in range(256):
        sign, e, m = -1.0 if code & 128 else 1.0, code >> 3 & 15, code & 7
        out.append(math.nan if e == 15 and m == 7 else sign * math.ldexp(m, -9) if e == 0 else sign * math.ldexp(8 + m, e - 10))
    return torch.tensor(out, dtype=F64, device="cuda")


def _nearest(x):
    """the e4m3 numbers nearest to x (|x| <= 448), ties to the even code"""
    a = x.abs()
    e = torch.frexp(a).exponent.clamp(min=-5)  # a < 2^e; below 2^-6 the steps stay 2^-9
    step = torch.ldexp(torch.ones_like(a), e - 4)
    return torch.sign(x) * torch.round(a / step) * step


def _exact_codes(v, ld, ld_s):
    T, W = v.shape
    codes, scales = torch.zeros(T, ld, dtype=F64, device="cuda"), torch.zeros(_blocks(W), ld_s, dtype=F64, device="cuda")
    for b in range(_blocks(W)):
        part = v[:, b * BLOCK:(b + 1) * BLOCK]
        scales[b, :T] = part.abs().max(1).values.clamp(min=LEAST) / 448
        codes[:, b * BLOCK:b * BLOCK + part.shape[1]] = _nearest(part / scales[b, :T, None])
    return {"codes": codes, "scales": scales}


def _exact_product(s, name, numbers):
    T, W, M = s["T"], s["W"], s["rows"]
    y = torch.zeros(T, M, dtype=F64, device="cuda")
    for b in range(_blocks(W)):
        k = slice(b * BLOCK, min(W, (b + 1) * BLOCK))
        x = numbers[s["xc"][:, k].long()] * s["x_scales"][b, :T, None].double()
        w = numbers[s[name][:, k].long()] * s[name + "_scales"][torch.arange(M, device="cuda") // BLOCK, b, None].double()
        y.addmm_(x, w.T)
    return y


def exact(c, seed):
    s = prepare(c, seed)
    numbers = _numbers()
    if c["op"] == "gemm":
        return {"y": _exact_product(s, "w", numbers)}
    if c["op"] == "gated":
        a = _exact_product(s, "w", numbers)
        a = torch.nn.functional.silu(a) if c["kind"] == "silu" else torch.nn.functional.relu(a) if c["kind"] == "relu_gate" else torch.nn.functional.gelu(a, approximate="tanh")
        return _exact_codes(a * _exact_product(s, "w2", numbers), s["ld"], s["ld_s"])
    if c["op"] == "weights":
        w = s["w"].double()
        M, W = w.shape
        codes, scales = torch.zeros(M, s["ld"], dtype=F64, device="cuda"), torch.zeros(_blocks(M), _blocks(W), dtype=F64, device="cuda")
        for i in range(_blocks(M)):
            rows = slice(i * BLOCK, (i + 1) * BLOCK)
            for b in range(_blocks(W)):
                part = w[rows, b * BLOCK:(b + 1) * BLOCK]
                scales[i, b] = part.abs().max().clamp(min=LEAST) / 448
            each = scales[i, torch.arange(W, device="cuda") // BLOCK]
            codes[rows, :W] = _nearest(w[rows] / each)
        return {"codes": codes, "scales": scales}
    if c["op"] == "act":
        W = s["W"]
        a, b = s["in"][:, :W].double(), s["in"][:, W:2 * W].double()
        f = torch.nn.functional
        v = {"silu": lambda: f.silu(a) * b, "relu2": lambda: f.relu(a).square(), "relu_gate": lambda: f.relu(a) * b, "gelu_gate": lambda: f.gelu(a, approximate="tanh") * b,
             "none": lambda: a}[c["kind"]]()
        return _exact_codes(v, s["ld"], s["ld_s"])
    x = s["x"].double()
    if c["add"]:
        x = x + s["y"].double()
    rms = torch.sqrt(x.square().sum(1, keepdim=True) / s["W"] + EPS)
    return {"x": x if c["add"] else s["x"].double(), **_exact_codes((s["offset"] + s["w"].double()) * (x / rms), s["ld"], s["ld_s"])}
