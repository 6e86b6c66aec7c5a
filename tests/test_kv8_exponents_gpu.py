"""The exponents of appended records (csrc/kv8_append.cu), K's and V's, rotated and with a bias: the least that hold the record's tokens, as in 64 bits wherever fp32
arithmetic can tell."""
import pytest
import torch

from tests import kv8_ref as K
from tests.test_kv8_gpu import BF16, DEV, F32, call_append, i32, lib  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G,D,V,H,dims", [(2, 64, 64, 4, 64), (4, 128, 128, 8, 128), (2, 128, 64, 2, 64), (1, 256, 256, 2, 256), (2, 96, 96, 4, 10), (3, 32, 160, 0, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_exponents(lib, G, D, V, H, dims, interleaved, f32, bias):
    E, W = F32 if f32 else BF16, H * D + G * (D + V)
    g = torch.Generator().manual_seed(D + V)
    calls = [[(0, 40)], [(0, 1), (1, 33)], [(0, 30), (1, 1)], [(1, 1), (0, 1)], [(0, 17), (1, 5)]]
    lens = [sum(n for call in calls for r, n in call if r == q) for q in (0, 1)]
    c = K.Cache(lens, G, D, V, 16, device=DEV)
    freq = (1.0 / 10000.0 ** (torch.arange(dims // 2) / (dims // 2))).float()
    b = torch.randn(W, generator=g).to(E) if bias else None
    have, want = [0, 0], {}  # (request, record) -> exponents [G] of K and of V, and whether fp32 may see them otherwise
    for call in calls:
        T = sum(n for _, n in call)
        qkv = (torch.randn(T, W, generator=g) * torch.exp(1.5 * torch.randn(T, 1, generator=g))).to(E)
        pos, req = torch.tensor([have[r] + i for r, n in call for i in range(n)], dtype=torch.int32), [r for r, n in call for _ in range(n)]
        call_append(lib, c, qkv.to(DEV), pos.to(DEV), i32(req), H, dims, interleaved, freq.to(DEV), bias=b.to(DEV) if bias else None)
        x = qkv.double() + (b.double() if bias else 0.0)
        k, v = K.rotate(x[:, H * D:H * D + G * D].view(T, G, D), pos, freq, dims, interleaved), x[:, H * D + G * D:].view(T, G, V)
        t = 0
        for r, n in call:
            for s in range(n):
                at = (r, (have[r] + s) // 16)
                if (have[r] + s) % 16 == 0:
                    want[at] = [[K.LOW, K.LOW, False, False] for _ in range(G)]
                for h in range(G):
                    w = want[at][h]
                    for i, (y, width) in enumerate(((k[t + s, h], D), (v[t + s, h], V))):
                        most, where = (z.item() for z in y.abs().max(0))
                        w[i] = max(w[i], K.exponent(most))
                        # the sum with the bias, two products and a sum of the rotation, its sine and cosine: 2^-21 of the two entries, at most twice the largest
                        # (entries that are only copied have none of that: next to a border they are on the one side or the other)
                        near = 448 * 2.0 ** round(torch.log2(torch.tensor(most / 448)).item())
                        w[2 + i] = w[2 + i] or ((bias or (i == 0 and where < dims)) and abs(most / near - 1) < 2.0 ** -19)
            have[r] += n
            t += n
        torch.cuda.synchronize()
        for (r, blk), heads in want.items():
            got = c.tail(r, blk)
            for h in range(G):
                for i in (0, 1):
                    e = got[h][i]
                    assert e == heads[h][i] or (heads[h][2 + i] and abs(e - heads[h][i]) == 1), (r, blk, h, i, e, heads[h])
    assert sum(x[2] or x[3] for heads in want.values() for x in heads) < 4  # (hardly ever)
