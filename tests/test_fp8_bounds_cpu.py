"""The bound that the 8-bit products' results are held to, without a GPU: what it lets through and what not."""
import math

import pytest
import torch

from tests import fp8_ref as R


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_product_holds_and_a_mistake_does_not(dtype):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(5, 300, generator=g), torch.randn(200, 300, generator=g)
    ops = *R.quant_rows(x), *R.quant_weights(w)
    want, size = R.product(*ops, 5, 200, 300)
    y = want.to(dtype)
    R.hold_product(y, want, size)
    for wrong in (math.nan, math.inf, -math.inf, 2 * want[3, 17].item()):
        z = y.clone()
        z[3, 17] = wrong
        with pytest.raises(AssertionError):
            R.hold_product(z, want, size)
    with pytest.raises(AssertionError):
        R.hold_product(torch.full_like(y, math.nan), want, size)
