"""The 8-bit products' cases of test_fp8_gpu.py with a comparison that NaN does not pass: NaN codes lie behind the rows' widths and NaN scales behind the last token, so an entry that is read
out of range is NaN in the output."""
import pytest

from tests import fp8_ref as R
from tests import test_fp8_gpu as base

pytestmark = pytest.mark.gpu
lib = base.lib


@pytest.fixture(autouse=True)
def nan_is_not_near(monkeypatch):
    monkeypatch.setattr(base, "near", R.hold_product)


test_gemm = base.test_gemm
test_gemm_of_many_parts_and_tiles = base.test_gemm_of_many_parts_and_tiles
test_gemm_rows_of_any_stride = base.test_gemm_rows_of_any_stride
test_gemm_of_tiles_of_any_width = base.test_gemm_of_tiles_of_any_width
test_products_use_nothing_behind_the_width = base.test_products_use_nothing_behind_the_width
test_gemm_with_scales_of_any_size_and_sign = base.test_gemm_with_scales_of_any_size_and_sign
test_gemm_of_model_sizes = base.test_gemm_of_model_sizes
