"""The 8-bit K/V cache's entry points without a GPU: sizes whose products or counters would pass 31 bits are refused before anything is launched."""
import pytest

from tests.test_kv8_cpu import APPEND, EVICT, lib  # noqa: F401


@pytest.mark.parametrize("change", [
    dict(heads=2 ** 25),                                     # heads * dim is 2^31: as an int it would be less than any ld
    dict(heads=2 ** 26 + 2),                                 # and here it would be 128
    dict(heads=65536, ld=65536 * 64 + 2 * 128), dict(kv_heads=65536, ld=2 * 64 + 65536 * 128, page_stride=65536 * (16 * 128 + 16)),
    dict(heads=65535, ld=65535 * 64 + 2 * 128 - 1)])
def test_append_refuses(lib, change):
    assert lib.pk_kv8_append(*{**APPEND, **change}.values()) == -1


@pytest.mark.parametrize("change", [dict(budget=2 ** 31 - 1, new_mass_ld=2 ** 31), dict(budget=2 ** 30 + 1, new_mass_ld=2 ** 31)])
def test_evict_refuses(lib, change):
    assert lib.pk_kv8_evict(*{**EVICT, **change}.values()) == -1
