"""The bytes that bench.py counts for the 8-bit cache."""
import pytest

import bench


@pytest.mark.parametrize("written,seen,hkv,d,block", [(0, 1, 1, 64, 32), (0, 320000, 4, 128, 32), (64, 0, 4, 128, 32),
                                                      (4096, 4096, 2, 96, 128), (1, 7, 3, 16, 8)])
def test_cache_bytes(written, seen, hkv, d, block):
    """Keys and values: 2 bytes of each new element and 1 of its code, 1 of each code seen, and the scales."""
    scales = 2 * hkv * 4 * (written + seen) / block
    assert bench.cache_bytes(written, seen, hkv, d, block) == round(2 * hkv * d * (3 * written + seen) + scales)
    assert bench.cache_bytes(0, block, 1, 16, block) == 2 * (16 * block + 4)
