"""QuantizedKVLayout: sizes and refusals (no GPU)."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("blocks,heads,bs,D", [(7, 3, 16, 128), (1, 1, 1, 1), (5, 2, 12, 80)])
def test_sizes(v2, blocks, heads, bs, D):
    layout = v2.QuantizedKVLayout(blocks, heads, bs, D, v2.QuantFormat.Int8)
    assert (layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size()) == (blocks, heads, bs, D)
    assert layout.format() == v2.QuantFormat.Int8
    assert layout.page_bytes() == heads * bs * D and layout.cache_bytes() == blocks * heads * bs * D
    assert layout.scale_bytes() == 4 * blocks * heads
    assert layout.cache_stride() % 256 == 0 and 0 <= layout.cache_stride() - layout.cache_bytes() < 256
    assert layout.total_bytes() == 2 * layout.cache_stride() + 2 * layout.scale_bytes()


def test_half_of_a_16_bit_cache(v2):
    eight = v2.QuantizedKVLayout(1000, 8, 16, 128, v2.QuantFormat.E4M3).total_bytes()
    sixteen = v2.PagedKVLayout(1000, 8, 16, 128, v2.DType.BFloat16).total_bytes()
    assert eight <= sixteen * 0.502


@pytest.mark.parametrize("shape", [(0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)])
def test_empty_shapes(v2, shape):
    with pytest.raises(ValueError):
        v2.QuantizedKVLayout(*shape, v2.QuantFormat.E4M3)


@pytest.mark.parametrize("shape", [(2 ** 62, 4, 1, 1), (2 ** 40, 2 ** 10, 2 ** 10, 2 ** 10), (2 ** 62, 1, 1, 1), (2 ** 61, 1, 1, 1)])
def test_sizes_past_64_bits(v2, shape):
    with pytest.raises(OverflowError):
        v2.QuantizedKVLayout(*shape, v2.QuantFormat.E4M3)
