"""kvflux_paged_attention_shared: pages of any size with every type and head size, whole pages and others."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import NONE, Batch

KINDS = [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f16", 64), ("f16", 128), ("f16", 256), ("f32", 64), ("f32", 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [1, 5, 8, 24, 32, 100])
@pytest.mark.parametrize("dtype,D", KINDS)
def test_pages(gpu, dtype, D, bs):
    """Prefixes of whole pages and one that ends inside a page, over several tiles; groups of 2 to 160 columns."""
    rng = np.random.default_rng(81)
    Batch(rng, [(bs * (1 + 500 // bs), [1, 20, 130]), (3 * bs + 2 * bs // 3, [50, 3])], dtype, D=D, bs=bs,
          before=[70]).check()
    Batch(rng, [(bs * (1 + 300 // bs), [5] * 20)], dtype, D=D, bs=bs, heads=(16, 2)).check()


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [8, 16])
@pytest.mark.parametrize("dtype,D", KINDS)
def test_missing_pages(gpu, dtype, D, bs):
    """Page ids past the pool, single ones and whole tiles of them, in the prefix and in a row's own part."""
    rng = np.random.default_rng(82)
    b = Batch(rng, [(640, [40, 300, 20])], dtype, D=D, bs=bs)
    b.table[:, 3] = b.pages
    b.table[:, 128 // bs:480 // bs] = NONE
    b.table[1, 720 // bs:800 // bs] = b.pages + 7
    b.check()
