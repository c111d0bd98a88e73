"""kvflux_paged_attention_shared: which table row a group's prefix is read through."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import NONE, Batch


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 8])
@pytest.mark.parametrize("short", [[0], [0, 1], [0, 2, 4], [0, 1, 2, 3], [0, 1, 2, 3, 4]], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_first_rows_shorter_than_the_prefix(gpu, dtype, short, bs):
    """Rows shorter than their group's prefix, the first among them, with pages of their own and none behind their
    tokens: the others' prefix is not read through theirs, and theirs not through the others'."""
    rng = np.random.default_rng(61)
    b = Batch(rng, [(64, [5, 9]), (320, [30, 1, 70, 16, 33])], dtype, bs=bs, before=[40])
    lens = [100, 319, 1, 0, 17]
    spare = [int(p) for p in b.table[0, :2]] + [int(p) for p in b.table[1, 64 // bs:] if p < b.pages]
    for i, r in enumerate(short):
        row = 3 + r
        b.lens[row] = lens[i]
        used = -(-lens[i] // bs)
        b.table[row] = NONE
        b.table[row, :used] = rng.choice(spare, used)
    b.check()


@pytest.mark.gpu
def test_pages_behind_a_short_first_row(gpu):
    """A short first row whose entries behind its tokens are pages of the pool: not the prefix either."""
    rng = np.random.default_rng(62)
    b = Batch(rng, [(640, [30, 50, 70])], heads=(32, 8))
    b.lens[0] = 100
    b.table[0] = rng.permutation(b.pages)[:b.table.shape[1]]
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix,length", [(330, 325), (330, 320), (330, 329), (17, 16), (343, 336)])
@pytest.mark.parametrize("bs", [16, 48])
def test_rows_shorter_than_a_prefix_inside_a_page(gpu, bs, prefix, length):
    """A prefix that ends inside a page, and a row that ends between the last whole step before it and its end: its pages
    are its own from the first on."""
    rng = np.random.default_rng(63)
    for row in (0, 2):
        b = Batch(rng, [(prefix, [20, 40, 60, 80])], bs=bs)
        b.lens[row] = length
        b.table[row, :-(-length // bs)] = rng.choice(b.table[3][b.table[3] < b.pages], -(-length // bs))
        b.check()
