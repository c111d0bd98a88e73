"""The ordinary decode on small pages: page ids past the pool drop out, and no others.

A tile of 16 tokens holds several pages there; one that is missing between others
takes its own tokens with it, and the pages behind it in the tile stay.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import NONE, TOL, Batch, ordinary


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [1, 2, 4, 8, 16, 3, 64])
@pytest.mark.parametrize("dtype,D,heads", [("bf16", 64, (8, 2)), ("bf16", 128, (8, 1)), ("f16", 128, (12, 1)),
                                           ("f32", 64, (4, 2)), ("f32", 128, (8, 2)), ("bf16", 256, (4, 2)),
                                           ("bf16", 80, (4, 2))])
def test_missing_pages(gpu, dtype, D, heads, bs):
    """Single pages, runs of them, a row's first and last, and all of a row's."""
    rng = np.random.default_rng(95)
    b = Batch(rng, [], dtype, heads=heads, D=D, bs=bs, before=[500, 17, 1, 64, 1300, 5])
    for r, share in ((0, 0.1), (1, 0.3), (3, 0.5), (4, 0.05)):
        n = -(-int(b.lens[r]) // bs)
        gone = rng.random(n) < share
        gone[n // 2] = True
        b.table[r, :n][gone] = rng.choice(np.array([b.pages, b.pages + 9, NONE], np.uint64), int(gone.sum()))
    b.table[0, 0] = NONE
    b.table[4, -(-1300 // bs) - 1] = b.pages
    b.table[5] = NONE
    b.upload(bound=None)
    got, want = ordinary(b), b.expected()
    assert (got[5] == 0).all()
    assert np.abs(got - want).max() <= TOL, np.abs(got - want).max()
