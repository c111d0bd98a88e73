"""Queries of any size on FP16 caches: the ordinary batch decode.

FP16 parts of a query end at 2^-24 and at 65504, whatever the query's size. With
keys of the inverse size the scores are those of unit data, and so is the 1e-5 of
the exact paths' contract.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import TOL, Batch, ordinary


def batch(size, heads, D, bs, lens=(1, 17, 300, 1500)):
    """Rows without a shared prefix; keys of 1 / size, at most 10000 and in steps of 2^-24."""
    rng = np.random.default_rng(41)
    b = Batch(rng, [], "f16", heads=heads, D=D, bs=bs, before=list(lens), scale=min(1 / size, 1e4))
    b.q *= np.float32(size)
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("heads,D,bs", [((4, 2), 64, 16), ((4, 1), 128, 16), ((8, 1), 128, 16), ((7, 1), 64, 16),
                                        ((12, 1), 128, 16), ((16, 1), 64, 64), ((2, 2), 256, 16), ((8, 1), 256, 16),
                                        ((5, 1), 128, 4), ((8, 4), 80, 16)])
@pytest.mark.parametrize("size", [1e-8, 1e-5, 1e-4, 1e-3, 0.1, 1024.0, 2.0 ** 18])
def test_decode(gpu, size, heads, D, bs):
    """One, two and three sets of columns, pages of whole and of part tiles, and a head size of the VALU kernels."""
    b = batch(size, heads, D, bs).upload(bound=None)
    got, want = ordinary(b), b.expected()
    assert np.abs(got - want).max() <= TOL, np.abs(got - want).max()
