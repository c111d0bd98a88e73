"""Rows of zero tokens give zeros in every kernel that a decode batch may run on."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import TOL, Batch, ordinary


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 4, 48, 3])
@pytest.mark.parametrize("dtype,D", [("f16", 64), ("bf16", 128), ("f32", 64), ("f32", 128), ("bf16", 256), ("f32", 256),
                                     ("bf16", 80), ("f16", 96), ("bf16", 40), ("f32", 512)])
def test_empty_rows(gpu, dtype, D, bs):
    """Empty rows alone, before and behind others, under bounds of one chunk and of many, as an ordinary batch and as
    one with a group (which runs as the ordinary decode where it shares nothing)."""
    rng = np.random.default_rng(97)
    for lens in ([0], [0, 0, 0], [0, 5, 0, 700, 0], [5, 0]):
        for bound in (None, 300, 5000):
            if bound is None and max(lens) == 0 or bound and bound < max(lens):
                continue
            for heads in ((9, 3), (4, 4)):
                b = Batch(rng, [(0, [0])], dtype, heads=heads, D=D, bs=bs, before=lens).upload(bound)
                want = b.expected()
                for got in (ordinary(b), b.run()):
                    assert np.abs(got - want).max() <= TOL
                    assert (got[b.lens == 0] == 0).all()
                    b.out.fill(0xff)
