"""The ordinary decode on FP32 caches: rows dominated by one key.

The 1e-5 of the decode's contract where the first key of a row lies 25 to 26 above
thousands of others in log2: their weights, 2^-25.5 each, come to 1e-4 and more of
the row, and their values lie about 1. 64 rows of 16400 tokens, so that a work item
takes thousands of tokens.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import TOL, Batch, from_bits, ordinary


@pytest.mark.gpu
@pytest.mark.parametrize("D,bs,heads", [(64, 16, (16, 8)), (128, 16, (16, 8)), (64, 4, (6, 3)), (128, 8, (4, 4)),
                                        (128, 64, (32, 4))])
def test_f32_rows(gpu, D, bs, heads):
    rng = np.random.default_rng(91)
    b = Batch(rng, [(16384, [16] * 64)], "f32", heads=heads, D=D, bs=bs)  # one set of pages for all rows
    a, top = 8.0, 30.0
    k = rng.uniform(-1, 1, b.k.shape).astype(np.float32)
    k[..., 0] = top - rng.uniform(25.0, 26.0, k.shape[:-1]) / (a * 1.4426950408889634 / np.sqrt(D))
    v = (1 + 0.5 * rng.standard_normal(b.v.shape)).astype(np.float32)
    first = int(b.table[0, 0])
    k[first, :, 0, 0] = top
    v[first, :, 0] = rng.standard_normal((b.H, D))
    b.k, b.v = k.view(np.uint32), v.view(np.uint32)
    b.q = (0.01 * rng.standard_normal(b.q.shape)).astype(np.float32)
    b.q[..., 0] = a
    got = ordinary(b.upload(bound=None))
    k, v, G = from_bits(b.k, "f32"), from_bits(b.v, "f32"), b.Hq // b.H
    for r in range(0, 64, 13):
        tokens = np.arange(int(b.lens[r]))
        page = b.table[r, tokens // bs].astype(np.int64)
        for h in range(b.H):
            s = b.q[r, h * G:(h + 1) * G].astype(np.float64) @ k[page, h, tokens % bs].T / np.sqrt(D)
            w = np.exp(s - s.max(-1, keepdims=True))
            want = w @ v[page, h, tokens % bs] / w.sum(-1, keepdims=True)
            error = np.abs(got[r, h * G:(h + 1) * G] - want).max()
            assert error <= TOL, (r, h, error)
