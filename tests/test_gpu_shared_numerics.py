"""Numbers that kvflux_paged_attention_shared has to hold: every bit of a query.

Tolerance: the 1e-5 of the decode attention's contract; what a case can lose is
worked out at the case.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import Batch, to_bits


def scale_of(D):
    """log2(e) / sqrt(D) as the kernels hold it."""
    return np.float32(1.4426950408889634 / np.sqrt(np.float64(D)))


def queries_past_22_bits(rng, D, e, sign):
    """D queries whose scaled value lies in [2^e, 1.01 * 2^e), is exact within 1/16 of a step, and needs the last of
    FP32's 24 bits: the first two FP16 parts miss it by a whole step, on the side of `sign` (and by 15/16 of one at
    least where the remainder is taken from the product before its rounding)."""
    scale = scale_of(D)
    q = (rng.uniform(2.0 ** e, 1.01 * 2.0 ** e, 1 << 21) / scale).astype(np.float32)
    x = q * scale
    step = 2.0 ** (e - 23)
    off = (q.astype(np.float64) * np.float64(scale) - x) * sign
    exact = (off <= 0) & (off > -step / 16)
    hi = x.astype(np.float16).astype(np.float32)
    mid = (x - hi).astype(np.float16).astype(np.float32)
    found = q[exact & ((x - hi - mid) * sign == np.float32(step))]
    assert len(found) >= D
    return found[:D]


@pytest.mark.gpu
@pytest.mark.parametrize("D,e", [(64, 4), (128, 3), (256, 2)])
def test_f16_every_bit_of_a_query(gpu, D, e):
    """Half the tokens have the key +1, -1, +1, ... and the value 1, the others the key 0 and the value -1, so with
    score s of the first, an output is tanh(s / 2). s is a sum of D values of 2^e with alternating signs, small itself;
    a step of 2^(e - 23) lost from each is D * 2^(e - 23) = 1.2e-4 in log2 and 4.2e-5 in the output. The queries'
    own rounding is at most a sixteenth of that, 2.7e-6, and the score chain's below 12 * 2^-20 in log2, 4e-6."""
    rng = np.random.default_rng(31)
    b = Batch(rng, [(512, [64, 2, 128])], "f16", D=D)
    at = np.arange(b.pages * b.bs).reshape(b.pages, b.bs) % 2 == 0  # whole pages: even tokens of every row
    sign = np.where(np.arange(D) % 2 == 0, 1.0, -1.0).astype(np.float32)
    k = np.where(at[:, None, :, None], sign, np.float32(0))
    v = np.where(at[:, None, :, None], np.float32(1), np.float32(-1))
    b.k = to_bits(np.broadcast_to(k, b.k.shape), "f16")
    b.v = to_bits(np.broadcast_to(v, b.v.shape), "f16")
    for r in range(b.q.shape[0]):
        for h in range(b.Hq):
            for s, first in ((1, 0), (-1, 1)):
                b.q[r, h, first::2] = rng.permutation(queries_past_22_bits(rng, D, e, s))[:D // 2]
    b.check()
