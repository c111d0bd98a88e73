"""Numbers that kvflux_paged_attention_shared has to hold: every bit of a query,
queries and keys of any size, rows dominated by one key.

Tolerance: the 1e-5 of the decode attention's contract; what a case can lose is
worked out at the case.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_shared_attention import TOL, Batch, from_bits, to_bits


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [("f16", 64), ("f16", 128), ("f16", 256), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-8, 1024.0, 2.0 ** 20])
def test_queries_of_any_size(gpu, dtype, D, size):
    """Queries of standard deviation `size` and keys of 1 / size (FP16 keys: at most 10000, and of 16 of their least
    steps at 2^-20): scores of the size of every other test's, or smaller ones, so the same error."""
    rng = np.random.default_rng(32)
    keys = min(1 / size, 1e4) if dtype == "f16" else 1 / size
    b = Batch(rng, [(300, [10, 200, 31]), (64, [3, 3])], dtype, D=D, scale=keys)
    b.q *= np.float32(size)
    b.check()


@pytest.mark.parametrize("size", [1e-30, 1e-8, 1e-3, 1.0, 1e3, 1e20])
def test_split_of_a_scaled_column(size):
    """The arithmetic of the split (no GPU needed): the column's largest value taken into [2^14, 2^15), then three FP16
    parts. Their least step is 2^-24, so a value is off by 2^-25 * 2^-14 of the largest at most, or, above 2^-15 of it,
    by nothing: 33 bits hold FP32's 24. Without the factor, values of 0.2 and less keep an error of 2^-25 whatever
    their size, and those past 65504 have no parts."""
    rng = np.random.default_rng(34)
    x = (rng.standard_normal((200, 128)) * size).astype(np.float32) * scale_of(128)
    largest = np.abs(x).max(-1, keepdims=True)
    up = np.ldexp(np.float32(1), np.minimum(15 - np.frexp(largest)[1], 126))
    y = x * up
    assert (np.abs(y).max(-1) >= 2.0 ** 14).all() and (np.abs(y) < 2.0 ** 15).all()
    rest, parts = y.copy(), np.zeros(y.shape)
    for _ in range(3):
        part = rest.astype(np.float16)
        rest = rest - part.astype(np.float32)
        parts += part.astype(np.float64)
    off = np.abs(parts - y.astype(np.float64))
    assert off.max() <= 2.0 ** -25
    assert (off[np.abs(y) >= 0.5] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_rows_dominated_by_one_key(gpu, dtype):
    """The first key 25 to 26 above all others in log2, whose weights, 2^-25.5 of it each, come to 3e-4 of the row and
    whose values lie about 1: they have to reach the numerator as they reach the sum. 128 columns in 64 streams, so a
    wavefront walks 4096 tokens."""
    rng = np.random.default_rng(33)
    D, prefix, rows, H, G = 64, 16384, 16, 8, 8
    b = Batch(rng, [(prefix, [16] * rows)] * 8, dtype, heads=(H * G, H), D=D)
    a, top = 8.0, 30.0
    k = rng.uniform(-1, 1, b.k.shape).astype(np.float32)
    k[..., 0] = top - rng.uniform(25.0, 26.0, b.k.shape[:-1]) / (a * scale_of(D))
    v = (1 + 0.5 * rng.standard_normal(b.v.shape)).astype(np.float32)
    for g in range(8):
        first = int(b.table[g * rows, 0])
        k[first, :, 0, 0] = top
        v[first, :, 0] = rng.standard_normal((H, D))
    b.k, b.v = to_bits(k, dtype), to_bits(v, dtype)
    b.q = (0.01 * rng.standard_normal(b.q.shape)).astype(np.float32)
    b.q[..., 0] = a
    got = b.upload().run()
    k, v = from_bits(b.k, dtype), from_bits(b.v, dtype)
    for r in range(0, len(b.lens), 7):
        h = r % H
        tokens = np.arange(int(b.lens[r]))
        page = b.table[r, tokens // b.bs].astype(np.int64)
        s = b.q[r, h * G:(h + 1) * G].astype(np.float64) @ k[page, h, tokens % b.bs].T / np.sqrt(D)
        w = np.exp(s - s.max(-1, keepdims=True))
        want = w @ v[page, h, tokens % b.bs] / w.sum(-1, keepdims=True)
        error = np.abs(got[r, h * G:(h + 1) * G] - want).max()
        assert error <= TOL, (r, error)
