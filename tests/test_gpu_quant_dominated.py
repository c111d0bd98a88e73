"""Rows on an 8-bit cache that one key dominates, its value as large as the others'.

A row's first key outweighs each of the others by 2^k, so that what they add at a time (a
tile of 32, or one token) lies just under half a step of a sum that holds the first key's
value in FP32: added to that one by one, all of them would be lost, up to (tokens a sum
runs over) * 2^-k of the value.

Tolerance: the contract of 1e-5 of the largest value. What the decode may leave out of it:
64 additions beside the dominant value of at most 2^-24 each (4e-6), a few merges, and the
weights' own error, 2^-20 of them, which are 1e-3 of the row.
"""
from __future__ import annotations

import numpy as np
import pytest

from quant_util import Cache
from test_gpu_quant_attention import run as decode
from test_gpu_quant_prefill import run as prefill

pytestmark = pytest.mark.gpu


def dominated(fmt, H, D, bs, n, weight, value):
    """A cache of n tokens whose first key's score is 0 beside ln(weight) for the others, V of 1 for
    the first and `value` for the others; a table row, a query for each kv head, the output."""
    pages = -(-n // bs)
    cache = Cache(fmt, pages, H, bs, D)
    held = {"e4m3": {0.0: 0, 1.0: 0x38, 1.5: 0x3c}, "int8": {0.0: 0, 1.0: 2, 1.5: 3}}[fmt]
    cache.scales[0], cache.scales[1] = 1.0, 1.0 if fmt == "e4m3" else 0.5
    cache.bytes[0], cache.bytes[1] = held[0.0], held[value]
    table = np.arange(pages, dtype=np.uint64)[None]
    cache.bytes[0, 0, :, 0], cache.bytes[1, 0, :, 0] = held[1.0], held[1.0]
    cache.upload()
    first = 1.0 if fmt == "e4m3" else 2.0  # the value of a byte of the first key
    q = np.float32(-np.log(weight) * np.sqrt(D) / (D * first))
    small = np.exp(-float(q) * first * D / np.sqrt(D)) * (n - 1)
    return cache, table, q, (1.0 + value * small) / (1.0 + small)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 16), (256, 16), (128, 5)])
@pytest.mark.parametrize("value", [1.0, 1.5])
def test_long_rows(gpu, fmt, D, bs, value):
    """As many streams as workgroups, so that each goes through a whole row."""
    n, rows, H, G = 65536, 256, 2, 4
    cache, table, q, want = dominated(fmt, H, D, bs, n, 0.98 * 2.0 ** -29, value)
    got = decode(cache, np.repeat(table, rows, 0), [n] * rows, np.full((rows, H * G, D), q, np.float32))
    assert np.abs(got - want).max() <= 1e-5 * value


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [100, 272])
@pytest.mark.parametrize("call", ["decode", "prompts"])
def test_other_head_sizes(gpu, fmt, D, call):
    """Head sizes of the generic kernel, a token at a time."""
    n, H, G = 16384, 1, 2
    cache, table, q, want = dominated(fmt, H, D, 16, n, 0.98 * 2.0 ** -24, 1.0)
    if call == "decode":
        got = decode(cache, table, [n], np.full((1, H * G, D), q, np.float32))
    else:
        _, got = prefill(cache, table, [n], [2], np.full((2, H * G, D), q, np.float32))
    assert np.abs(got - want).max() <= 1e-5


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,bs,seqs,m", [(128, 16, 128, 8), (128, 5, 128, 8), (64, 16, 128, 8), (256, 16, 128, 8), (128, 1, 128, 8),
                                         (128, 16, 64, 64), (128, 5, 64, 64), (128, 16, 64, 32), (64, 16, 64, 32)])
@pytest.mark.parametrize("value", [1.0, 1.5])
def test_long_prompts(gpu, fmt, D, bs, seqs, m, value):
    """Chunks behind 32768 tokens, as many as fill the GPU, so that each workgroup goes through all keys, in every
    order of work. At most 144 additions of 2^-24 beside the dominant value here: 8.6e-6."""
    n, H, G = 32768, 4, 4
    cache, table, q, _ = dominated(fmt, H, D, bs, n, 0.98 * 2.0 ** -30, value)
    first = 1.0 if fmt == "e4m3" else 2.0
    _, got = prefill(cache, np.repeat(table, seqs, 0), [n] * seqs, [m] * seqs, np.full((seqs * m, H * G, D), q, np.float32))
    small = np.exp(-float(q) * first * np.sqrt(D)) * (n - m + np.arange(m))
    want = (1.0 + value * small) / (1.0 + small)
    assert np.abs(got.reshape(seqs, m, -1) - want[None, :, None]).max() <= 1e-5 * value
