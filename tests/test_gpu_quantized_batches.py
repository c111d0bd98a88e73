"""Calls of the C++ layer on an 8-bit cache that the shape limits of a kernel end, and ones
that they must not end: what fails changes nothing, what fits is done."""
from __future__ import annotations

import numpy as np
import pytest

from kvflux_amd import device
from quant_util import from_bits, to_bits
from test_gpu_quantized_kv import Model, pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,Hq", [(576, 4), (64, 1 << 20)])
def test_a_decode_step_that_attention_refuses_changes_nothing(gpu, v2, D, Hq):
    """A head size that the writes take and the attention does not; more query heads than it takes."""
    pool = v2.PhysicalBlockPool(20, 16)
    storage = v2.QuantizedKVStorage(pool, 2, D, v2.QuantFormat.E4M3)
    seqs = [v2.SequenceState(i, pool) for i in range(2)]
    counts = [20, 5]
    for s, n in zip(seqs, counts):
        s.append_tokens(n)
    rng = np.random.default_rng(D)
    kv = device.to_device(to_bits(rng.standard_normal((25, 2, 2 * D)), "bf16"))
    v2.write_quantized_kv(storage, seqs, counts, v2.NewRows(kv.ptr, kv.ptr + 4 * D, v2.DType.BFloat16, 4 * D, 4 * D))
    kv = device.to_device(to_bits(100 * rng.standard_normal((2, 2, 2 * D)), "bf16"))  # would raise every scale
    q, out = device.DeviceBuffer(2 * Hq * D * 4), device.DeviceBuffer(2 * Hq * D * 4)
    batch = v2.DeviceBatchTable(storage, seqs, 4)
    before = Model(storage)
    for _ in range(2):
        with pytest.raises(RuntimeError):
            v2.decode_step(storage, batch, v2.NewRows(kv.ptr, kv.ptr + 4 * D, v2.DType.BFloat16, 4 * D, 4 * D), q.ptr, out.ptr, Hq)
        assert [s.num_tokens() for s in seqs] == counts and [s.num_allocated_blocks() for s in seqs] == [2, 1]
        after = Model(storage)
        assert np.array_equal(after.bytes, before.bytes) and np.array_equal(after.scales, before.scales, equal_nan=True)


def test_one_long_prompt_beside_many_single_tokens(gpu, v2):
    """8200 pages of one sequence and a token each of 511 others: the bound of the one for each of the others would
    be more wavefronts than a launch counts."""
    H, D, bs, long, others = 2, 8, 1, 8200, 511
    pool = v2.PhysicalBlockPool(long + others, bs)
    storage = v2.QuantizedKVStorage(pool, H, D, v2.QuantFormat.Int8)
    seqs = [v2.SequenceState(i, pool) for i in range(others + 1)]
    counts = [1] * (others + 1)
    counts[300] = long
    for s, n in zip(seqs, counts):
        s.append_tokens(n)
    x = np.random.default_rng(5).standard_normal((sum(counts), 2, H, D))
    bits = to_bits(x, "bf16")
    x = from_bits(bits, "bf16")
    kv = device.to_device(bits)
    v2.write_quantized_kv(storage, seqs, counts, v2.NewRows(kv.ptr, kv.ptr + H * D * 2, v2.DType.BFloat16, 2 * H * D, 2 * H * D))
    model = Model(storage)
    got = model.values()
    table, at = pages(seqs), 0
    for r, n in enumerate(counts):  # a page is a token: within half a step of 127ths of its largest value's power of two
        ids = table[r, :n].astype(np.int64)
        assert (np.abs(got[:, ids][:, :, :, 0].transpose(1, 0, 2, 3) - x[at:at + n]) <= model.scales[:, ids].transpose(1, 0, 2)[..., None] / 2).all()
        assert (model.scales[:, ids].transpose(1, 0, 2) <= np.abs(x[at:at + n]).max(-1) * 2 / 127).all()
        at += n


def test_a_decode_step_of_more_units_than_a_launch(gpu, v2):
    """129 rows of 65535 heads: the new tokens' writes take two launches."""
    H, rows = 65535, 129
    pool = v2.PhysicalBlockPool(2 * rows, 1)
    storage = v2.QuantizedKVStorage(pool, H, 1, v2.QuantFormat.Int8)
    seqs = [v2.SequenceState(i, pool) for i in range(rows)]
    for s in seqs:
        s.append_tokens(1)
    batch = v2.DeviceBatchTable(storage, seqs, 2)
    x = np.random.default_rng(6).standard_normal((rows, 2, H))
    bits = to_bits(x, "bf16")
    x = from_bits(bits, "bf16")
    kv, out = device.to_device(bits), device.DeviceBuffer(rows * H * 4)
    q = device.to_device(np.zeros((rows, H), np.float32))
    v2.decode_step(storage, batch, v2.NewRows(kv.ptr, kv.ptr + H * 2, v2.DType.BFloat16, 2 * H, 2 * H), q.ptr, out.ptr, H)
    model = Model(storage)
    ids = pages(seqs)[:, 1].astype(np.int64)
    got, scales = model.values()[:, ids][..., 0, 0], model.scales[:, ids]
    assert (np.abs(got.transpose(1, 0, 2) - x) <= scales.transpose(1, 0, 2) / 2).all()
    assert (scales.transpose(1, 0, 2) <= np.abs(x) * 2 / 127).all()
