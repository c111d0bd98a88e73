"""Calls of the C++ layer on an 8-bit cache that the shape limits of a kernel end, and ones
that they must not end: what fails changes nothing, what fits is done."""
from __future__ import annotations

import numpy as np
import pytest

from kvflux_amd import device
from quant_util import to_bits
from test_gpu_quantized_kv import Model

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
