"""When the shared attention runs: by the tokens that the rows really share.

The C entry knows only bounds and counts every row behind the longest prefix; the
C++ layer knows the groups. A batch whose few sharers cannot pay runs as the
ordinary decode, recognised by its bits.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from test_gpu_projected_step import Model, filled


def pays(rows, kv_len, groups, tokens, H=8, Hq=32, bs=16, D=128, dtype=capi.DTYPE_BF16):
    out = C.c_int(7)
    capi.call("kvflux_paged_attention_shared_pays", rows, kv_len, H, Hq, bs, D, dtype, groups, tokens, C.byref(out))
    return out.value


def test_by_the_tokens_shared():
    """K and V of a token are 4 KiB here: 9 MB a microsecond against 5 us and 4.5 for each 256 rows and kv heads."""
    limit = 9e6 * (5 + 4.5 * 64 * 8 / 256) / 4096
    assert pays(64, 9000, 1, int(limit) + 1) == 1 and pays(64, 9000, 1, int(limit)) == 0
    assert pays(64, 9000, 1, 0) == 0
    # 128 rows of about 600 tokens, two of them behind 512 common ones, as they are and as the bounds count them
    assert pays(128, 700, 2, 512) == 0 and pays(128, 700, 2, 126 * 512) == 1
    # 2 rows behind 32768 tokens beside 126 others
    assert pays(128, 33000, 2, 32768) == 0
    assert pays(64, 9000, 1, 2 ** 64 - 1) == 1


@pytest.mark.parametrize("shape", [dict(rows=2049), dict(groups=513), dict(groups=0), dict(D=80), dict(kv_len=2 ** 31),
                                   dict(D=256, dtype=capi.DTYPE_F32)])
def test_shapes_that_the_kernel_does_not_take(shape):
    assert pays(**{**dict(rows=64, kv_len=9000, groups=1, tokens=10 ** 9), **shape}) == 0


def test_refusals():
    out = C.c_int(7)
    fn = capi.lib().kvflux_paged_attention_shared_pays
    assert fn(64, 9000, 8, 32, 16, 128, 1, 1, 10 ** 9, None) == capi.ERR_INVALID
    for bad in ((64, 9000, 8, 33, 16, 128, 1), (64, 9000, 0, 32, 16, 128, 1), (64, 9000, 8, 32, 0, 128, 1),
                (64, 9000, 8, 32, 16, 128, 5)):
        assert fn(*bad, 1, 10 ** 9, C.byref(out)) == capi.ERR_INVALID and out.value == 0


def test_workspace_holds_the_columns_there_are():
    """Partials of every row and query head once for the prefix and once for the row's own tokens, and of 256 workgroups'
    128 columns more for each, whatever the number of groups (2000 rows in 512 groups, 32/32 heads of 128: 84 MB)."""
    for rows, groups, H, Hq, D in ((2000, 512, 32, 32, 128), (2048, 1, 8, 64, 256), (64, 1, 8, 32, 128), (3, 2, 1, 300, 64)):
        size = C.c_size_t()
        capi.call("kvflux_paged_attention_shared_workspace_size", rows, 200, H, Hq, 16, D, capi.DTYPE_BF16, groups,
                  C.byref(size))
        tiles = -(-Hq // H // 128) * min(Hq // H, 128) * H  # a row's own columns, in whole streams
        most = (rows * Hq + rows * tiles + 2 * 256 * 128) * (D + 2) * 4 + rows * 64 + 5 * 256
        assert 0 < size.value <= most


@pytest.mark.gpu
@pytest.mark.parametrize("sharers", [2, 63])
def test_batches_with_few_and_many_sharers(gpu, v2, sharers):
    """64 rows, some behind 4096 common tokens, the others short ones of their own: 256 bytes a token, so two sharers
    read 1 MB again and 63 of them 65 MB, against 55 MB. The bounds alone count 64 rows both times."""
    rng = np.random.default_rng(71)
    H, Hq, D, bs, n = 1, 4, 64, 16, 64
    pool, storage = filled(v2, "BFloat16", H, D, bs, 4096 // bs + 3 * n, 5)
    base = v2.SequenceState(1, pool)
    base.append_tokens(4096 + 5)
    seqs = [base] + [base.fork_shared(10 + i) for i in range(sharers - 1)]
    for i in range(n - sharers):
        s = v2.SequenceState(100 + i, pool)
        s.append_tokens(20)
        seqs.append(s)
    table = v2.DeviceBatchTable(storage, seqs, 4096 // bs + 2)
    model = Model(rng, "BFloat16", Hq, H, D, D, False)
    q, shared, plain = (device.DeviceBuffer(n * Hq * D * 4) for _ in range(3))
    v2.decode_step_projected(storage, table, model.project(v2, rng, n), model.form(v2), q.ptr, shared.ptr, Hq)
    outs = [shared.download(np.float32)]
    for batch in (seqs, table):
        shared.fill(0xff)
        v2.paged_attention_batch_shared(storage, batch, q.ptr, shared.ptr, Hq)
        outs.append(shared.download(np.float32))
    v2.paged_attention_batch(storage, table, q.ptr, plain.ptr, Hq)
    want = plain.download(np.float32)
    for got in outs:
        assert np.array_equal(got, want) == (sharers == 2)
        assert np.abs(got - want).max() <= 1e-5
