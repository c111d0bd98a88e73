"""Queries of any size on FP16 caches: the ordinary batch decode
and the exact prefill.

FP16 parts of a query end at 2^-24 and at 65504, whatever the query's size. With
keys of the inverse size the scores are those of unit data, and so is the 1e-5 of
the exact paths' contract.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from test_gpu_shared_attention import TOL, Batch, from_bits, ordinary


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


PREFILLS = [  # heads, head size, tokens, queries of them, and (key splits, key parts) of the launch
    ((4, 2), 64, 200, 200, (1, 1)), ((32, 32), 64, 400, 400, (1, 2)), ((4, 2), 128, 200, 77, (1, 2)),
    ((64, 64), 128, 600, 600, (1, 1)), ((8, 1), 128, 3000, 64, (10, 2)), ((2, 1), 64, 6000, 100, (19, 1))]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREFILLS, ids=lambda c: f"{c[0][0]}x{c[0][1]}x{c[1]}-{c[2]}-{c[3]}")
@pytest.mark.parametrize("size", [1e-8, 1e-4, 1e-3, 0.1, 1024.0, 2.0 ** 20])
def test_exact_prefill(gpu, size, case):
    """One and two key parts, whole keys and keys split over workgroups; seven query rows compared."""
    (Hq, H), D, kv, n, plan = case
    b = batch(size, (Hq, H), D, 16, lens=(kv,)).upload(bound=None)
    rng = np.random.default_rng(42)
    q = (rng.standard_normal((n, Hq, D)) * size).astype(np.float32)
    qd, out = device.to_device(q), device.to_device(np.full(q.shape, 999.0, np.float32))
    nbytes = C.c_size_t()
    capi.call("kvflux_paged_prefill_workspace_size", H, D, kv, n, Hq, C.byref(nbytes))
    splits, parts = C.c_uint32(), C.c_uint32()
    capi.call("kvflux_paged_prefill_plan", H, D, capi.DTYPE_F16, 1, kv, n, Hq, int(nbytes.value > 0), C.byref(splits),
              C.byref(parts))
    assert (splits.value, parts.value) == plan
    ws = device.DeviceBuffer(max(1, nbytes.value))
    capi.call("kvflux_paged_prefill_exact", b.dev["k"].ptr, b.dev["v"].ptr, b.pages, H, 16, D, capi.DTYPE_F16,
              b.dev["table"].ptr, b.table.shape[1], kv, n, Hq, qd.ptr, out.ptr, ws.ptr, nbytes.value, None)
    device.synchronize()
    got = out.download(np.float32).reshape(q.shape)
    t = np.arange(kv)
    page = b.table[0, t // 16].astype(np.int64)
    k, v = (from_bits(x, "f16")[page, :, t % 16] for x in (b.k, b.v))  # [kv][H][D]
    for r in range(0, n, -(-n // 7)):
        seen = kv - n + r + 1
        for h in range(Hq):
            s = k[:seen, h // (Hq // H)] @ q[r, h].astype(np.float64) / np.sqrt(D)
            w = np.exp(s - s.max())
            want = w @ v[:seen, h // (Hq // H)] / w.sum()
            assert np.abs(got[r, h] - want).max() <= TOL, (r, h, np.abs(got[r, h] - want).max())
