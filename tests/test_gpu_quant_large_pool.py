"""8-bit caches of more than 2^32 bytes: every call gives on pages from both ends of such a pool,
bit for bit, what it gives on a small one that holds the same tokens."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from quant_util import CODE, FORMAT, random_table, to_bits, u64

pytestmark = pytest.mark.gpu

H, G, BS = 4, 4, 16
LENS = np.array([700, 33, 1, 130])
TOKENS = int(LENS.sum())


class Pool:
    def __init__(self, blocks, D, shift=0):
        self.cache = [device.DeviceBuffer(blocks * H * BS * D + shift) for _ in range(2)]
        self.scales = [device.DeviceBuffer(blocks * H * 4) for _ in range(2)]
        for s in self.scales:
            s.fill(0)
        self.head = (self.cache[0].ptr + shift, self.cache[1].ptr + shift, self.scales[0].ptr, self.scales[1].ptr, blocks, H, BS, D)


def everything(pool, fmt, D, table, rows, q, bound):
    """The prompts written, one more token each by the tail form, read back, decoded, and attended to as prompts."""
    head, table_at, width = (*pool.head, FORMAT[fmt]), u64(table), table.shape[1]
    bits = device.to_device(to_bits(rows, "bf16"))
    prompts = LENS - 1
    lens, new, offsets = u64(LENS), u64(prompts), u64(np.cumsum(prompts) - prompts)
    kv = (bits.ptr, bits.ptr + H * D * 2, CODE["bf16"], 2 * H * D, 2 * H * D)
    capi.call("kvflux_quant_write", *head, *kv, table_at.ptr, width, new.ptr, new.ptr, offsets.ptr, len(LENS), int(prompts.max()), None)
    tail = bits.ptr + int(prompts.sum()) * 4 * H * D
    capi.call("kvflux_quant_write_tail", *head, tail, tail + H * D * 2, *kv[2:], table_at.ptr, width, lens.ptr, len(LENS), None)
    pages = -(-LENS // BS)
    starts, outs = u64(np.cumsum(LENS) - LENS), [device.DeviceBuffer(TOKENS * H * D * 4) for _ in range(2)]
    page_starts = u64(np.cumsum(pages) - pages)
    capi.call("kvflux_quant_gather", *head, table_at.ptr, width, lens.ptr, starts.ptr, page_starts.ptr, len(LENS), int(pages.sum()),
              outs[0].ptr, outs[1].ptr, CODE["f32"], None)
    results = [o.download(np.float32) for o in outs]
    query, size = device.to_device(q), C.c_size_t()
    out = device.DeviceBuffer(q.nbytes)
    capi.call("kvflux_quant_attention_workspace_size", len(LENS), bound, H, H * G, BS, D, C.byref(size))
    work = device.DeviceBuffer(size.value + 8)
    capi.call("kvflux_quant_attention", *head, table_at.ptr, width, lens.ptr, bound, len(LENS), H * G, query.ptr, out.ptr, work.ptr,
              size.value, None)
    results.append(out.download(np.float32, len(LENS) * H * G * D))
    most = int(LENS.max())
    capi.call("kvflux_quant_prefill_workspace_size", len(LENS), most, bound, H, H * G, BS, D, C.byref(size))
    more = device.DeviceBuffer(size.value + 8)
    capi.call("kvflux_quant_prefill", *head, table_at.ptr, width, lens.ptr, lens.ptr, starts.ptr, len(LENS), most, bound, H * G,
              query.ptr, out.ptr, more.ptr, size.value, None)
    results.append(out.download(np.float32))
    device.synchronize()
    return results


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,shift,bound", [(128, 0, 700), (128, 0, 5000), (64, 0, 2049), (96, 0, 700), (100, 0, 700), (128, 4, 700)])
def test_pages_past_32_bits(gpu, fmt, D, shift, bound):
    rng = np.random.default_rng(D + shift)
    used = int((-(-LENS // BS)).sum())
    blocks = (1 << 32) // (H * BS * D) + used + 1
    rows = rng.standard_normal((TOKENS, 2, H, D)).astype(np.float32)
    q = rng.standard_normal((TOKENS, H * G, D)).astype(np.float32)
    small = random_table(rng, LENS, BS, used + 1)
    # The same pages: the upper half of them at the large pool's end.
    large = np.where(small <= used // 2, small, np.where(small <= used, small + np.uint64(blocks - used - 1), small))
    got = everything(Pool(blocks, D, shift), fmt, D, large, rows, q, bound)
    want = everything(Pool(used + 1, D, shift), fmt, D, small, rows, q, bound)
    assert int(large[large < blocks].max()) * H * BS * D > 1 << 32
    for a, b in zip(got, want):
        assert np.isfinite(b).all() and np.array_equal(a, b)


@pytest.mark.parametrize("call", ["decode", "prompts"])
def test_more_rows_than_a_grid_holds(gpu, call):
    """20000 rows of 1024 heads, a workgroup each: past 2^32 threads. One token a row: its values come back."""
    rows, heads, D, blocks = 20000, 1024, 8, 50
    rng = np.random.default_rng(3)
    v = rng.integers(0, 0x7f, (blocks, heads, 1, D)).astype(np.uint8)
    cache, scales = [device.to_device(v), device.to_device(v)], device.to_device(np.full((blocks, heads), 0.5, np.float32))
    pages = rng.integers(0, blocks, rows)
    table, ones, offsets = u64(pages[:, None]), u64(np.ones(rows)), u64(np.arange(rows))
    q, out = device.DeviceBuffer(rows * heads * D * 4), device.DeviceBuffer(rows * heads * D * 4)
    q.fill(0)
    out.fill(0xa5)
    head = (cache[0].ptr, cache[1].ptr, scales.ptr, scales.ptr, blocks, heads, 1, D, capi.QUANT_INT8, table.ptr, 1)
    if call == "decode":
        capi.call("kvflux_quant_attention", *head, ones.ptr, 1, rows, heads, q.ptr, out.ptr, None, 0, None)
    else:
        capi.call("kvflux_quant_prefill", *head, ones.ptr, ones.ptr, offsets.ptr, rows, 1, 1, heads, q.ptr, out.ptr, None, 0, None)
    for r in (0, 1, 9999, 16382, 16383, 16384, 19999):
        got = out.download(np.float32, heads * D, offset=r * heads * D * 4).reshape(heads, D)
        assert np.array_equal(got, v[pages[r], :, 0].astype(np.float32) * 0.5), r
