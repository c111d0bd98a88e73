"""Writes to and reads from an 8-bit cache against their definition in 64 bits.

Scales are powers of two, so a value's division by its scale is exact in FP32 and
one rounding is left, to the nearest byte: bytes and scales are compared bit for
bit. A value read back is a product of a byte and a power of two, exact in FP32, and
rounded once to the output's type: bits again.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from quant_util import CODE, FORMAT, ITEM, VALUES, Cache, from_bits, random_table, to_bits, u64

pytestmark = pytest.mark.gpu


class Rows:
    """New rows of K and V inside a wider projection, `pad` elements between tokens."""

    def __init__(self, x, name, pad=0, shift=0):
        n, H, D = x[0].shape
        self.stride = 2 * H * D + pad
        bits = [to_bits(a, name) for a in x]
        self.x = [from_bits(b, name) for b in bits]
        flat = np.zeros(max(1, n) * self.stride + shift, bits[0].dtype)
        view = flat[shift:].reshape(-1, self.stride)
        for i in range(2):
            view[:n, i * H * D:(i + 1) * H * D] = bits[i].reshape(n, -1)
        self.buffer = device.to_device(flat)
        at = self.buffer.ptr + shift * ITEM[name]
        self.args = (at, at + H * D * ITEM[name], CODE[name], self.stride, self.stride)


def write(cache, rows, table, lens, new, offsets, most=None, stream=None):
    held = [u64(a) for a in (table, lens, new, offsets)]
    capi.call("kvflux_quant_write", *cache.args(), *rows.args, held[0].ptr, table.shape[1], held[1].ptr, held[2].ptr,
              held[3].ptr, len(lens), int(max(new)) if most is None else most, stream)
    return held


def write_tail(cache, rows, table, lens, stream=None):
    held = [u64(a) for a in (table, lens)]
    capi.call("kvflux_quant_write_tail", *cache.args(), *rows.args, held[0].ptr, table.shape[1], held[1].ptr, len(lens),
              stream)
    return held


def same(cache):
    """Scales bit for bit, and the bytes of every page and head whose scale is a number."""
    got, scales = cache.download()
    assert np.array_equal(scales, cache.scales, equal_nan=True)
    number = ~np.isnan(scales)
    assert np.array_equal(got[number], cache.bytes[number])


def step(cache, rng, table, lens, new, name, size=1.0, pad=0, shift=0, tail=False):
    lens, new = np.asarray(lens, np.int64), np.asarray(new, np.int64)
    offsets = np.cumsum(new) - new
    x = [(rng.standard_normal((int(new.sum()), cache.H, cache.D)) * size).astype(np.float32) for _ in range(2)]
    rows = Rows(x, name, pad, shift)
    held = write_tail(cache, rows, table, lens) if tail else write(cache, rows, table, lens, new, offsets)
    device.synchronize()
    del held
    for i in range(2):
        cache.write(i, table, lens, new, offsets, rows.x[i])
    same(cache)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,bs,H", [(128, 16, 8), (64, 16, 3), (256, 8, 2), (128, 64, 1), (256, 64, 2), (96, 12, 2),
                                    (72, 1, 2), (20, 5, 3), (128, 256, 1)])
def test_prompts_in_chunks(gpu, fmt, name, D, bs, H):
    """Prompts of any length in chunks that end and start inside pages, growing and shrinking values."""
    rng = np.random.default_rng([D, bs, H])
    ends = np.array([[1, 0, 3 * bs, bs + 1], [bs, 2, 3 * bs + 1, bs + 2], [4 * bs + 3, 2, 5 * bs - 1, 6 * bs]])
    cache = Cache(fmt, 25, H, bs, D)
    table = random_table(rng, ends[-1], bs, 25)
    before = np.zeros(4, np.int64)
    for now, size in zip(ends, [1.0, 30.0, 0.1]):
        step(cache, rng, table, now, now - before, name, size, pad=8)
        before = now


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("D,bs,H", [(128, 16, 8), (64, 32, 2), (80, 3, 2), (100, 16, 1)])
def test_tokens_one_by_one(gpu, fmt, name, D, bs, H):
    """A decode loop's writes: each may raise the scale of what its page holds."""
    rng = np.random.default_rng(D + bs)
    lens = np.array([1, bs, bs - 1 or 1, 2 * bs + 1, 0])
    cache = Cache(fmt, 30, H, bs, D)
    table = random_table(rng, lens + 6 * (lens > 0), bs, 30)
    for i in range(6):
        now = lens + i * (lens > 0)
        live = (now > 0).astype(np.int64)
        x = [(rng.standard_normal((len(lens), H, D)) * 2.0 ** rng.integers(-3, 4)).astype(np.float32) for _ in range(2)]
        rows = Rows(x, name)
        held = write_tail(cache, rows, table, now)
        device.synchronize()
        del held
        for which in range(2):
            cache.write(which, table, now, live, np.arange(len(lens)), rows.x[which])
        same(cache)


@pytest.mark.parametrize("shift,cache_shift", [(1, 0), (0, 4), (3, 1)])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_arrays_at_any_element(gpu, fmt, shift, cache_shift):
    rng = np.random.default_rng(5)
    cache = Cache(fmt, 9, 2, 16, 64, shift=cache_shift)
    table = random_table(rng, [40, 33], 16, 9)
    step(cache, rng, table, [30, 20], [30, 20], "bf16", shift=shift)
    step(cache, rng, table, [40, 33], [10, 13], "bf16", 4.0, shift=shift, pad=3)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_every_byte_and_the_borders_of_a_scale(gpu, fmt):
    """All values of the format, half steps between them, the top and what is just above it, the
    smallest scales, subnormals of FP32, and zeros."""
    v = VALUES[fmt][~np.isnan(VALUES[fmt])]
    p = np.unique(np.abs(v[np.abs(v) <= (448 if fmt == "e4m3" else 127)]))
    mid = (p[1:] + p[:-1]) / 2
    top = p[-1]
    x = np.concatenate([p, -p, mid, -mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    x = np.concatenate([x, np.zeros(-len(x) % 64)]).reshape(-1, 1, 64)
    rows = [x, np.full((1, 1, 64), top * (1 + 2.0 ** -23)), np.full((1, 1, 64), top * 2.0 ** -110),
            np.full((1, 1, 64), 2.0 ** -119), np.full((1, 1, 64), 2.0 ** -140), np.zeros((1, 1, 64)),
            np.full((1, 1, 64), 3.4e38), np.full((1, 1, 64), top * 2.0 ** 100)]
    x = np.concatenate(rows).astype(np.float32)
    for bs in (len(x), 1):
        cache = Cache(fmt, len(x), 1, bs, 64)
        table = np.arange(len(x) // bs, dtype=np.uint64)[None]
        r = Rows([x, -x], "f32")
        held = write(cache, r, table, [len(x)], [len(x)], [0])
        device.synchronize()
        del held
        for i in range(2):
            cache.write(i, table, [len(x)], [len(x)], [0], r.x[i])
        same(cache)
    cache = Cache(fmt, 1, 1, len(rows[0]), 64)
    r = Rows([x[:len(rows[0])]] * 2, "f32")
    held = write(cache, r, np.zeros((1, 1), np.uint64), [len(rows[0])], [len(rows[0])], [0])
    device.synchronize()
    del held
    for i in range(2):
        cache.write(i, np.zeros((1, 1), np.uint64), [len(rows[0])], [len(rows[0])], [0], r.x[i])
    same(cache)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_what_is_no_number_makes_its_page_and_head_nan(gpu, fmt, bad):
    rng = np.random.default_rng(3)
    cache = Cache(fmt, 4, 3, 16, 64)
    table = random_table(rng, [40], 16, 4)
    step(cache, rng, table, [20], [20], "f32")
    x = [rng.standard_normal((4, 3, 64)).astype(np.float32) for _ in range(2)]
    x[0][2, 1, 5] = bad
    rows = Rows(x, "f32")
    held = write(cache, rows, table, [24], [4], [0])
    device.synchronize()
    for i in range(2):
        cache.write(i, table, [24], [4], [0], rows.x[i])
    same(cache)
    page = int(table[0, 1])
    assert np.isnan(cache.scales[0, page]).tolist() == [False, True, False] and not np.isnan(cache.scales[1, page]).any()
    step(cache, rng, table, [30], [6], "f32")   # stays so
    assert np.isnan(cache.scales[0, page, 1])
    step(cache, rng, table, [30], [14], "f32")  # the page anew
    assert not np.isnan(cache.scales[0, page]).any()
    del held


def test_bad_pages_short_tables_and_bounds(gpu):
    """Page ids past the pool, positions past the table's rows, more new tokens than tokens and than
    the bound: nothing but the documented places is written."""
    rng = np.random.default_rng(4)
    cache = Cache("e4m3", 6, 2, 16, 64)
    table = random_table(rng, [64, 30], 16, 6)
    table[0, 1], table[1, 1] = 6, 2 ** 63
    step(cache, rng, table, [100, 30], [100, 30], "bf16")  # 100 tokens, pages for 64
    step(cache, rng, table, [0, 10], [0, 10], "bf16")
    x = [rng.standard_normal((64, 2, 64)).astype(np.float32) for _ in range(2)]
    rows = Rows(x, "bf16")
    held = write(cache, rows, table, [64, 10], [2 ** 40, 2 ** 40], [0, 0], most=64)
    device.synchronize()
    for i in range(2):
        cache.write(i, table, [64, 10], [64, 10], [0, 0], rows.x[i])
    same(cache)
    for most in (17, 1, 16):  # the first of them
        held += write(cache, rows, table, [64, 10], [64, 10], [0, 0], most=most)
        device.synchronize()
        for i in range(2):
            cache.write(i, table, [most, min(most, 10)], [most, min(most, 10)], [0, 0], rows.x[i])
        same(cache)
    del held


def gather(cache, table, lens, name, shift=0):
    lens = np.asarray(lens, np.int64)
    total = int(lens.sum())
    pages = -(-lens // cache.bs)
    held = [u64(a) for a in (table, lens, np.cumsum(lens) - lens, np.cumsum(pages) - pages)]
    size = total * cache.H * cache.D
    out = [device.DeviceBuffer((size + 64 + shift) * ITEM[name]) for _ in range(2)]
    for o in out:
        o.fill(0xa5)
    capi.call("kvflux_quant_gather", *cache.args(), held[0].ptr, table.shape[1], *(h.ptr for h in held[1:]), len(lens),
              int(pages.sum()), *(o.ptr + shift * ITEM[name] for o in out), CODE[name], None)
    device.synchronize()
    raw = [o.download({"f32": np.uint32}.get(name, np.uint16)) for o in out]
    for r in raw:
        assert np.all(r[:shift].view(np.uint8) == 0xa5) and np.all(r[shift + size:].view(np.uint8) == 0xa5)
    return [r[shift:shift + size].reshape(total, cache.H, cache.D) for r in raw]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,bs,H,shift,cache_shift", [(128, 16, 8, 0, 0), (64, 8, 3, 0, 0), (256, 64, 2, 0, 0),
                                                      (96, 12, 2, 0, 0), (20, 5, 3, 0, 0), (64, 16, 2, 1, 0),
                                                      (64, 16, 2, 0, 2)])
def test_read_back(gpu, fmt, name, D, bs, H, shift, cache_shift):
    rng = np.random.default_rng([D, bs])
    lens = np.array([1, 0, 3 * bs, 2 * bs + 1, 0, bs - 1 or 1, 70])
    blocks = int((-(-lens // bs)).sum()) + 2
    cache = Cache(fmt, blocks, H, bs, D, shift=cache_shift)
    cache.fill(rng, spread=6.0)
    table = random_table(rng, lens, bs, blocks)
    got = gather(cache, table, lens, name, shift)
    values = cache.values()
    for i in range(2):
        want = np.concatenate([values[i, table[r, :-(-n // bs)].astype(np.int64)].transpose(0, 2, 1, 3).reshape(-1, H, D)[:n]
                               for r, n in enumerate(lens) if n])
        assert np.array_equal(got[i], to_bits(want, name))


def test_read_back_of_all_bytes_and_scales(gpu):
    """Every byte at scales of every kind, NaN among them, in every output type."""
    for fmt in FORMAT:
        cache = Cache(fmt, 8, 1, 4, 64)
        cache.bytes[:] = np.arange(256, dtype=np.uint8).reshape(4, 64)
        cache.scales[:, :, 0] = np.float32([1.0, 2.0 ** -110, 0.0123, 2.0 ** -20, 3e4, 7.7e-7, np.nan, 0.0])
        cache.upload()
        table = np.arange(8, dtype=np.uint64)[None]
        for name in CODE:
            got = gather(cache, table, [32], name)
            with np.errstate(over="ignore"):
                want = cache.values().astype(np.float32).transpose(0, 1, 3, 2, 4).reshape(2, 32, 1, 64)
                want = [from_bits(to_bits(w, name), name) for w in want]
            for i in range(2):
                assert np.array_equal(from_bits(got[i], name), want[i], equal_nan=True), (fmt, name)


def test_read_back_skips_bad_pages(gpu):
    rng = np.random.default_rng(8)
    cache = Cache("int8", 5, 2, 16, 64)
    cache.fill(rng)
    table = random_table(rng, [48, 20], 16, 5)
    table[0, 1] = 5
    got = gather(cache, table, [48, 20], "f32")
    assert np.all(got[0][16:32].view(np.uint8) == 0xa5) and np.all(got[1][16:32].view(np.uint8) == 0xa5)
    want = cache.values()[0, int(table[0, 2])].transpose(1, 0, 2)
    assert np.array_equal(got[0][32:48].view(np.float32), want.astype(np.float32))
