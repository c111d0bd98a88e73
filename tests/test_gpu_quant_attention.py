"""kvflux_quant_attention against attention in 64 bits over the values the cache holds.

Tolerance: 1e-5 of the largest value of V that a row sees, the contract of the other
exact attention calls. Where it comes from: a score is a sum of D products of FP32
queries (in parts, 2^-23 of each) and bytes, rounded D times to FP32: for scores of
up to 6 sqrt(D) 2^-24 6 = 4e-6 (the roundings' signs differ); an error d of a score
moves an output by at most 2 d max|v|, and by far less where many keys share the weight.
The weights' parts (2^-23 each), their sums (compensated) and the exponential (2^-22)
add 1e-6.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from quant_util import VALUES, Cache, attention, random_table, u64

pytestmark = pytest.mark.gpu


def workspace_size(rows, kv_len, H, Hq, bs, D):
    size = C.c_size_t(99)
    capi.call("kvflux_quant_attention_workspace_size", rows, kv_len, H, Hq, bs, D, C.byref(size))
    return size.value


class Decode:
    def __init__(self, cache, table, lens, q, kv_len=None, fill=0xff):
        rows, Hq, D = q.shape
        self.q, self.rows = q, rows
        self.held = [u64(table), u64(lens), device.to_device(q.astype(np.float32))]
        self.kv_len = int(max(lens)) if kv_len is None else kv_len
        size = workspace_size(rows, self.kv_len, cache.H, Hq, cache.bs, D)
        self.work = device.DeviceBuffer(size + 256)
        self.work.fill(fill)  # needs no initialisation
        self.out = device.DeviceBuffer(q.size * 4 + 256)
        self.out.fill(0xa5)
        self.args = (*cache.args(), self.held[0].ptr, table.shape[1], self.held[1].ptr, self.kv_len, rows, Hq,
                     self.held[2].ptr, self.out.ptr, self.work.ptr if size else None, size)
        self.size = size

    def run(self, stream=None):
        capi.call("kvflux_quant_attention", *self.args, stream)

    def result(self):
        device.synchronize()
        assert np.all(self.out.download(np.uint8, offset=self.q.size * 4) == 0xa5)
        assert np.all(self.work.download(np.uint8)[self.size:] == self.work.download(np.uint8)[-1])
        return self.out.download(np.float32, self.q.size).reshape(self.q.shape)


def biggest(cache, table, n):
    pages = [int(p) for p in table[:-(-n // cache.bs)] if p < cache.blocks]
    if not pages:
        return 1.0
    return np.nanmax(np.abs(VALUES[cache.fmt][cache.bytes[1, pages]] * cache.scales[1, pages, :, None, None].astype(np.float64)))


def check(cache, table, lens, q, got, tolerance=1e-5):
    for r, n in enumerate(lens):
        want = attention(cache, table[r], int(n), q[r:r + 1])[0]
        assert np.isfinite(got[r]).all(), r
        assert np.abs(got[r] - want).max() <= tolerance * biggest(cache, table[r], int(n)), (r, n)


def make(fmt, H, G, D, bs, lens, seed, spare=3, **fill):
    rng = np.random.default_rng(seed)
    blocks = int(sum(-(-int(n) // bs) for n in lens)) + spare
    cache = Cache(fmt, blocks, H, bs, D)
    cache.fill(rng, **fill)
    table = random_table(rng, lens, bs, blocks)
    q = rng.standard_normal((len(lens), H * G, D)).astype(np.float32)
    return rng, cache, table, q


def run(cache, table, lens, q, **kw):
    d = Decode(cache, table, lens, q, **kw)
    d.run()
    return d.result()


# A bound of the lengths from which every call is cut into shares.
SHARES = 2049


def check_both(cache, table, lens, q):
    """With the lengths' own bound, and in shares."""
    check(cache, table, lens, q, run(cache, table, lens, q))
    if max(lens) < SHARES:
        check(cache, table, lens, q, run(cache, table, lens, q, kv_len=SHARES))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 8, 32, 64, 1, 5, 12])
def test_lengths_and_pages(gpu, fmt, D, bs):
    """Every length around a tile's and a page's borders, in one launch (of four wavefronts, of eight) and in shares."""
    lens = np.array([0, 1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 300, 511, 512])
    rng, cache, table, q = make(fmt, 2, 4, D, bs, lens, [D, bs])
    for bound in (None, 1000, table.shape[1] * bs + SHARES):
        check(cache, table, lens, q, run(cache, table, lens, q, kv_len=bound))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [16, 32, 48, 80, 96, 112, 144, 192, 240])
@pytest.mark.parametrize("bs", [16, 5])
def test_head_sizes_that_fill_part_of_a_kernel(gpu, fmt, D, bs):
    lens = np.array([0, 1, 33, 300, 512])
    rng, cache, table, q = make(fmt, 3, 5, D, bs, lens, [D, bs], spare=0)
    for bound in (None, 1000, SHARES):
        check(cache, table, lens, q, run(cache, table, lens, q, kv_len=bound))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("H,G", [(8, 4), (4, 7), (1, 12), (8, 1), (2, 16), (1, 17), (2, 33), (3, 5), (1, 71)])
def test_groups(gpu, fmt, H, G):
    lens = np.array([700, 1, 45, 0, 1300])
    rng, cache, table, q = make(fmt, H, G, 128, 16, lens, [H, G])
    for most in (1300, 1000, 200):
        short = np.minimum(lens, most)
        check(cache, table, short, q, run(cache, table, short, q))


@pytest.mark.parametrize("D,bs,H,G,rows,hi", [(128, 16, 8, 4, 1, 40000), (128, 16, 8, 4, 40, 3000), (64, 64, 4, 4, 9, 6000),
                                              (256, 16, 2, 8, 6, 5000), (128, 3, 2, 4, 5, 2500), (128, 16, 1, 12, 1, 9000),
                                              (64, 16, 1, 1, 300, 700)])
def test_many_and_long_rows(gpu, D, bs, H, G, rows, hi):
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, hi + 1, rows)
    lens[rng.integers(rows)] = hi
    if rows > 20:
        lens[[3, 7]] = 0
    rng, cache, table, q = make("e4m3" if rows % 2 else "int8", H, G, D, bs, lens, rows)
    check_both(cache, table, lens, q)


def test_more_rows_than_a_launch_plans(gpu):
    lens = np.random.default_rng(1).integers(0, 40, 4100)
    lens[[5, 2047, 2048, 4099]] = [900, 700, 650, 530]
    rng, cache, table, q = make("e4m3", 1, 2, 64, 16, lens, 3)
    check_both(cache, table, lens, q)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs", [8, 16, 48, 3])
def test_missing_pages_drop_out(gpu, fmt, bs):
    lens = np.array([600, 90, 33, 20])
    rng, cache, table, q = make(fmt, 2, 4, 128, bs, lens, bs)
    table[0, [0, 3, 7]], table[1, 1], table[3, :] = cache.blocks, 2 ** 64 - 1, 2 ** 63
    for bound in (None, SHARES):
        got = run(cache, table, lens, q, kv_len=bound)
        check(cache, table, lens, q, got)
        assert not got[3].any()
    short = table[:, :2].copy()  # rows end before their tokens do
    check(cache, short, np.minimum(lens, 2 * bs), q, run(cache, short, lens, q))


@pytest.mark.parametrize("bs,D", [(16, 128), (64, 64), (5, 128), (16, 256), (16, 96), (16, 100)])
def test_what_lies_behind_a_row_is_not_seen(gpu, bs, D):
    """NaN bytes and scales behind a row's end, in its last page and in pages it does not use."""
    lens = np.array([1, 37, 70, 530])
    rng, cache, table, q = make("e4m3", 2, 4, D, bs, lens, bs)
    used = {int(p) for r, n in enumerate(lens) for p in table[r, :-(-int(n) // bs)]}
    for page in set(range(cache.blocks)) - used:
        cache.scales[:, page] = np.nan
    for r, n in enumerate(lens):
        if n % bs:
            cache.bytes[:, int(table[r, n // bs]), :, n % bs:] = 0x7f
    cache.upload()
    check_both(cache, table, lens, q)


@pytest.mark.parametrize("D", [128, 96, 100])
def test_a_scale_or_byte_that_is_nan_is_seen(gpu, D):
    lens = np.array([40, 600, 33])
    rng, cache, table, q = make("e4m3", 2, 2, D, 16, lens, 1)
    cache.scales[0, int(table[0, 1]), 0] = np.nan
    cache.scales[1, int(table[1, 30]), 1] = np.nan
    cache.bytes[1, int(table[2, 2]), 1, 0, 5] = 0xff
    cache.upload()
    for bound in (None, SHARES):
        got = run(cache, table, lens, q, kv_len=bound).reshape(3, 2, 2, D)
        assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()
        assert np.isnan(got[1, 1]).all() and np.isfinite(got[1, 0]).all()
        assert np.isnan(got[2, 1, :, 5]).all() and np.isfinite(np.delete(got[2], 5, -1)).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scales_of_any_origin(gpu, fmt):
    """Scales that are no powers of two, sizes from 2^-60 to 2^40 in one row."""
    lens = np.array([900, 64])
    rng, cache, table, q = make(fmt, 2, 4, 128, 16, lens, 4, scales=1.37)
    check_both(cache, table, lens, q)
    cache.scales[1] *= np.exp2(rng.integers(-60, 41, cache.scales[1].shape)).astype(np.float32)
    cache.upload()
    check_both(cache, table, lens, q)


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** 30])
def test_queries_and_keys_of_any_size(gpu, size):
    """Queries times `size`, keys over it: the same scores."""
    lens = np.array([600, 100])
    rng, cache, table, q = make("e4m3", 2, 4, 128, 16, lens, 6)
    want = run(cache, table, lens, q)
    cache.scales[0] /= np.float32(size)
    cache.upload()
    q *= np.float32(size)
    got = run(cache, table, lens, q)
    check(cache, table, lens, q, got)
    assert np.array_equal(got, want)  # powers of two throughout


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [500, 9000])
def test_a_dominant_key_and_thousands_of_small_ones(gpu, fmt, n):
    """One key 17 above the others (their weights 2^-25): their sum is not lost. A weight's parts end
    2^-40 below the largest weight; four FP32 roundings of a score of 24.5 (in powers of two) are 2^-20 each."""
    rng, cache, table, q = make(fmt, 1, 4, 128, 16, [n], 8)
    cache.scales[:] = 2.0 ** -6
    one = np.uint8(0x38 if fmt == "e4m3" else 1)  # 1.0
    big = np.uint8(0x7e if fmt == "e4m3" else 127)
    cache.bytes[0] = 0
    cache.bytes[1] = big
    page = int(table[0, 3])
    cache.bytes[0, page, 0, 5] = one
    cache.bytes[1, page, 0, 5] = 0
    cache.upload()
    q[:] = 17.0 * np.sqrt(128) / 128 * 64
    got = run(cache, table, [n], q)
    want = attention(cache, table[0], n, q)
    assert want.min() > 0
    top = biggest(cache, table[0], n)
    np.testing.assert_allclose(got, want, rtol=4 * 2.0 ** -20, atol=n * 2.0 ** -40 * top)


def test_rows_of_equal_keys_give_the_mean(gpu):
    """No score differs: weights of 1 for up to 20000 tokens."""
    lens = np.array([20000])
    rng, cache, table, q = make("int8", 1, 2, 64, 16, lens, 8, spread=0.0)
    cache.bytes[0] = 5
    cache.scales[0] = 1.0
    cache.upload()
    check_both(cache, table, lens, q)


def test_the_same_bits_again(gpu):
    lens = np.random.default_rng(2).integers(0, 2500, 50)
    rng, cache, table, q = make("e4m3", 4, 7, 128, 16, lens, 2)
    d = Decode(cache, table, lens, q)
    d.run()
    first = d.result()
    for _ in range(3):
        d.work.fill(0x5a)
        d.run()
        assert np.array_equal(d.result(), first)


@pytest.mark.parametrize("D,shift", [(84, 0), (100, 0), (512, 0), (20, 0), (128, 1), (64, 8)])
def test_generic_head_sizes_and_alignments(gpu, D, shift):
    rng = np.random.default_rng(D)
    lens = np.array([0, 1, 63, 64, 65, 400, 700])
    blocks = int(sum(-(-n // 6) for n in lens))
    for fmt in ("e4m3", "int8"):
        cache = Cache(fmt, blocks, 2, 6, D, shift=shift)
        cache.fill(rng)
        table = random_table(rng, lens, 6, blocks)
        q = rng.standard_normal((len(lens), 6, D)).astype(np.float32)
        check_both(cache, table, lens, q)


@pytest.mark.parametrize("H,G", [(300, 1), (255, 2), (100, 17)])
def test_more_heads_than_a_workgroup_has_threads(gpu, H, G):
    """A row without tokens beside a long one, or alone: whatever the workspace held, it gives zeros."""
    for lens in ([0], [2100], [0, 70]):
        lens = np.array(lens)
        rng, cache, table, q = make("int8", H, G, 64, 16, lens, [H, G])
        for fill in (0, 0xff):
            got = run(cache, table, lens, q, kv_len=max(SHARES, lens.max()), fill=fill)
            check(cache, table, lens, q, got)
            assert not got[lens == 0].any()


def test_two_streams_with_workspaces_of_their_own(gpu):
    lens = np.random.default_rng(3).integers(1, 3000, 30)
    rng, cache, table, q = make("int8", 4, 4, 128, 32, lens, 5)
    a, b = Decode(cache, table, lens, q), Decode(cache, table, lens[::-1].copy().clip(max=lens), q)
    streams = [device.Stream(), device.Stream()]
    for _ in range(5):
        a.run(streams[0].handle)
        b.run(streams[1].handle)
    for s in streams:
        s.synchronize()
    check(cache, table, lens, q, a.result())
    check(cache, table, lens[::-1].clip(max=lens), q, b.result())


def test_an_undersized_workspace_is_refused(gpu):
    lens = np.array([600, 2100])
    rng, cache, table, q = make("e4m3", 2, 4, 128, 16, lens, 1)
    d = Decode(cache, table, lens, q)
    with pytest.raises(capi.KvfluxError) as e:
        capi.call("kvflux_quant_attention", *d.args[:-1], d.size - 1, None)
    assert e.value.status == capi.ERR_INVALID


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,G", [(8, 4), (1, 1), (4, 40), (300, 1)])
def test_a_workspace_for_the_largest_call_does_for_smaller_ones(gpu, H, G, D):
    rows = [1, 2, 7, 31, 32, 33, 63, 64, 128, 255, 256, 300, 2048, 5000]
    bounds = [1, 512, 513, 1024, 1025, 2048, 2049, 4096, 100000]
    sizes = np.array([[workspace_size(r, n, H, H * G, 16, D) for n in bounds] for r in rows])
    assert (np.diff(sizes, axis=0) >= 0).all() and (np.diff(sizes, axis=1) >= 0).all()
    assert sizes[0, -1] > 0 and not sizes[:, :2].any()


@pytest.mark.parametrize("H,rows", [(8, 40), (1, 260)])
def test_a_bound_at_which_many_rows_take_one_launch_and_few_are_cut(gpu, H, rows):
    lens = np.random.default_rng(H).integers(0, 1500, rows)
    lens[[0, 30]] = 1500
    rng, cache, table, q = make("e4m3", H, 2, 128, 16, lens, 7)
    check(cache, table, lens, q, run(cache, table, lens, q))
    check(cache, table[:9], lens[:9], q[:9], run(cache, table[:9].copy(), lens[:9], q[:9].copy()))
