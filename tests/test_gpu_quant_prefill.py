"""kvflux_quant_prefill against causal attention in 64 bits over the values the cache holds.

Tolerance: as the decode's (test_gpu_quant_attention.py), 1e-5 of the largest value of V
that a query sees: the same parts, sums and scales.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from quant_util import VALUES, Cache, attention, random_table, u64

pytestmark = pytest.mark.gpu


class Prefill:
    def __init__(self, cache, table, lens, new, q, offsets=None, most=None, kv_len=None):
        Hq = q.shape[1]
        lens, new = np.asarray(lens), np.asarray(new)
        self.offsets = np.cumsum(new) - new if offsets is None else np.asarray(offsets)
        self.lens, self.new, self.q = lens, new, q
        self.held = [u64(table), u64(lens), u64(new), u64(self.offsets), device.to_device(q.astype(np.float32))]
        most, kv_len = int(max(new)) if most is None else most, int(max(lens)) if kv_len is None else kv_len
        size = C.c_size_t(0)
        capi.call("kvflux_quant_prefill_workspace_size", len(lens), most, kv_len, cache.H, Hq, cache.bs, cache.D, C.byref(size))
        self.size = size.value
        self.work = device.DeviceBuffer(self.size + 256)
        self.work.fill(0xff)  # needs no initialisation
        self.out = device.DeviceBuffer(q.size * 4 + 256)
        self.out.fill(0xa5)
        self.args = (*cache.args(), self.held[0].ptr, table.shape[1], self.held[1].ptr, self.held[2].ptr, self.held[3].ptr,
                     len(lens), most, kv_len, Hq, self.held[4].ptr, self.out.ptr, self.work.ptr if self.size else None,
                     self.size)

    def run(self, stream=None):
        capi.call("kvflux_quant_prefill", *self.args, stream)

    def result(self):
        device.synchronize()
        assert np.all(self.out.download(np.uint8, offset=self.q.size * 4) == 0xa5)
        assert np.all(self.work.download(np.uint8, offset=self.size) == 0xff)
        return self.out.download(np.float32, self.q.size).reshape(self.q.shape)


def biggest(cache, table, n):
    pages = [int(p) for p in table[:-(-n // cache.bs)] if p < cache.blocks]
    if not pages:
        return 1.0
    return np.nanmax(np.abs(VALUES[cache.fmt][cache.bytes[1, pages]] * cache.scales[1, pages, :, None, None].astype(np.float64)))


def check(cache, table, call, got, tolerance=1e-5, some=None):
    """All queries, or `some` of every sequence (its first, last and some between)."""
    for r, (n, m) in enumerate(zip(call.lens, call.new)):
        n, m, at = int(n), int(m), int(call.offsets[r])
        if m == 0:
            continue
        rows = np.arange(m) if some is None or m <= some else np.unique(np.r_[0, m - 1, np.random.default_rng(r).integers(0, m, some)])
        want = attention(cache, table[r], n, call.q[at + rows], visible=n - m + rows + 1)
        assert np.isfinite(got[at + rows]).all(), r
        err = np.abs(got[at + rows] - want).max((1, 2))
        assert err.max() <= tolerance * biggest(cache, table[r], n), (r, n, m, rows[err.argmax()], err.max())


def make(fmt, H, G, D, bs, lens, new, seed, spare=3, **fill):
    rng = np.random.default_rng(seed)
    blocks = int(sum(-(-int(n) // bs) for n in lens)) + spare
    cache = Cache(fmt, blocks, H, bs, D)
    cache.fill(rng, **fill)
    table = random_table(rng, lens, bs, blocks)
    q = rng.standard_normal((int(sum(new)), H * G, D)).astype(np.float32)
    return rng, cache, table, q


def run(cache, table, lens, new, q, **kw):
    call = Prefill(cache, table, lens, new, q, **kw)
    call.run()
    return call, call.result()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 8, 64, 1, 5, 48])
def test_whole_prompts(gpu, fmt, D, bs):
    lens = new = np.array([1, 63, 0, 64, 65, 130, 200])
    rng, cache, table, q = make(fmt, 2, 4, D, bs, lens, new, [D, bs])
    call, got = run(cache, table, lens, new, q)
    check(cache, table, call, got)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [16, 32, 48, 80, 96, 112, 144, 192, 240])
@pytest.mark.parametrize("bs", [16, 5])
def test_head_sizes_that_fill_part_of_a_kernel(gpu, fmt, D, bs):
    lens, new = np.array([1, 0, 65, 130, 300]), np.array([1, 0, 65, 3, 290])
    rng, cache, table, q = make(fmt, 2, 5, D, bs, lens, new, [D, bs], spare=0)
    for most, bound in ((290, 300), (290, 3000), (290, 6000), (1000, 200000)):
        call, got = run(cache, table, lens, new, q, most=most, kv_len=bound)
        check(cache, table, call, got, some=10)
    few = np.minimum(lens, 200)
    call, got = run(cache, table, few, np.minimum(new, few), q[:int(np.minimum(new, few).sum())])
    check(cache, table, call, got, some=10)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs,H,G", [(16, 2, 4), (8, 2, 4), (64, 1, 7), (1, 2, 1), (5, 1, 17), (48, 1, 300)])
def test_bounds_past_the_lengths(gpu, fmt, D, bs, H, G):
    """What is chosen by the bounds (wavefronts, splits) on short sequences, with a page missing."""
    lens, new = np.array([1, 63, 0, 64, 65, 130, 200]), np.array([1, 63, 0, 2, 65, 1, 190])
    rng, cache, table, q = make(fmt, H, G, D, bs, lens, new, [D, bs])
    for bound in (400, 3000, 4096, 20000):
        call, got = run(cache, table, lens, new, q, most=max(200, 129 // G + 1), kv_len=bound)
        check(cache, table, call, got, some=20)
        table[6, 1] = cache.blocks


@pytest.mark.parametrize("D,bs,H,G", [(128, 16, 8, 4), (64, 32, 4, 7), (256, 16, 2, 8), (128, 3, 1, 12), (128, 16, 1, 17),
                                      (64, 16, 1, 71), (128, 16, 8, 1), (128, 16, 1, 300)])
def test_chunks_behind_a_prefix(gpu, D, bs, H, G):
    """The next tokens of sequences that are cached already, one token to many."""
    lens, new = np.array([700, 45, 1000, 33, 129]), np.array([100, 45, 1, 2, 64])
    rng, cache, table, q = make("e4m3" if G % 2 else "int8", H, G, D, bs, lens, new, [H, G])
    call, got = run(cache, table, lens, new, q)
    check(cache, table, call, got, some=12)


@pytest.mark.parametrize("fmt,D,bs,n,m", [("e4m3", 128, 16, 9000, 40), ("int8", 64, 16, 40000, 70), ("e4m3", 256, 16, 5000, 9),
                                          ("int8", 128, 1, 5000, 300), ("e4m3", 128, 7, 3001, 1), ("e4m3", 128, 16, 33000, 130)])
def test_keys_split_over_workgroups(gpu, fmt, D, bs, n, m):
    """A short chunk behind a long prefix; pages of several windows."""
    rng, cache, table, q = make(fmt, 2, 4, D, bs, [n, 20], [m, 20], [n, m])
    call, got = run(cache, table, [n, 20], [m, 20], q)
    assert call.size > 0
    check(cache, table, call, got, some=6)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs,D,bound", [(16, 128, 300), (16, 128, 900), (16, 128, 5000), (5, 128, 900), (32, 64, 900), (3, 64, 300),
                                        (16, 256, 900)])
@pytest.mark.parametrize("order", ["rising", "mixed", "falling"])
def test_scales_that_a_query_does_not_see(gpu, fmt, bs, D, bound, order):
    """Scales of V from 2^-60 to 2^60 along a sequence: each query is as exact as the values that it sees are
    large, whatever the pages behind it hold."""
    n, m = 280, 200
    rng, cache, table, q = make(fmt, 2, 4, D, bs, [n], [m], [D, bs])
    pages = table[0].astype(np.int64)
    sizes = np.linspace(-60, 60, len(pages)).round()
    sizes = {"rising": sizes, "falling": sizes[::-1], "mixed": rng.permutation(sizes)}[order]
    cache.scales[1, pages] *= np.exp2(sizes).astype(np.float32)[:, None]
    cache.upload()
    q *= 0.1  # weights of one size: the seen values, not the scores, decide
    call, got = run(cache, table, [n], [m], q, kv_len=bound)
    for i in range(m):
        see = n - m + i + 1
        want = attention(cache, table[0], see, q[i:i + 1])[0]
        values = np.abs(VALUES[fmt][cache.bytes[1, pages]] * cache.scales[1, pages, :, None, None].astype(np.float64))
        top = values.transpose(0, 2, 1, 3).reshape(-1, 2 * D)[:see].max()
        assert np.abs(got[i] - want).max() <= 1e-5 * top, i


@pytest.mark.parametrize("seqs", [1, 3, 17])
def test_every_sequence_and_block_is_reached(gpu, seqs):
    """The order of workgroups is a permutation: outputs of prompts of many lengths, whole ones at that."""
    lens = np.random.default_rng(seqs).integers(1, 420, seqs)
    rng, cache, table, q = make("int8", 4, 2, 64, 16, lens, lens, seqs)
    call, got = run(cache, table, lens, lens, q)
    check(cache, table, call, got, some=24)
    assert (got.view(np.uint32) != 0xa5a5a5a5).all()


def test_long_prompts(gpu):
    lens = np.array([2100, 1500])
    rng, cache, table, q = make("e4m3", 2, 4, 128, 16, lens, lens, 1)
    call, got = run(cache, table, lens, lens, q)
    check(cache, table, call, got, some=40)


@pytest.mark.parametrize("bs", [16, 6])
@pytest.mark.parametrize("split", [False, True])
def test_missing_pages_drop_out(gpu, bs, split):
    lens, new = np.array([400, 90, 20, 2500 if split else 30]), np.array([60, 90, 20, 5])
    rng, cache, table, q = make("e4m3", 2, 4, 128, bs, lens, new, bs)
    table[0, [0, 3, 7]], table[1, 1], table[2, :] = cache.blocks, 2 ** 64 - 1, 2 ** 63
    table[1, 0] = cache.blocks + 1  # queries that see no key: zeros
    call, got = run(cache, table, lens, new, q)
    assert call.size > 0 or not split
    check(cache, table, call, got)
    assert not got[150:170].any()


def test_rows_that_end_before_their_tokens(gpu):
    lens, new = np.array([100, 40]), np.array([30, 40])
    rng, cache, table, q = make("int8", 2, 2, 64, 16, lens, new, 2)
    short = table[:, :2].copy()
    call, got = run(cache, short, lens, new, q)
    check(cache, short, call, got)


@pytest.mark.parametrize("bs,D,n,m", [(16, 128, 100, 100), (32, 64, 200, 200), (5, 128, 70, 40), (16, 256, 100, 64), (16, 128, 3000, 40)])
def test_bytes_of_a_page_without_numbers_reach_what_sees_them_alone(gpu, bs, D, n, m):
    """A NaN that was written makes a page's V NaN bytes under a NaN scale: queries before it share its tile."""
    rng, cache, table, q = make("e4m3", 2, 2, D, bs, [n], [m], 1)
    first = (n - m // 2) // bs * bs  # of the last page that begins by the middle query
    page = int(table[0, first // bs])
    cache.scales[1, page, 1] = np.nan
    cache.bytes[1, page, 1] = 0xff
    cache.upload()
    results = [run(cache, table, [n], [m], q, kv_len=bound)[1] for bound in (n, max(n, 400), 5000)]
    before = first - (n - m)
    assert 0 < before < m
    cache.scales[1, page, 1], cache.bytes[1, page, 1] = 1.0, 0
    want = attention(cache, table[0], n, q[:before], visible=np.arange(n - m + 1, n - m + 1 + before))
    for got in results:
        assert np.isnan(got[before:, 2:]).all() and np.isfinite(got[:before]).all() and np.isfinite(got[:, :2]).all()
        assert np.abs(got[:before] - want).max() <= 1e-5 * biggest(cache, table[0], n)


@pytest.mark.parametrize("bs,D", [(16, 128), (64, 64), (5, 128), (16, 256)])
def test_what_lies_behind_a_sequence_is_not_seen(gpu, bs, D):
    lens, new = np.array([1, 37, 70, 530]), np.array([1, 30, 70, 100])
    rng, cache, table, q = make("e4m3", 2, 4, D, bs, lens, new, bs)
    used = {int(p) for r, n in enumerate(lens) for p in table[r, :-(-int(n) // bs)]}
    for page in set(range(cache.blocks)) - used:
        cache.scales[:, page] = np.nan
    for r, n in enumerate(lens):
        if n % bs:
            cache.bytes[:, int(table[r, n // bs]), :, n % bs:] = 0x7f
    cache.upload()
    call, got = run(cache, table, lens, new, q)
    check(cache, table, call, got)


def test_a_scale_that_is_nan_reaches_what_sees_it(gpu):
    """Queries before the page stay as they are, those behind it are NaN, whether K's scale or V's."""
    for which in range(2):
        rng, cache, table, q = make("e4m3", 2, 2, 128, 16, [100], [100], 1)
        cache.scales[which, int(table[0, 3]), 1] = np.nan
        cache.upload()
        call, got = run(cache, table, [100], [100], q)
        assert np.isnan(got[48:, 2:]).all() and np.isfinite(got[:48]).all() and np.isfinite(got[:, :2]).all()
        cache.scales[which, int(table[0, 3]), 1] = 1.0
        want = attention(cache, table[0], 100, q[:48], visible=np.arange(1, 49))
        assert np.abs(got[:48] - want).max() <= 1e-5 * biggest(cache, table[0], 100)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs", [16, 3])
def test_scales_of_any_origin(gpu, fmt, bs):
    lens, new = np.array([300, 64]), np.array([100, 64])
    rng, cache, table, q = make(fmt, 2, 4, 128, bs, lens, new, 4, scales=1.37)
    call, got = run(cache, table, lens, new, q)
    check(cache, table, call, got)
    cache.scales[1] *= np.exp2(rng.integers(-60, 41, cache.scales[1].shape)).astype(np.float32)
    cache.upload()
    call, got = run(cache, table, lens, new, q)
    check(cache, table, call, got)


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** 30])
def test_queries_and_keys_of_any_size(gpu, size):
    lens, new = np.array([200, 100]), np.array([60, 100])
    rng, cache, table, q = make("e4m3", 2, 4, 128, 16, lens, new, 6)
    _, want = run(cache, table, lens, new, q)
    cache.scales[0] /= np.float32(size)
    cache.upload()
    call, got = run(cache, table, lens, new, q * np.float32(size))
    check(cache, table, call, got)
    assert np.array_equal(got, want)  # powers of two throughout


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n,m", [(500, 500), (9000, 4)])
def test_a_dominant_key_and_thousands_of_small_ones(gpu, fmt, n, m):
    """One key 17 above the others (their weights 2^-25): their sum is not lost. A weight's parts end
    2^-40 below the largest weight; four FP32 roundings of a score of 24.5 (in powers of two) are 2^-20 each."""
    rng, cache, table, q = make(fmt, 1, 4, 128, 16, [n], [m], 8)
    cache.scales[:] = 2.0 ** -6
    cache.bytes[0], cache.bytes[1] = 0, 0x7e if fmt == "e4m3" else 127
    page = int(table[0, 0])
    cache.bytes[0, page, 0, 0] = 0x38 if fmt == "e4m3" else 1  # 1.0
    cache.bytes[1, page, 0, 0] = 0
    cache.upload()
    q[:] = 17.0 * np.sqrt(128) / 128 * 64
    call, got = run(cache, table, [n], [m], q)
    rows = np.arange(m)[-4:]
    want = attention(cache, table[0], n, q[rows], visible=n - m + rows + 1)
    assert want.min() > 0
    np.testing.assert_allclose(got[rows], want, rtol=4 * 2.0 ** -20, atol=n * 2.0 ** -40 * biggest(cache, table[0], n))


def test_values_whose_scales_grow_along_a_row(gpu):
    """Scales of V from 2^-30 up by a factor of two a page, over several windows of pages."""
    rng, cache, table, q = make("int8", 1, 4, 64, 1, [5000], [20], 3, spread=0.0)
    cache.scales[1, table[0].astype(np.int64)] *= np.exp2(np.arange(5000) // 100 - 30.0).astype(np.float32)[:, None]
    cache.upload()
    call, got = run(cache, table, [5000], [20], q)
    check(cache, table, call, got)


def test_offsets_in_any_order_and_rows_between(gpu):
    """Sequences' queries need not follow each other: what lies between is left as it was."""
    lens, new, offsets = np.array([50, 90, 20]), np.array([7, 90, 5]), np.array([120, 10, 2])
    rng, cache, table, q = make("e4m3", 2, 4, 64, 16, lens, [140, 0, 0], 5)
    call, got = run(cache, table, lens, new, q, offsets=offsets)
    check(cache, table, call, got)
    written = np.zeros(140, bool)
    for o, m in zip(offsets, new):
        written[o:o + m] = True
    assert np.all(got[~written].view(np.uint8) == 0xa5)


def test_lengths_past_the_bounds(gpu):
    """More queries than tokens or than the bounds say: the documented part, nothing outside."""
    lens, new = np.array([50, 30, 90]), np.array([60, 30, 20])
    rng, cache, table, q = make("e4m3", 2, 4, 64, 16, lens, [60, 30, 20], 5)
    call, got = run(cache, table, lens, new, q, most=60, kv_len=90)
    call.new = np.array([50, 30, 20])
    check(cache, table, call, got)
    assert np.all(got[50:60].view(np.uint8) == 0xa5)


def test_the_same_bits_again(gpu):
    lens, new = np.array([3000, 1500]), np.array([30, 40])
    rng, cache, table, q = make("e4m3", 4, 7, 128, 16, lens, new, 2)
    call, first = run(cache, table, lens, new, q)
    for _ in range(3):
        call.run()
        assert np.array_equal(call.result(), first)


@pytest.mark.parametrize("D,shift", [(84, 0), (100, 0), (512, 0), (20, 0), (128, 1), (64, 8)])
def test_generic_head_sizes_and_alignments(gpu, D, shift):
    rng = np.random.default_rng(D)
    lens, new = np.array([0, 1, 63, 70, 200]), np.array([0, 1, 63, 3, 10])
    blocks = int(sum(-(-n // 6) for n in lens))
    for fmt in ("e4m3", "int8"):
        cache = Cache(fmt, blocks, 2, 6, D, shift=shift)
        cache.fill(rng)
        table = random_table(rng, lens, 6, blocks)
        q = rng.standard_normal((int(new.sum()), 6, D)).astype(np.float32)
        call, got = run(cache, table, lens, new, q)
        check(cache, table, call, got)


def test_an_undersized_workspace_is_refused(gpu):
    rng, cache, table, q = make("e4m3", 2, 4, 128, 16, [5000], [3], 1)
    call = Prefill(cache, table, [5000], [3], q)
    with pytest.raises(capi.KvfluxError) as e:
        capi.call("kvflux_quant_prefill", *call.args[:-1], call.size - 1, None)
    assert e.value.status == capi.ERR_INVALID
