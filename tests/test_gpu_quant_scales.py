"""An 8-bit cache whose scales are not the writes' own, or lie far apart.

Attention: within 1e-5 of the largest value that a query itself sees, of its kv head
(test_gpu_quant_attention.py says where that comes from). Writes: bytes and scales bit for
bit with the definition, a value over a scale that is no power of two by way of FP32.
"""
from __future__ import annotations

import numpy as np
import pytest

from kvflux_amd import device
from quant_util import VALUES, Cache, attention, hold, scale_of
from test_gpu_quant_attention import SHARES
from test_gpu_quant_attention import check as check_decode
from test_gpu_quant_attention import run as decode
from test_gpu_quant_prefill import Prefill
from test_gpu_quant_prefill import make as make_prompts
from test_gpu_quant_prefill import run as prefill
from test_gpu_quant_write import Rows, same, write

pytestmark = pytest.mark.gpu


def check_visible(cache, table, call, got, some=None):
    """Every query, or `some` of each sequence, within 1e-5 of the largest value that it sees."""
    G = got.shape[1] // cache.H
    for r, (n, m) in enumerate(zip(call.lens, call.new)):
        n, m, at = int(n), int(m), int(call.offsets[r])
        rows = np.arange(m) if some is None or m <= some else np.unique(np.r_[0, m - 1, np.random.default_rng(r).integers(0, m, some)])
        pages = table[r, :-(-n // cache.bs)].astype(np.int64)
        sizes = np.abs(VALUES[cache.fmt][cache.bytes[1, pages]]).max(-1) * cache.scales[1, pages][..., None].astype(np.float64)
        sizes = sizes.transpose(1, 0, 2).reshape(cache.H, -1)  # of every token's V
        want = attention(cache, table[r], n, call.q[at + rows], visible=n - m + rows + 1)
        for i, row in enumerate(rows):
            top = np.repeat(sizes[:, :n - m + row + 1].max(1), G)[:, None]
            err = np.abs(got[at + row] - want[i])
            assert (err <= 1e-5 * top).all(), (r, row, (err / top).max())


# ------------------------------------------------- what each query sees
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs,D,bound", [(16, 128, None), (16, 128, 900), (16, 128, 5000), (16, 64, 900), (16, 256, None), (5, 128, 900),
                                        (3, 64, None), (5, 128, 5000), (64, 128, 5000)])
def test_each_query_by_what_it_sees(gpu, fmt, bs, D, bound):
    """Scales of V from 2^-60 to 2^40 at random by page and head, ordinary queries."""
    lens, new = np.array([300, 64, 700]), np.array([100, 64, 300])
    rng, cache, table, q = make_prompts(fmt, 2, 4, D, bs, lens, new, [D, bs], scales=1.37)
    cache.scales[1] *= np.exp2(rng.integers(-60, 41, cache.scales[1].shape)).astype(np.float32)
    cache.upload()
    call, got = prefill(cache, table, lens, new, q, kv_len=bound)
    check_visible(cache, table, call, got)


@pytest.mark.parametrize("fmt,D,bs,n,m", [("e4m3", 128, 16, 9000, 40), ("int8", 64, 16, 40000, 70), ("int8", 128, 1, 5000, 300),
                                          ("e4m3", 128, 16, 33000, 130)])
def test_each_query_of_split_keys(gpu, fmt, D, bs, n, m):
    """A chunk behind a long prefix, its keys split over workgroups and windows, scales far apart in its last pages."""
    rng, cache, table, q = make_prompts(fmt, 2, 4, D, bs, [n], [m], [n, m])
    last = table[0, -(-m // bs) - 3:].astype(np.int64)
    cache.scales[1, last] *= np.exp2(rng.integers(0, 60, (len(last), 2))).astype(np.float32)
    cache.upload()
    call, got = prefill(cache, table, [n], [m], q)
    check_visible(cache, table, call, got, some=12)


def zero_pages(rng, cache, table, count):
    """V of `count` pages all zeros, as the writes leave them: with the least scale."""
    pages = rng.choice(table[table < cache.blocks].astype(np.int64), count, replace=False)
    cache.bytes[1, pages] = 0
    cache.scales[1, pages] = 2.0 ** -110
    cache.upload()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs,D,bound", [(16, 128, None), (16, 128, 5000), (16, 64, None), (16, 64, 2000), (16, 256, None), (5, 128, None),
                                        (5, 128, 5000), (3, 64, 2000), (128, 128, 5000), (200, 64, None)])
def test_pages_of_zeros_among_others(gpu, fmt, bs, D, bound):
    lens, new = np.array([300, 64, 700, 1600]), np.array([100, 64, 300, 40])
    rng, cache, table, q = make_prompts(fmt, 2, 4, D, bs, lens, new, [D, bs])
    zero_pages(rng, cache, table, 5)
    call, got = prefill(cache, table, lens, new, q, kv_len=bound)
    check_visible(cache, table, call, got)


def test_a_page_of_zeros_costs_no_pass_over_the_others(gpu):
    """512 tokens behind 16384 with two pages of zeros among them: the time without, and half of it more at most
    (4.5 times as long where every 2^16 between the scales had its pass)."""
    rng, cache, table, q = make_prompts("e4m3", 8, 4, 128, 16, [16896], [512], 1)
    call = Prefill(cache, table, [16896], [512], q)

    def time():
        best = np.inf
        for _ in range(5):
            a, b = device.Event(), device.Event()
            a.record()
            call.run()
            b.record()
            device.synchronize()
            best = min(best, a.elapsed_ms(b))
        return best

    time()
    without = time()
    zero_pages(rng, cache, table, 2)
    assert time() < 1.5 * without


# ------------------------------------------------- scales of any size
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bs", [16, 3])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scales_near_the_end_of_fp32(gpu, fmt, bs, D):
    """Scales of V of 2^-125 that are no powers of two: values of 2^-125 to 2^-116, outputs that FP32 holds in full."""
    lens, new = np.array([900, 64]), np.array([100, 64])
    rng, cache, table, q = make_prompts(fmt, 2, 4, D, bs, lens, new, 4)
    cache.scales[1] = (rng.uniform(1, 2, cache.scales[1].shape) * 2.0 ** -125).astype(np.float32)
    cache.upload()
    for bound in (None, 5000):
        call, got = prefill(cache, table, lens, new, q, kv_len=bound)
        check_visible(cache, table, call, got)
    rows = q[[0, -1]]
    for bound in (None, SHARES):
        check_decode(cache, table, lens, rows, decode(cache, table, lens, rows, kv_len=bound))


# ------------------------------------------------- writes behind scales of another origin
def half_page(fmt, scale, D=128, bs=16):
    """One page and head with 8 tokens of bytes at a scale of another origin, and its table."""
    rng = np.random.default_rng(3)
    cache = Cache(fmt, 1, 1, bs, D)
    cache.bytes[:] = hold(np.rint(rng.uniform(-100, 100, cache.bytes.shape)), fmt)
    cache.scales[:] = np.float32(scale)
    cache.upload()
    return rng, cache, np.zeros((1, 1), np.uint64)


def append(cache, table, x, name="f32"):
    """Tokens behind the first 8; the model's bytes and scales by the definition, divided in FP32."""
    n = x[0].shape[0]
    rows = Rows(x, name)
    held = write(cache, rows, table, [8 + n], [n], [0])
    device.synchronize()
    del held
    for i in range(2):
        before = cache.scales[i, 0, 0]
        s = np.float32(scale_of(np.abs(rows.x[i]).max(), cache.fmt))
        if abs(before) >= s:
            s = before
        else:
            cache.bytes[i, 0, 0, :8] = hold(VALUES[cache.fmt][cache.bytes[i, 0, 0, :8]] * (float(before) / float(s)), cache.fmt)
        cache.bytes[i, 0, 0, 8:8 + n] = hold((rows.x[i][:, 0].astype(np.float32) / s).astype(np.float64), cache.fmt)
        cache.scales[i, 0, 0] = s
    same(cache)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [128, 100])
def test_a_kept_scale_that_is_no_power_of_two(gpu, fmt, D):
    """Values half way between two bytes, whose quotient by the scale is exact where their product with
    its rounded reciprocal is a step beside it."""
    for scale in np.random.default_rng(1).uniform(1, 2, 40).astype(np.float32):
        rng, cache, table = half_page(fmt, scale, D)
        steps = np.arange(8 * D) % 63 + 0.5  # of at most half the top, so that the scale is large enough
        if fmt == "e4m3":
            steps = np.exp2(steps // 8) * (8 + steps % 8) / 8  # between two of the eight of a power of two
            steps = np.where(steps <= 224, steps, 1.0)
        x = (steps * float(scale)).astype(np.float32).reshape(8, 1, D)
        append(cache, table, [x, -x])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("scale", [-4.0, -0.37])
@pytest.mark.parametrize("size", [1.0, 1e4])
def test_a_negative_scale(gpu, fmt, scale, size):
    """It stays while its size is enough for the new values, and is replaced by a positive one where it is not."""
    rng, cache, table = half_page(fmt, scale)
    append(cache, table, [(rng.standard_normal((5, 1, 128)) * size).astype(np.float32) for _ in range(2)])
