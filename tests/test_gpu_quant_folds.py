"""Calls on an 8-bit cache whose workgroups go through more tiles than they add at a time: a prompt's sums
folded into the output, or into the partials of split keys, a decode's into a second set, with scales,
missing pages and pages without numbers on either side of a fold. Within 1e-5 of the largest value that a query sees
(test_gpu_quant_attention.py says where that comes from)."""
from __future__ import annotations

import numpy as np
import pytest

from kvflux_amd import device
from quant_util import VALUES, Cache, attention
from test_gpu_projected_step import Graph
from test_gpu_quant_attention import run as decode
from test_gpu_quant_prefill import run as prefill

pytestmark = pytest.mark.gpu


def long_rows(fmt, D, bs, n, seqs, m, H=4, G=4, seed=0):
    """A cache of one row of n tokens, that row for each of `seqs` sequences, and their queries."""
    rng = np.random.default_rng([D, bs, seqs, seed])
    pages = -(-n // bs)
    cache = Cache(fmt, pages + 1, H, bs, D)
    if fmt == "e4m3":  # 2^-5 to 2.75, either sign
        cache.bytes = rng.integers(0x10, 0x44, cache.bytes.shape, np.uint8) | (rng.integers(0, 2, cache.bytes.shape, np.uint8) << 7)
    else:
        cache.bytes = rng.integers(-127, 128, cache.bytes.shape, np.int8).view(np.uint8)
    cache.scales = (rng.uniform(1, 2, cache.scales.shape) * (1.0 if fmt == "e4m3" else 2.0 ** -6)).astype(np.float32)
    cache.upload()
    table = rng.permutation(pages + 1)[:pages].astype(np.uint64)
    q = rng.standard_normal((seqs * m, H * G, D)).astype(np.float32)
    return rng, cache, table, q


def check(cache, table, n, m, q, got, rows):
    """Queries `rows` of all; NaN where a query sees one, in the kv heads that hold it."""
    H, G = cache.H, q.shape[1] // cache.H
    ids = np.where(table < cache.blocks, table, 0).astype(np.int64)
    sizes = np.abs(VALUES[cache.fmt][cache.bytes[1, ids]]).max(-1) * np.abs(cache.scales[1, ids][..., None].astype(np.float64))
    sizes = np.where((table < cache.blocks)[:, None, None], sizes, 0.0).transpose(1, 0, 2).reshape(H, -1)
    rows = np.asarray(rows)
    sees = n - m + rows % m + 1
    for i, see, want in zip(rows, sees, attention(cache, table, n, q[rows], visible=sees)):
        top = np.repeat(sizes[:, :see].max(1), G)[:, None]
        bad = np.isnan(want)
        assert np.array_equal(np.isnan(got[i]), bad), i
        assert (np.abs(got[i] - want)[~bad] <= np.broadcast_to(1e-5 * top, want.shape)[~bad]).all(), i


# Sequences and their queries such that every CU has a workgroup (sums folded into the output), or
# a half or a quarter of them has (into the partials), in each order of work.
SHAPES = [(128, 16, 64, 64), (128, 16, 32, 64), (128, 16, 128, 8), (128, 16, 32, 8), (64, 16, 128, 8), (64, 16, 32, 8),
          (256, 16, 128, 8), (256, 16, 24, 8), (128, 5, 64, 64), (128, 5, 32, 8), (64, 3, 128, 8), (128, 1, 32, 64),
          (96, 16, 64, 64), (48, 5, 128, 8), (192, 64, 128, 8), (128, 1000, 64, 64)]


@pytest.mark.parametrize("D,bs,seqs,m", SHAPES)
@pytest.mark.parametrize("fmt,scales", [("e4m3", "far"), ("int8", "rising")])
def test_folded_sums(gpu, fmt, D, bs, seqs, m, scales):
    n = 40000
    rng, cache, table, q = long_rows(fmt, D, bs, n, seqs, m)
    ids = table.astype(np.int64)
    if scales == "far":  # a few pages and heads of another size, the others within one power of two
        some = rng.choice(len(ids), min(12, len(ids)), replace=False)
        cache.scales[1, ids[some]] *= np.exp2(rng.integers(-60, 41, (len(some), 4))).astype(np.float32)
    else:  # 2^-60 to 1 along the row
        cache.scales[1, ids] *= np.exp2(np.linspace(-60, 0, len(ids)).round()).astype(np.float32)[:, None]
    cache.upload()
    _, got = prefill(cache, np.repeat(table[None], seqs, 0), [n] * seqs, [m] * seqs, q)
    assert np.isfinite(got).all()
    check(cache, table, n, m, q, got, [0, seqs * m // 2, seqs * m - 1])


@pytest.mark.parametrize("D,bs,seqs,m", [(128, 16, 64, 64), (128, 16, 32, 64), (64, 5, 128, 8), (256, 16, 128, 8)])
def test_missing_pages_and_pages_without_numbers(gpu, D, bs, seqs, m):
    n = 40000
    rng, cache, table, q = long_rows("e4m3", D, bs, n, seqs, m)
    table[rng.choice(len(table), len(table) // 3, replace=False)] = 2 ** 40
    live = np.flatnonzero(table < cache.blocks)
    cache.scales[0, int(table[live[1]]), 0] = np.nan                # seen by all, before the first fold
    cache.scales[1, int(table[live[len(live) // 2]]), 1] = np.nan   # in the middle
    cache.scales[1, int(table[live[-1]]), 2] = np.inf               # at the end
    cache.upload()
    _, got = prefill(cache, np.repeat(table[None], seqs, 0), [n] * seqs, [m] * seqs, q)
    nan = np.isnan(got).reshape(seqs * m, 4, 4 * D)
    assert nan[:, :2].all() and not nan[:, 3].any()
    sees = n - m + np.arange(m) + 1 > live[-1] * bs
    assert np.array_equal(nan[:, 2].all(-1), np.tile(sees, seqs)) and np.array_equal(nan[:, 2].any(-1), np.tile(sees, seqs))
    cache.scales[1, int(table[live[-1]]), 2] = np.nan  # what it counts as
    check(cache, table, n, m, q, got, [0, m - 1, seqs * m - 1])


def test_a_row_of_missing_pages_before_the_first_that_is_there(gpu):
    """Nothing to fold, then something."""
    D, bs, seqs, m, n = 128, 16, 64, 64, 40000
    rng, cache, table, q = long_rows("int8", D, bs, n, seqs, m)
    table[:2000] = 2 ** 63
    _, got = prefill(cache, np.repeat(table[None], seqs, 0), [n] * seqs, [m] * seqs, q)
    check(cache, table, n, m, q, got, [0, 5, seqs * m - 1])
    table[:] = 2 ** 63
    _, got = prefill(cache, np.repeat(table[None], seqs, 0), [n] * seqs, [m] * seqs, q)
    assert not got.any()


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 16), (256, 16), (128, 5), (96, 16), (64, 3), (240, 12)])
@pytest.mark.parametrize("fmt,scales", [("e4m3", "far"), ("int8", "rising")])
def test_a_decodes_folded_sums(gpu, fmt, scales, D, bs):
    """As many streams as workgroups, so that each goes through a whole row; half of the rows end in the middle."""
    n, rows, H = 40000, 256, 2
    rng, cache, table, q = long_rows(fmt, D, bs, n, rows, 1, H=H)
    ids = table.astype(np.int64)
    if scales == "far":
        some = rng.choice(len(ids), min(12, len(ids)), replace=False)
        cache.scales[1, ids[some]] *= np.exp2(rng.integers(-60, 41, (len(some), H))).astype(np.float32)
        table[rng.choice(len(table), len(table) // 5, replace=False)] = 2 ** 40
    else:
        cache.scales[1, ids] *= np.exp2(np.linspace(-60, 0, len(ids)).round()).astype(np.float32)[:, None]
    cache.scales[0, ids[-1], 1] = np.nan  # of the last page, in the second kv head
    cache.upload()
    lens = np.where(np.arange(rows) % 2, n - 17000, n)
    got = decode(cache, np.repeat(table[None], rows, 0), lens, q, kv_len=n)
    for r in (0, 101, 255):
        check(cache, table[:-(-int(lens[r]) // bs)], int(lens[r]), 1, q[r:r + 1], got[r:r + 1], [0])


def test_the_same_bits_again(gpu):
    rng, cache, table, q = long_rows("e4m3", 128, 16, 30000, 64, 64)
    args = (cache, np.repeat(table[None], 64, 0), [30000] * 64, [64] * 64, q)
    call, first = prefill(*args)
    for _ in range(3):
        call.run()
        assert np.array_equal(call.result(), first)


@pytest.mark.parametrize("D,seqs,m", [(128, 64, 64), (128, 32, 64), (64, 128, 8)])
def test_captured_and_replayed_at_other_lengths(gpu, D, seqs, m):
    """A captured call at a bound of 40000 tokens, lengths from none to that: every replay is the eager call's bits,
    whatever the output held before."""
    rng, cache, table, q = long_rows("e4m3", D, 16, 40000, seqs, m)
    tables = np.repeat(table[None], seqs, 0)
    call, _ = prefill(cache, tables, [40000] * seqs, [m] * seqs, q)
    stream = device.Stream()
    graph = Graph(stream, lambda h: call.run(h))
    for seed in range(3):
        r = np.random.default_rng(seed)
        lens = r.integers(0, 40001, seqs)
        lens[:4] = 40000, 9216, 9217, 0
        call.held[1].upload(lens.astype(np.uint64))
        call.held[2].upload(np.minimum(lens, m).astype(np.uint64))
        call.out.fill(0xa5)
        call.run()
        want = call.result().copy()
        call.out.fill(0xa5 if seed == 0 else 0xff)
        call.out.upload(np.full(256, 0xa5, np.uint8), call.q.size * 4)
        graph.replay()
        got = call.result()
        written = (np.arange(m)[None] < np.minimum(lens, m)[:, None]).reshape(-1)
        assert np.array_equal(got[written], want[written]), seed
    graph.close()
