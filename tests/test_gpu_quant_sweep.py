"""Seeded draws over the shapes of the calls on an 8-bit cache, each against 64 bits: prompts written
in one or two steps (bit for bit), single tokens behind them, what is read back, decode and prompt
attention at bounds of several sizes. KVFLUX_SWEEP_CASES and KVFLUX_SWEEP_SEED widen it.

Tolerance of the attentions: 1e-5 of the largest value a row sees where sum_i |q_i k_i| / sqrt(D) is at
most sqrt(D) (1.6 times what unit normals give); beyond it, in proportion. Every rounding on the way to
a score is relative to a partial sum of its terms or to a term (FP32 sums, 2^-23 of each q_i, the
scales' products, the difference to the reference), so at most c 2^-24 of that sum with a c that knows
the number of terms only: an error d of the scores moves an output by at most 2 d of the largest
value, and d grows with the sum as its bound does. The draws hold keys of up to 2^6 times a unit normal."""
from __future__ import annotations

import os

import numpy as np
import pytest

from quant_util import VALUES, Cache, attention, random_table
from test_gpu_quant_attention import biggest
from test_gpu_quant_attention import run as decode
from test_gpu_quant_prefill import run as prompts
from test_gpu_quant_write import Rows, gather, same, write, write_tail

pytestmark = pytest.mark.gpu

CASES = int(os.environ.get("KVFLUX_SWEEP_CASES", "30"))
SEED = int(os.environ.get("KVFLUX_SWEEP_SEED", "5"))


def tolerance(cache, table, n, q):
    """Of queries [rows][Hq][D] on the first n tokens of a table row."""
    G = q.shape[1] // cache.H
    ids = [int(p) for p in table[:-(-n // cache.bs)] if p < cache.blocks]
    if not ids:
        return 1e-5
    k = np.abs(VALUES[cache.fmt][cache.bytes[0, ids]]) * cache.scales[0, ids][..., None, None].astype(np.float64)
    k = np.nan_to_num(k).transpose(1, 0, 2, 3).reshape(cache.H, -1, cache.D)
    terms = max(float((np.abs(q[:, h * G:(h + 1) * G].reshape(-1, cache.D)).astype(np.float64) @ k[h].T).max()) for h in range(cache.H))
    return 1e-5 * max(1.0, terms / cache.D) * biggest(cache, table, n)  # terms / sqrt(D) over sqrt(D)


@pytest.mark.parametrize("case", range(CASES))
def test_draws(gpu, case):
    rng = np.random.default_rng([SEED, case])
    pick = lambda *x: x[rng.integers(len(x))]  # noqa: E731
    fmt, name = pick("e4m3", "int8"), pick("bf16", "f16", "f32")
    D = int(pick(64, 128, 128, 256, 16 * rng.integers(1, 17), rng.integers(1, 300)))
    bs, H, G = int(pick(16, 16, 32, 64, 8, 1, 5, 24, rng.integers(1, 70))), int(pick(1, 2, 3, 4, 8)), int(pick(1, 2, 4, 7, 8, 12, 17))
    rows = int(pick(1, 2, 5, 16, 40))
    budget = 3_000_000 // (H * D)  # tokens of the cache
    hi = max(2, min(budget // rows, int(pick(40, 200, 700, 2600, 9000))))
    lens = rng.integers(0, hi + 1, rows)
    lens[rng.integers(rows)] = hi
    blocks = int((-(-lens // bs)).sum()) + int(rng.integers(1, 4))
    cache = Cache(fmt, blocks, H, bs, D)
    table = random_table(rng, lens, bs, blocks, width=int(-(-hi // bs) + rng.integers(0, 3)))
    # The tokens in up to two steps, the last one of some rows by the tail form.
    first = np.minimum(lens, rng.integers(0, hi + 1, rows))
    tail = (lens > first) & (rng.random(rows) < 0.5)
    held, had = [], np.zeros(rows, np.int64)
    for upto in (first, lens - tail):
        new = upto - had
        if new.sum() == 0:
            continue
        size = np.exp2(rng.uniform(-6, 6))
        data = Rows([rng.standard_normal((int(new.sum()), H, D)) * size for _ in range(2)], name, pad=int(pick(0, 8, 3)))
        offsets = np.cumsum(new) - new
        held.append((data, write(cache, data, table, upto, new, offsets)))
        for i in range(2):
            cache.write(i, table, upto, new, offsets, data.x[i])
        had = upto.copy()
    if tail.any():
        data = Rows([rng.standard_normal((rows, H, D)) for _ in range(2)], name)
        at = np.where(tail, lens, 0)  # rows of zero tokens: nothing
        held.append((data, write_tail(cache, data, table, at)))
        for i in range(2):
            cache.write(i, table, at, tail.astype(np.int64), np.arange(rows), data.x[i])
    same(cache)
    if lens.sum():
        got = gather(cache, table, lens, "f32")
        values = cache.values()
        for i in range(2):
            want = [values[i, table[r, :-(-n // bs)].astype(np.int64)].transpose(0, 2, 1, 3).reshape(-1, H, D)[:n] for r, n in enumerate(lens)]
            assert np.array_equal(got[i].view(np.float32), np.concatenate(want).astype(np.float32))
    cache.bytes, cache.scales = cache.download()  # behind the tokens whatever is there
    q = rng.standard_normal((rows, H * G, D)).astype(np.float32) * np.float32(pick(0.3, 1.0, 2.0))
    if rng.random() < 0.3 and table[0, 0] < blocks:
        table[0, 0] = blocks  # a missing page
    bound = int(max(hi, pick(hi, 600, 1024, 1500, 2500, 6000)))
    got = decode(cache, table, lens, q, kv_len=bound)
    for r in rng.permutation(rows)[:6]:
        n = int(lens[r])
        want = attention(cache, table[r], n, q[r:r + 1])[0]
        assert np.abs(got[r] - want).max() <= tolerance(cache, table[r], n, q[r:r + 1]), (r, n)
    new = np.minimum(lens, rng.integers(0, int(pick(3, 40, 300)) + 1, rows))
    if new.sum() == 0:
        return
    q = rng.standard_normal((int(new.sum()), H * G, D)).astype(np.float32)
    call, got = prompts(cache, table, lens, new, q, most=int(max(new.max(), min(bound, pick(new.max(), 200, 1000)))), kv_len=bound)
    for r in rng.permutation(rows)[:4]:
        n, m, o = int(lens[r]), int(new[r]), int(call.offsets[r])
        if m:
            i = np.unique(np.r_[0, m - 1, rng.integers(0, m, 4)])
            want = attention(cache, table[r], n, q[o + i], visible=n - m + i + 1)
            assert np.abs(got[o + i] - want).max() <= tolerance(cache, table[r], n, q[o + i]), (r, n, m)
