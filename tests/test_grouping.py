"""find_shared_prefixes on batches of many rows: runs of forks at several depths, against the grouping that saves the
most by trying every cut; and a batch whose rows all share, in little time."""
from __future__ import annotations

import time

import numpy as np
import pytest

from test_gpu_projected_step import common, pages_of


def most_saved(rows):
    """Pages that the best grouping of the rows does not read again: O(n^2)."""
    edge = [common([a, b]) for a, b in zip(rows, rows[1:])]
    best = [0] * (len(rows) + 1)
    for end in range(1, len(rows) + 1):
        best[end], least = best[end - 1], None
        for begin in range(end - 2, -1, -1):
            least = edge[begin] if least is None else min(least, edge[begin])
            best[end] = max(best[end], best[begin] + (end - begin - 1) * least)
    return best[-1]


@pytest.mark.parametrize("seed", range(30))
def test_runs_of_forks(v2, seed):
    rng = np.random.default_rng(seed)
    bs = 2
    pool = v2.PhysicalBlockPool(4000, bs)
    seqs, keep = [], []
    for _ in range(int(rng.integers(1, 8))):
        s = v2.SequenceState(len(keep), pool)
        s.append_tokens(bs * int(rng.integers(0, 6)))
        keep.append(s)
        for _ in range(int(rng.integers(1, 5))):  # a run at this depth, then deeper
            run = [s.fork_shared(1000 + len(keep) + i) for i in range(int(rng.integers(1, 7)))]
            keep += run
            seqs += run
            s = s.fork_shared(5000 + len(keep))
            s.append_tokens(bs * int(rng.integers(0, 4)))
            keep.append(s)
    if seed % 3 == 0:
        seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    rows = [pages_of(s) for s in seqs]
    starts, prefixes = v2.find_shared_prefixes(seqs)
    for a, b, p in zip(starts, starts[1:], prefixes):
        assert p == 0 or p == common(rows[a:b]) * bs
    assert sum((b - a - 1) * p // bs for a, b, p in zip(starts, starts[1:], prefixes)) == most_saved(rows)
    assert starts == [] or (starts[0] == 0 and starts[-1] == len(rows) and starts == sorted(set(starts)))


def test_many_rows_of_one_prefix(v2):
    """200000 rows behind one prefix: trying every cut takes 2e10 steps, many seconds."""
    pool = v2.PhysicalBlockPool(8, 4)
    base = v2.SequenceState(1, pool)
    base.append_tokens(8)
    rows = [base] * 200000
    start = time.perf_counter()
    assert v2.find_shared_prefixes(rows) == ([0, 200000], [8])
    assert time.perf_counter() - start < 2
