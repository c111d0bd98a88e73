"""The decode step from a projection's output: norm, rotation and paged write,
then attention with shared prefixes, through the C++ layer and as captured graphs.

* The grouping of rows is checked against every partition of small batches (CPU).
* The step is checked against the formulas in 64 bits, and against the append,
  write and attention calls that it replaces.
Tolerances: queries and keys as in test_gpu_norm_rope_write, attention 1e-5.
"""
from __future__ import annotations

import ctypes as C
import itertools

import numpy as np
import pytest

from gpu_util import DTYPES, decode, encode, read_cache
from kvflux_amd import capi, device
from test_gpu_norm_rope_write import EPS, HALF_LEAST, HALF_STEP, Call, reference
from test_gpu_shared_attention import TOL, Batch

SHORT = {"Float16": "f16", "BFloat16": "bf16", "Float32": "f32"}


# ------------------------------------------------------------------ grouping

def pages_of(s):
    return [s.physical_block_id(i) for i in range(s.num_tokens() // s.block_size())]


def common(rows):
    """Whole pages that all the rows start with."""
    n = 0
    for ids in zip(*rows):
        if len(set(ids)) > 1:
            break
        n += 1
    return n


def saved(rows, cuts):
    return sum((b - a - 1) * common(rows[a:b]) for a, b in zip(cuts, cuts[1:]))


@pytest.mark.parametrize("seed", range(12))
def test_grouping_saves_the_most(v2, seed):
    rng = np.random.default_rng(seed)
    bs = 4
    pool = v2.PhysicalBlockPool(400, bs)
    roots = []
    for i in range(2):
        s = v2.SequenceState(i, pool)
        s.append_tokens(int(rng.integers(0, 20)))
        roots.append(s)
    seqs = []
    for i in range(8):  # forks of forks, some grown past a page
        s = (roots + seqs)[int(rng.integers(0, 2 + len(seqs)))].fork_shared(10 + i)
        if s.num_tokens() % bs == 0:
            s.append_tokens(int(rng.integers(0, 3)) * bs)
        seqs.append(s)
    order = sorted(seqs, key=lambda s: [s.physical_block_id(i) for i in range(s.num_allocated_blocks())])
    for batch in (seqs, order):
        rows = [pages_of(s) for s in batch]
        most = max(saved(rows, (0, *c, len(rows))) for n in range(len(rows))
                   for c in itertools.combinations(range(1, len(rows)), n))
        starts, prefixes = v2.find_shared_prefixes(batch)
        if most == 0:
            assert starts == [] and prefixes == []
            continue
        assert starts[0] == 0 and starts[-1] == len(rows) and starts == sorted(set(starts))
        assert len(prefixes) == len(starts) - 1
        for a, b, p in zip(starts, starts[1:], prefixes):
            assert p % bs == 0 and (p == 0 or p == common(rows[a:b]) * bs)
        assert sum((b - a - 1) * p // bs for a, b, p in zip(starts, starts[1:], prefixes)) == most


def test_grouping_edges(v2):
    pool = v2.PhysicalBlockPool(40, 4)
    assert v2.find_shared_prefixes([]) == ([], [])
    s = v2.SequenceState(1, pool)
    assert v2.find_shared_prefixes([s]) == ([], [])
    s.append_tokens(7)
    f = s.fork_shared(2)
    assert v2.find_shared_prefixes([s]) == ([], [])
    assert v2.find_shared_prefixes([s, f]) == ([0, 2], [4])  # the partial page is not counted
    assert v2.find_shared_prefixes([s, s]) == ([0, 2], [4])  # the same sequence twice
    empty = v2.SequenceState(3, pool)
    other = v2.SequenceState(4, pool)
    other.append_tokens(9)
    assert v2.find_shared_prefixes([empty, other, s, f, empty]) == ([0, 2, 4, 5], [0, 4, 0])
    with pytest.raises(ValueError):
        v2.find_shared_prefixes([s, None])
    away = v2.SequenceState(5, v2.PhysicalBlockPool(4, 4))
    with pytest.raises(ValueError):
        v2.find_shared_prefixes([s, away])


# ------------------------------------------------------------------ the step

class Model:
    """Weights and one step's projections, packed [q heads | k heads | v heads] a token."""

    def __init__(self, rng, name, Hq, H, D, rotary, interleaved):
        self.name, self.Hq, self.H, self.D, self.rotary, self.interleaved = name, Hq, H, D, rotary, interleaved
        self.weights = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
        self.dev = [device.to_device(w) for w in self.weights]
        self.inv_freq = 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
        self.inv_dev = device.to_device(self.inv_freq)

    def form(self, v2):
        return v2.NormRope(self.dev[0].ptr, self.dev[1].ptr, EPS, self.inv_dev.ptr, self.rotary, self.interleaved)

    def project(self, v2, rng, tokens):
        x = rng.standard_normal((tokens, self.Hq + 2 * self.H, self.D)).astype(np.float32)
        bits = encode(x.ravel(), self.name)
        self.x = decode(bits, self.name).astype(np.float64).reshape(x.shape)
        self.bits = bits.reshape(x.shape)
        self.input = device.to_device(bits)
        item, row = bits.itemsize, (self.Hq + 2 * self.H) * self.D
        at = [self.input.ptr + h * self.D * item for h in (0, self.Hq, self.Hq + self.H)]
        return v2.ProjectedRows(*at, getattr(v2.DType, self.name), row, row, row)

    def check(self, query, keys, values, positions):
        """The step's queries [n][Hq][D], and the K and V bits [n][H][D] that it wrote."""
        kind = SHORT[self.name]
        p = np.asarray(positions, np.float64)
        want, tol = reference(self.x[:, :self.Hq], self.weights[0], p, self.inv_freq, self.rotary, self.interleaved)
        assert (np.abs(query - want) <= tol).all()
        want, tol = reference(self.x[:, self.Hq:self.Hq + self.H], self.weights[1], p, self.inv_freq, self.rotary,
                              self.interleaved)
        tol = tol * (1 + HALF_STEP[kind]) + np.abs(want) * HALF_STEP[kind] + HALF_LEAST[kind]
        got = decode(np.ascontiguousarray(keys).ravel(), self.name).reshape(want.shape)
        assert (np.abs(got - want) <= tol).all()
        assert np.array_equal(values, self.bits[:, self.Hq + self.H:])


def filled(v2, name, H, D, bs, pages, seed):
    pool = v2.PhysicalBlockPool(pages, bs)
    storage = v2.PagedKVStorage(pool, H, D, getattr(v2.DType, name))
    code = DTYPES[name][0]
    for i, base in enumerate((storage.key_base(), storage.value_base())):
        device.fill_random(base, pages * H * bs * D, code, 0, seed + i)
    device.synchronize()
    return pool, storage


def attention(storage, seqs, query, name, Hq):
    """Each row's attention over its pages, in 64 bits."""
    layout = storage.layout()
    H, D, bs = layout.num_kv_heads(), layout.head_size(), layout.block_size()
    k, v = (decode(x, name).reshape(-1, H, bs, D) for x in read_cache(storage, name))
    out = np.zeros(query.shape)
    G = Hq // H
    for r, s in enumerate(seqs):
        t = np.arange(s.num_tokens())
        page = np.array([s.physical_block_id(i) for i in range(s.num_allocated_blocks())])[t // bs]
        for h in range(H):
            kk, vv = (x[page, h, t % bs].astype(np.float64) for x in (k, v))
            w = query[r, h * G:(h + 1) * G].astype(np.float64) @ kk.T / np.sqrt(D)
            w = np.exp(w - w.max(-1, keepdims=True))
            out[r, h * G:(h + 1) * G] = (w @ vv) / w.sum(-1, keepdims=True)
    return out


STEPS = [  # type, query heads, kv heads, head size, page, shared tokens, forks
    ("BFloat16", 8, 2, 128, 16, 4800, 12), ("Float16", 4, 2, 64, 16, 9000, 12), ("Float32", 4, 2, 64, 8, 4720, 12),
    ("BFloat16", 4, 2, 128, 16, 70, 3), ("BFloat16", 4, 2, 80, 16, 100, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", STEPS, ids=lambda c: f"{c[0]}-{c[3]}-{c[5]}x{c[6]}")
def test_decode_step_projected(gpu, v2, case):
    name, Hq, H, D, bs, shared, forks = case
    rng = np.random.default_rng(31)
    pool, storage = filled(v2, name, H, D, bs, -(-shared // bs) + 8 * forks + 8, 5)
    base = v2.SequenceState(1, pool)
    base.append_tokens(shared + 3)
    seqs = [base] + [base.fork_shared(10 + i) for i in range(forks - 1)]
    lone = v2.SequenceState(2, pool)
    lone.append_tokens(5)
    seqs.append(lone)
    table = v2.DeviceBatchTable(storage, seqs, -(-shared // bs) + 8)
    model = Model(rng, name, Hq, H, D, D // 2, bool(rng.integers(0, 2)))
    n = len(seqs)
    query, out = device.DeviceBuffer(n * Hq * D * 4), device.DeviceBuffer(n * Hq * D * 4)
    plain = device.DeviceBuffer(n * Hq * D * 4)
    for step in range(bs + 2):  # copies the tail, crosses a page's end
        before = [s.num_tokens() for s in seqs]
        rows = model.project(v2, rng, n)
        got = v2.decode_step_projected(storage, table, rows, model.form(v2), query.ptr, out.ptr, Hq)
        assert [s.num_tokens() for s in seqs] == [b + 1 for b in before]
        assert [(g.physical_block, g.offset_in_block) for g in got] == \
               [(s.physical_block_id(b // bs), b % bs) for s, b in zip(seqs, before)]
        v2.paged_attention_batch(storage, table, query.ptr, plain.ptr, Hq)
        o, p = (x.download(np.float32).reshape(n, Hq, D) for x in (out, plain))
        assert np.abs(o - p).max() <= TOL
        if shared < 1000:  # sharing cannot pay for so little
            assert np.array_equal(o, p)
        if step in (0, bs + 1):
            q = query.download(np.float32).reshape(n, Hq, D)
            caches = [x.reshape(-1, H, bs, D) for x in read_cache(storage, name)]
            wrote = [np.stack([c[g.physical_block, :, g.offset_in_block] for g in got]) for c in caches]
            model.check(q, *wrote, before)
            assert np.abs(o - attention(storage, seqs, q, name, Hq)).max() <= TOL
            if shared >= 1000:
                assert not np.array_equal(o, p)
    # The forms over a list of sequences and over the table give the step's bits.
    for batch in (seqs, table):
        plain.fill(0xff)
        v2.paged_attention_batch_shared(storage, batch, query.ptr, plain.ptr, Hq)
        assert np.array_equal(plain.download(np.float32).reshape(o.shape), o)


@pytest.mark.gpu
def test_groups_follow_the_rows(gpu, v2):
    """A table's groups hold while rows grow; rows without sharers run as the ordinary decode."""
    rng = np.random.default_rng(32)
    pool, storage = filled(v2, "BFloat16", 2, 64, 16, 80, 7)
    seqs = []
    for i in range(3):
        s = v2.SequenceState(i, pool)
        s.append_tokens(30 + 20 * i)
        seqs.append(s)
    table = v2.DeviceBatchTable(storage, seqs, 12)
    q = device.to_device(rng.standard_normal((3, 4, 64)).astype(np.float32))
    a, b = device.DeviceBuffer(q.nbytes), device.DeviceBuffer(q.nbytes)
    for _ in range(3):
        v2.paged_attention_batch_shared(storage, table, q.ptr, a.ptr, 4)
        v2.paged_attention_batch(storage, table, q.ptr, b.ptr, 4)
        assert np.array_equal(a.download(np.float32), b.download(np.float32))
        for s in seqs:
            s.append_tokens(9)
            table.refresh()


@pytest.mark.gpu
def test_norm_rope_write_through_storage(gpu, v2):
    """A prompt's tokens over a slot mapping, then read back in order."""
    rng = np.random.default_rng(33)
    H, Hq, D, bs, n = 2, 6, 128, 16, 45
    pool, storage = filled(v2, "BFloat16", H, D, bs, 12, 9)
    s = v2.SequenceState(1, pool)
    s.append_tokens(n)
    slots = v2.build_slot_mapping([(s, t) for t in range(n)])
    for interleaved in (False, True):
        model = Model(rng, "BFloat16", Hq, H, D, D, interleaved)
        rows = model.project(v2, rng, n)
        query = device.DeviceBuffer(n * Hq * D * 4)
        v2.norm_rope_write(storage, rows, model.form(v2), Hq, list(range(n)), slots, query.ptr)
        k, v = device.DeviceBuffer(n * H * D * 2), device.DeviceBuffer(n * H * D * 2)
        v2.read_paged_kv(storage, s, k.ptr, v.ptr)
        model.check(query.download(np.float32).reshape(n, Hq, D),
                    *(x.download(np.uint16).reshape(n, H, D) for x in (k, v)), np.arange(n))


@pytest.mark.gpu
def test_refusals_change_nothing(gpu, v2):
    rng = np.random.default_rng(34)
    H, Hq, D, bs, n = 2, 4, 64, 16, 2
    pool, storage = filled(v2, "BFloat16", H, D, bs, 12, 9)
    seqs = []
    for i in range(n):
        s = v2.SequenceState(i, pool)
        s.append_tokens(3)
        seqs.append(s)
    table = v2.DeviceBatchTable(storage, seqs, 1)
    model = Model(rng, "BFloat16", Hq, H, D, D, False)
    rows, form = model.project(v2, rng, n), model.form(v2)
    at = model.input.ptr
    q, o = device.DeviceBuffer(n * Hq * D * 4), device.DeviceBuffer(n * Hq * D * 4)
    cache = [x.copy() for x in read_cache(storage, "BFloat16")]
    DT = v2.DType.BFloat16
    w, f = model.dev[0].ptr, model.inv_dev.ptr
    host = np.zeros(4096, np.uint16)

    def step(rows=rows, form=form, q=q.ptr, o=o.ptr, heads=Hq):
        v2.decode_step_projected(storage, table, rows, form, q, o, heads)

    def write(rows=rows, form=form, positions=(0, 1), slots=(0, 1), q=q.ptr, heads=Hq):
        v2.norm_rope_write(storage, rows, form, heads, list(positions), list(slots), q)

    for call in (step, write):
        for bad in (dict(heads=3), dict(heads=0), dict(q=0), dict(q=storage.key_base()), dict(q=at), dict(q=w),
                    dict(rows=v2.ProjectedRows(0, at, at, DT)), dict(rows=v2.ProjectedRows(at, host.ctypes.data, at, DT)),
                    dict(rows=v2.ProjectedRows(at, at, at, DT, Hq * D - 1)),
                    dict(rows=v2.ProjectedRows(at, at, at, DT, 0, 0, H * D - 1)),
                    dict(rows=v2.ProjectedRows(at, storage.key_base(), at, DT)),
                    dict(form=v2.NormRope(w, w, EPS, f, D - 1)), dict(form=v2.NormRope(w, w, EPS, f, D + 2)),
                    dict(form=v2.NormRope(w, w, EPS, 0, D)), dict(form=v2.NormRope(host.ctypes.data, w, EPS, f, D)),
                    dict(form=v2.NormRope(w, w, -1.0, f, D)), dict(form=v2.NormRope(w + 2, w, EPS, f, D)),
                    dict(rows=v2.ProjectedRows(at + 1, at, at, DT)), dict(q=q.ptr + 2)):
            with pytest.raises(ValueError):
                call(**bad)
            assert [s.num_tokens() for s in seqs] == [3, 3]
    with pytest.raises(ValueError):
        write(positions=(0,))
    with pytest.raises(IndexError):
        write(slots=(0, 12 * bs))
    with pytest.raises(ValueError):
        write(slots=(5, 5))
    write(positions=(), slots=())
    with pytest.raises(ValueError):
        step(o=q.ptr)
    for a, b in zip(cache, read_cache(storage, "BFloat16")):
        assert np.array_equal(a, b)
    assert [s.num_tokens() for s in seqs] == [3, 3]
    for s in seqs:
        s.append_tokens(13)
    table.refresh()
    with pytest.raises(v2.LogicError):
        step()  # a second page does not fit the table's rows
    assert [s.num_tokens() for s in seqs] == [16, 16]
    empty = v2.SequenceState(9, pool)
    with pytest.raises(ValueError):
        v2.paged_attention_batch_shared(storage, [seqs[0], empty], q.ptr, o.ptr, Hq)
    with pytest.raises(ValueError):
        v2.paged_attention_batch_shared(storage, seqs, host.ctypes.data, o.ptr, Hq)
    with pytest.raises(ValueError):
        v2.paged_attention_batch_shared(storage, seqs, q.ptr, o.ptr, 3)
    v2.paged_attention_batch_shared(storage, [], 0, 0, Hq)


# ------------------------------------------------------------------ graphs and streams

class Graph:
    """Calls captured from a stream, through the HIP runtime that the library links."""

    def __init__(self, stream, calls):
        self.hip, self.stream = C.CDLL(str(capi.LIB_PATH)), stream
        self.graph, self.exec = C.c_void_p(), C.c_void_p()
        self.do("hipStreamBeginCapture", C.c_void_p(stream.handle), 1)
        try:
            calls(stream.handle)
        finally:
            self.do("hipStreamEndCapture", C.c_void_p(stream.handle), C.byref(self.graph))
        self.do("hipGraphInstantiate", C.byref(self.exec), self.graph, None, None, C.c_size_t(0))

    def do(self, name, *args):
        status = getattr(self.hip, name)(*args)
        assert status == 0, (name, status)

    def replay(self):
        self.do("hipGraphLaunch", self.exec, C.c_void_p(self.stream.handle))
        self.stream.synchronize()

    def close(self):
        self.do("hipGraphExecDestroy", self.exec)
        self.do("hipGraphDestroy", self.graph)


def tail_call(rng, b):
    """A projection whose keys and values go to the last slots of the batch's rows, its queries to the batch's q."""
    c = Call(rng, b.dtype, heads=(b.Hq, b.H), D=b.D, bs=b.bs, tokens=len(b.lens))
    h = list(c.head())
    h[0], h[1], h[2] = b.dev["k"].ptr, b.dev["v"].ptr, b.pages
    d = b.dev
    return c, lambda stream: capi.call("kvflux_norm_rope_write_tail", *h, d["table"].ptr, b.table.shape[1],
                                       d["lens"].ptr, len(b.lens), d["q"].ptr, stream)


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [1 << 18, None], ids=["shared", "ordinary"])
def test_captured_step(gpu, bound):
    """Write and attention in one graph, replayed with other rows, lengths and groups between: each replay is the eager
    call's bits. Two graphs share a workspace, one after the other on a stream."""
    rng = np.random.default_rng(35)
    b = Batch(rng, [(1600, [30, 70, 9, 200]), (64, [5, 1])], heads=(8, 2)).upload(bound)
    c, write = tail_call(rng, b)
    attend = lambda stream: capi.call("kvflux_paged_attention_shared", *b.args(stream))
    write(0)
    attend(0)
    device.synchronize()
    s = device.Stream()

    def both(stream):
        write(stream)
        attend(stream)

    graphs = Graph(s, both), Graph(s, attend)
    lens, starts, prefixes = b.lens.copy(), b.starts.copy(), b.prefixes.copy()
    for turn in range(4):
        x = rng.standard_normal(c.x.shape).astype(np.float32)
        bits = (x.view(np.uint32) >> 16).astype(np.uint16)
        c.input.upload(bits)
        b.dev["lens"].upload(lens - np.uint64(min(turn, 1)))
        b.dev["starts"].upload(starts if turn != 2 else np.array([0, 2, 6], np.uint64))
        b.dev["prefixes"].upload(prefixes if turn != 2 else np.array([1600, 0], np.uint64))
        both(0)
        device.synchronize()
        eager = [x.download(np.uint16) for x in (b.dev["k"], b.dev["v"])], b.out.download(np.uint32)
        b.out.fill(0xff)
        b.ws.fill(0x11 * turn)
        graphs[0].replay()
        assert np.array_equal(b.out.download(np.uint32), eager[1])
        for x, want in zip((b.dev["k"], b.dev["v"]), eager[0]):
            assert np.array_equal(x.download(np.uint16), want)
        b.out.fill(0xff)
        graphs[1].replay()
        assert np.array_equal(b.out.download(np.uint32), eager[1])
    for g in graphs:
        g.close()


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Two batches at once, each with its own workspace, give what they give alone."""
    rng = np.random.default_rng(36)
    batches = [Batch(rng, [(2000, [30, 70, 9, 200])], heads=(8, 2)).upload(),
               Batch(rng, [(900, [300, 5]), (320, [8] * 9)], "f16", heads=(8, 4), D=64).upload()]
    alone = [b.run() for b in batches]
    streams = [device.Stream(), device.Stream()]
    for _ in range(10):
        for b in batches:
            b.out.fill(0xff)
        for _ in range(3):
            for b, s in zip(batches, streams):
                capi.call("kvflux_paged_attention_shared", *b.args(s.handle))
        for b, s, want in zip(batches, streams, alone):
            s.synchronize()
            assert np.array_equal(b.out.download(np.float32).reshape(want.shape), want)
