"""kvflux_paged_attention_shared against the softmax in 64 bits.

Tolerance: the decode attention's contract, 1e-5 for unit-scale data (scores of
standard deviation 1, values of 1). With u = 2^-24: a score is a sum of D
products of FP32-exact parts (FP16: a query value and a weight are off by 2u) in
FP32 chains, off by at most 3 D u |q||k| in the worst case and about 2 sqrt(D) u
of its size in practice, under 3e-7 here; a
weight is off by its score's error and exp2's 2u; an output is a weighted mean
of values below 5, so off by under 5 * (3e-7 + 4u + merge 4u) = 4e-6.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device

CODE = {"f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16, "f32": capi.DTYPE_F32}
TOL = 1e-5
NONE = 2 ** 64 - 1
# Small batches run as an ordinary decode by their bounds; these bounds, as large
# as a caller may give, choose the shared kernel.
BOUND = 1 << 18


def to_bits(x, name):
    x = np.ascontiguousarray(x, np.float32)
    if name == "f32":
        return x.view(np.uint32).copy()
    if name == "f16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bits(b, name):
    if name == "f32":
        return b.view(np.float32).astype(np.float64)
    if name == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Batch:
    """Caches, tables and groups of a batch. `groups`: (prefix tokens, own tokens of each row)."""

    def __init__(self, rng, groups, dtype="bf16", heads=(8, 2), D=128, bs=16, before=(), after=(), scale=1.0):
        self.dtype, self.D, self.bs = dtype, D, bs
        self.Hq, self.H = heads
        rows = [(None, n) for n in before]
        starts, prefixes = [len(before)], []
        for prefix, own in groups:
            rows += [(len(prefixes), n) for n in own]
            prefixes.append(prefix)
            starts.append(len(rows))
        rows += [(None, n) for n in after]
        self.starts, self.prefixes = np.array(starts, np.uint64), np.array(prefixes or [0], np.uint64)
        self.groups = len(prefixes)
        self.lens = np.array([(prefixes[g] if g is not None else 0) + n for g, n in rows], np.uint64)
        counts = [-(-int(n) // bs) for n in self.lens]
        shared = [p // bs for p in prefixes]
        width = max(counts + [1])
        total = sum(shared) + sum(c - (shared[g] if g is not None else 0) for (g, _), c in zip(rows, counts))
        self.pages = total + 3
        order = rng.permutation(self.pages)
        at = 0
        common = []
        for s in shared:
            common.append(order[at:at + s])
            at += s
        self.table = np.full((len(rows), width), NONE, np.uint64)
        for r, ((g, _), c) in enumerate(zip(rows, counts)):
            s = shared[g] if g is not None else 0
            if s:
                self.table[r, :s] = common[g][:s]
            self.table[r, s:c] = order[at:at + max(0, c - s)]
            at += max(0, c - s)
        # A prefix that ends inside a page: the rows' pages there hold the same tokens.
        shape = (self.pages, self.H, bs, D)
        self.k = to_bits(rng.standard_normal(shape) * scale, dtype)
        self.v = to_bits(rng.standard_normal(shape), dtype)
        for g, p in enumerate(prefixes):
            if p % bs:
                mine = [r for r, (x, _) in enumerate(rows) if x == g]
                first = int(self.table[mine[0], p // bs])
                for r in mine[1:]:
                    page = int(self.table[r, p // bs])
                    self.k[page, :, :p % bs], self.v[page, :, :p % bs] = self.k[first, :, :p % bs], self.v[first, :, :p % bs]
        self.q = rng.standard_normal((len(rows), self.Hq, D)).astype(np.float32)

    def expected(self):
        k, v = from_bits(self.k, self.dtype), from_bits(self.v, self.dtype)
        out = np.zeros(self.q.shape)
        G = self.Hq // self.H
        for r, n in enumerate(self.lens):
            n = min(int(n), self.table.shape[1] * self.bs)
            tokens = np.arange(n)
            page = self.table[r, tokens // self.bs]
            tokens = tokens[page < self.pages]
            if not len(tokens):
                continue
            page = page[page < self.pages].astype(np.int64)
            for h in range(self.H):
                kk, vv = k[page, h, tokens % self.bs], v[page, h, tokens % self.bs]
                s = self.q[r, h * G:(h + 1) * G].astype(np.float64) @ kk.T / np.sqrt(self.D)
                w = np.exp(s - s.max(-1, keepdims=True))
                out[r, h * G:(h + 1) * G] = (w @ vv) / w.sum(-1, keepdims=True)
        return out

    def upload(self, bound=BOUND):
        self.dev = {n: device.to_device(getattr(self, n)) for n in ("k", "v", "table", "lens", "starts", "prefixes", "q")}
        self.out = device.to_device(np.full(self.q.shape, 999.0, np.float32))
        size = C.c_size_t()
        self.max_len = bound or int(self.lens.max())
        self.max_prefix = bound or int(self.prefixes.max())
        capi.call("kvflux_paged_attention_shared_workspace_size", len(self.lens), self.max_len, self.H, self.Hq, self.bs,
                  self.D, CODE[self.dtype], self.groups, C.byref(size))
        self.ws = device.DeviceBuffer(size.value)
        self.ws.fill(0xff)  # NaNs: no partial may be read that was not written
        return self

    def args(self, stream=0):
        d = self.dev
        return (d["k"].ptr, d["v"].ptr, self.pages, self.H, self.bs, self.D, CODE[self.dtype], d["table"].ptr,
                self.table.shape[1], d["lens"].ptr, self.max_len, len(self.lens), self.Hq, d["starts"].ptr,
                d["prefixes"].ptr, self.groups, self.max_prefix, d["q"].ptr, self.out.ptr, self.ws.ptr,
                self.ws.nbytes, stream)

    def run(self, stream=0):
        capi.call("kvflux_paged_attention_shared", *self.args(stream))
        device.synchronize(stream)
        return self.out.download(np.float32).reshape(self.q.shape)

    def check(self, tol=TOL, bound=BOUND):
        got, want = self.upload(bound).run(), self.expected()
        assert np.isfinite(got).all()
        assert np.abs(got - want).max() <= tol, np.abs(got - want).max()
        return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f16", 64), ("f16", 128),
                                     ("f16", 256), ("f32", 64), ("f32", 128)])
def test_types_and_head_sizes(gpu, dtype, D):
    rng = np.random.default_rng(1)
    Batch(rng, [(96, [1, 17, 40]), (300, [5, 200])], dtype, D=D).check()


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (28, 4), (12, 1), (40, 2), (130, 1), (300, 1), (18, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_head_layouts(gpu, heads, dtype):
    """Groups of 1 to 300 heads: columns of a row in one block, several, several streams."""
    rng = np.random.default_rng(2)
    Batch(rng, [(64, [3, 30, 70]), (200, [9, 1])], dtype, heads=heads, D=64).check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 3, 5, 9, 17, 33, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_columns_of_a_prefix(gpu, rows, D):
    """1 to 18 blocks of 16 columns: every layout of the wavefronts, and a second stream of columns."""
    rng = np.random.default_rng(3)
    Batch(rng, [(272, list(rng.integers(1, 40, rows)))], "bf16", heads=(4, 1), D=D).check()


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [1, 2, 5, 8, 16, 48, 64, 256, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(gpu, bs, D):
    """Pages of any size, whole ones shared."""
    rng = np.random.default_rng(4)
    for dtype in ("bf16", "f32"):
        Batch(rng, [(3 * bs, [1, 20, 130]), (bs * (1 + 200 // bs), [50, 3])], dtype, D=D, bs=bs).check()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 700])
def test_prefix_lengths(gpu, prefix):
    """Prefixes that end anywhere in a tile and in a page (the pages there hold the same tokens)."""
    rng = np.random.default_rng(5)
    for D in (64, 128):
        Batch(rng, [(prefix, [1, 2, 100])], "bf16", D=D).check()


@pytest.mark.gpu
@pytest.mark.parametrize("own", [0, 1, 2, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 256, 300])
def test_own_lengths(gpu, own):
    """Rows whose own part is empty, one token, and around the tiles' sizes."""
    rng = np.random.default_rng(6)
    for dtype in ("bf16", "f32"):
        Batch(rng, [(160, [own, 5, own])], dtype).check()


@pytest.mark.gpu
def test_rows_without_a_group(gpu):
    rng = np.random.default_rng(7)
    Batch(rng, [(128, [4, 9]), (32, [1, 70, 2])], before=[100, 0, 1], after=[5, 260]).check()


@pytest.mark.gpu
def test_groups_of_one_and_no_prefix(gpu):
    rng = np.random.default_rng(8)
    Batch(rng, [(128, [4]), (0, [10, 20]), (64, []), (48, [1, 1]), (200, [7])]).check()


@pytest.mark.gpu
def test_empty_batch_rows(gpu):
    rng = np.random.default_rng(9)
    b = Batch(rng, [(64, [3, 4, 5])], before=[0], after=[0, 0])
    b.check()
    b.lens[:] = 0  # a batch of padding
    got = b.upload().run()
    assert (got == 0).all()


@pytest.mark.gpu
def test_rows_shorter_than_the_prefix(gpu):
    """Such a row reads its own table row: other pages, no tokens, or one."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [(160, [30, 30, 30, 30, 30])])
    b.lens[1], b.lens[2], b.lens[4] = 50, 0, 1
    b.table[1, :4] = b.table[3, 10:12].tolist() * 2  # pages that the group does not share
    b.check()
    b.lens[3] = 160  # exactly the prefix
    b.check()
    b.lens[0] = 159  # the row whose table the prefix is read through
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_missing_pages(gpu, dtype):
    """Page ids past the pool drop out, in the prefix and in a row's own part, up to whole tiles."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(640, [40, 300, 20])], dtype)
    b.table[:, 3] = b.pages
    b.table[:, 8:30] = NONE
    b.table[1, 45:50] = b.pages + 7
    b.check()
    b.table[:, :] = NONE
    assert (b.upload().run() == 0).all()


@pytest.mark.gpu
def test_short_table(gpu):
    """Tokens past the table's width have no page."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [(64, [200, 100])])
    b.table = np.ascontiguousarray(b.table[:, :9])
    b.check()


@pytest.mark.gpu
def test_unwritten_slots_do_not_matter(gpu):
    """NaN and infinity in slots past every row's end."""
    rng = np.random.default_rng(13)
    for dtype in ("bf16", "f16", "f32"):
        b = Batch(rng, [(160, [5, 33, 100])], dtype)
        nan = to_bits(np.array([np.nan]), dtype)[0]
        inf = to_bits(np.array([np.inf]), dtype)[0]
        for r, n in enumerate(b.lens):
            page, off = int(b.table[r, int(n) // b.bs]) if int(n) % b.bs else None, int(n) % b.bs
            if page is not None:
                b.k[page, :, off:], b.v[page, :, off:] = nan, nan
                b.v[page, :, off:, ::2] = inf
        free = sorted(set(range(b.pages)) - set(b.table[b.table < b.pages].astype(int).tolist()))
        b.k[free], b.v[free] = nan, nan
        b.check()


@pytest.mark.gpu
def test_nan_stays_with_its_rows(gpu):
    """A NaN in a row's own values, query or length-masked keys reaches that row alone; one in the prefix, its group."""
    rng = np.random.default_rng(14)
    b = Batch(rng, [(160, [5, 33, 100]), (64, [3, 3])])
    want = b.expected()
    b.v[int(b.table[1, 11]), 0, 0, 3] = 0x7fc0  # token 176 of row 1, kv head 0, dim 3
    b.q[2, 7, 0] = np.nan
    b.k[int(b.table[3, 2]), 1, 5] = 0x7fc0      # prefix of the second group, kv head 1
    got = b.upload().run()
    bad = np.zeros(got.shape, bool)
    bad[1, :4, 3] = True
    bad[2, 7] = True
    bad[3:, 4:] = True
    assert np.isnan(got[bad]).all()
    assert np.abs(got - want)[~bad].max() <= TOL


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_scores(gpu, dtype):
    """Scores of standard deviation 12: one key dominates, and maxima move from tile to tile. Each score, of size up
    to 60, is off by about 60 * sqrt(D) u = 4e-5 at the most; so are the weights, and the outputs by 5 times that at
    the worst, where two keys weigh the same."""
    rng = np.random.default_rng(15)
    Batch(rng, [(500, [60, 300, 9]), (64, [20, 20])], dtype, scale=12.0).check(tol=2e-4)


@pytest.mark.gpu
def test_small_weights_are_kept(gpu):
    """One key 16 above thousands of others: their 2^-23 each, 4.6e-4 together, are in the sums."""
    rng = np.random.default_rng(16)
    for dtype in ("bf16", "f16", "f32"):
        b = Batch(rng, [(4096, [1, 2])], dtype, heads=(2, 1), D=64)
        b.k[...] = 0
        b.q[...] = 0
        b.q[:, :, 0] = 16 * np.sqrt(64)
        b.k[int(b.table[0, 0]), :, 0, 0] = to_bits(np.array([1.0]), dtype)[0]
        b.check()


@pytest.mark.gpu
def test_many_rows_and_groups(gpu):
    rng = np.random.default_rng(17)
    groups = [(int(rng.integers(0, 120)) // 16 * 16, list(rng.integers(0, 60, rng.integers(1, 9)))) for _ in range(150)]
    Batch(rng, groups, "bf16", heads=(4, 2), D=64).check()


@pytest.mark.gpu
@pytest.mark.parametrize("more", [0, 1], ids=["most rows", "a row more"])
def test_most_rows_and_groups(gpu, more):
    """2048 rows in 512 groups, the most that one plan holds; a row more runs as the ordinary decode."""
    rng = np.random.default_rng(28)
    b = Batch(rng, [(16 * int(rng.integers(0, 4)), list(rng.integers(0, 30, 4))) for _ in range(512)], "bf16",
              heads=(2, 1), D=64, after=[9] * more)
    got = b.check()
    assert np.array_equal(got, ordinary(b)) == bool(more)


@pytest.mark.gpu
def test_long_prefix(gpu):
    """A prefix over many tiles, so its streams are split over workgroups, beside short and long own parts."""
    rng = np.random.default_rng(18)
    for dtype, D in (("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256)):
        Batch(rng, [(6000, [1, 700, 33, 2, 2, 90]), (2500, [40, 3])], dtype, heads=(8, 2), D=D).check()


@pytest.mark.gpu
def test_same_bits_every_time(gpu):
    rng = np.random.default_rng(19)
    b = Batch(rng, [(2000, [100, 300, 5]), (500, [10, 700])]).upload()
    first = b.run()
    for fill in (0x00, 0xff, 0x3f):
        b.ws.fill(fill)
        assert np.array_equal(b.run(), first)


@pytest.mark.gpu
def test_near_the_ordinary_decode(gpu):
    """The result is that of kvflux_paged_attention on the same batch."""
    rng = np.random.default_rng(20)
    b = Batch(rng, [(1000, [100, 3, 5, 800]), (64, [10, 70])], before=[300], heads=(32, 8)).upload()
    shared, plain = b.run(), ordinary(b)
    assert np.abs(plain - shared).max() <= TOL


def ordinary(b):
    """kvflux_paged_attention's output for the batch."""
    size = C.c_size_t()
    capi.call("kvflux_paged_attention_workspace_size", len(b.lens), b.max_len, b.H, b.Hq, b.bs, b.D, C.byref(size))
    ws = device.DeviceBuffer(size.value)
    a = b.args()
    b.out.fill(0xff)
    capi.call("kvflux_paged_attention", *a[:13], a[17], a[18], ws.ptr, size.value, None)
    device.synchronize()
    return b.out.download(np.float32).reshape(b.q.shape)


@pytest.mark.gpu
def test_calls_that_sharing_cannot_pay_for(gpu):
    """Short prefixes and batches without sharers run as the ordinary decode, bit for bit; long prefixes do not."""
    rng = np.random.default_rng(25)
    for groups in ([(96, [3, 40, 7])], [(700, [5]), (40, [9]), (900, [1])]):
        b = Batch(rng, groups)
        got = b.check(bound=None)
        assert np.array_equal(got, ordinary(b))
    b = Batch(rng, [(6000, [5, 9, 40, 2, 3, 8, 1, 1, 7, 200])], heads=(8, 4))
    got = b.check(bound=None)
    plain = ordinary(b)
    assert not np.array_equal(got, plain) and np.abs(got - plain).max() <= TOL


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [dict(D=80), dict(D=96, heads=(4, 4)), dict(D=4, heads=(2, 1), bs=4),
                                   dict(D=256, dtype="f32")])
def test_shapes_left_to_the_ordinary_decode(gpu, shape):
    rng = np.random.default_rng(21)
    Batch(rng, [(96, [3, 40]), (32, [9, 9, 9])], **shape).check()


@pytest.mark.gpu
def test_no_groups(gpu):
    rng = np.random.default_rng(22)
    Batch(rng, [], before=[100, 0, 700]).check()


@pytest.mark.gpu
def test_odd_group_arrays_stay_in_bounds(gpu):
    """Starts that descend or pass the batch, prefixes past every row: other results are allowed, other memory is not.
    The rows that no group holds keep theirs."""
    rng = np.random.default_rng(23)
    b = Batch(rng, [(64, [3, 4]), (64, [5, 6]), (64, [7, 8])], before=[30])
    want = b.expected()
    for starts, prefixes in (([5, 2, 9, 1], [64, 64, 64]), ([1, 1, 1, 1], [64, 64, 64]),
                             ([7, 100, 2 ** 63, NONE], [64, 64, 64]), ([1, 3, 5, 7], [NONE, 2 ** 40, 100000])):
        b.starts, b.prefixes = np.array(starts, np.uint64), np.array(prefixes, np.uint64)
        got = b.upload().run()
        assert np.isfinite(got).all()
        assert np.abs(got[0] - want[0]).max() <= TOL
        if prefixes[0] == NONE:  # every row is shorter: all on their own
            assert np.abs(got - want).max() <= TOL


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pages_past_32_bits(gpu, dtype):
    """The batch's pages are the last of a cache of over 2^32 elements a tensor; whole pages and small ones."""
    rng = np.random.default_rng(26)
    for bs in (16, 8):
        b = Batch(rng, [(200 // bs * bs, [30, 5, 70])], dtype, heads=(16, 8), bs=bs)
        want, used, page = b.expected(), b.pages, b.k[0].nbytes
        b.pages = (1 << 32) // b.k[0].size + used + 1
        first = b.pages - used
        b.table[b.table != NONE] += np.uint64(first)
        k, v, b.k, b.v = b.k, b.v, b.k[:1], b.v[:1]
        b.upload()
        for name, part in (("k", k), ("v", v)):
            b.dev[name] = device.DeviceBuffer(b.pages * page)
            b.dev[name].upload(part, first * page)
        assert np.abs(b.run() - want).max() <= TOL


@pytest.mark.gpu
def test_queries_and_outputs_at_any_float(gpu):
    """Query and output arrays aligned to 4 bytes, and nothing written past the output."""
    rng = np.random.default_rng(27)
    for dtype, D in (("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 256)):
        b = Batch(rng, [(300, [10, 20, 30])], dtype, D=D).upload()
        q, out = device.DeviceBuffer(b.q.nbytes + 16), device.to_device(np.full(b.q.size + 2, 999.0, np.float32))
        q.upload(b.q, 4)
        a = list(b.args())
        a[17], a[18] = q.ptr + 4, out.ptr + 4
        capi.call("kvflux_paged_attention_shared", *a)
        got = out.download(np.float32)
        assert got[0] == 999.0 and got[-1] == 999.0
        assert np.abs(got[1:-1].reshape(b.q.shape) - b.expected()).max() <= TOL


@pytest.mark.gpu
def test_on_another_stream(gpu):
    rng = np.random.default_rng(24)
    b = Batch(rng, [(300, [10, 20, 30])]).upload()
    s = device.Stream()
    assert np.abs(b.run(s.handle) - b.expected()).max() <= TOL


def test_refusals():
    """Checked on the host before anything is launched (no GPU needed)."""
    ok = dict(k=4096, v=4096, blocks=8, H=2, bs=16, D=128, dtype=1, table=4096, width=4, lens=4096, kv=BOUND, rows=3, Hq=4,
              starts=4096, prefixes=4096, groups=1, most=BOUND, q=4096, out=4096, ws=4096, size=1 << 40)

    def status(**change):
        return capi.lib().kvflux_paged_attention_shared(*({**ok, **change}[x] for x in ok), None)

    assert status(rows=0) == capi.OK
    for name in ("k", "v", "table", "lens", "starts", "prefixes", "q", "out", "ws"):
        assert status(**{name: None}) == capi.ERR_INVALID, name
    for name in ("blocks", "H", "bs", "D", "Hq", "width"):
        assert status(**{name: 0}) == capi.ERR_INVALID, name
    for change in ({"dtype": 7}, {"Hq": 5}, {"size": 1000}, {"k": 4104}, {"v": 4098}, {"ws": 4100}):
        assert status(**change) == capi.ERR_INVALID, change
    size = C.c_size_t(7)
    fn = capi.lib().kvflux_paged_attention_shared_workspace_size
    assert fn(3, 64, 2, 4, 16, 128, 1, 1, None) == capi.ERR_INVALID
    assert fn(3, 64, 2, 5, 16, 128, 1, 1, C.byref(size)) == capi.ERR_INVALID and size.value == 0
    assert fn(3, 64, 2, 4, 16, 128, 9, 1, C.byref(size)) == capi.ERR_INVALID
    assert fn(3, 64, 2, 4, 16, 128, 1, 1, C.byref(size)) == capi.OK and size.value > 0
    assert fn(3, BOUND, 2, 4, 16, 128, 1, 1, C.byref(size)) == capi.OK
    assert status(size=100000) == capi.ERR_INVALID  # less than the shared kernel takes
    ordinary = C.c_size_t()
    capi.call("kvflux_paged_attention_workspace_size", 3, 9000, 2, 4, 16, 128, C.byref(ordinary))
    assert fn(3, 9000, 2, 4, 16, 128, 1, 0, C.byref(size)) == capi.OK and size.value == ordinary.value
    assert fn(5000, 9000, 2, 4, 16, 128, 1, 4, C.byref(size)) == capi.OK
    capi.call("kvflux_paged_attention_workspace_size", 5000, 9000, 2, 4, 16, 128, C.byref(ordinary))
    assert size.value == ordinary.value
    # Where either kernel may take the call the workspace serves both.
    for kv in (64, 100000):
        capi.call("kvflux_paged_attention_workspace_size", 64, kv, 8, 32, 16, 128, C.byref(ordinary))
        assert fn(64, kv, 8, 32, 16, 128, 1, 3, C.byref(size)) == capi.OK and size.value >= max(1, ordinary.value)
