"""kvflux_norm_rope_write and its _tail form against the formula in 64 bits.

Tolerances, with u = 2^-24 (half an FP32 step): the sum of squares of up to 512
values in FP32 is off by at most 14u, the scale by half of that and 3u more, and
two products make a normed value off by at most 12u of itself. cos and sin are
off by at most 5u (2 units in the last place, and the angle rounded to FP32 below
an eighth of a turn). So y = a cos - b sin is off by at most 20u (|a| + |b|).
A key is then rounded once: half a step of its type, and half the least step.
Values of the cache's type are bits; others are rounded to nearest even.
"""
from __future__ import annotations

import numpy as np
import pytest

from kvflux_amd import capi, device

U = 2.0 ** -24
CODE = {"f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16, "f32": capi.DTYPE_F32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
HALF_LEAST = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}
STORAGE = {"f16": np.uint16, "bf16": np.uint16, "f32": np.uint32}
EPS = 1e-5


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


def reference(x, weight, positions, inv_freq, rotary, interleaved):
    """(result, tolerance) of normed and rotated rows, [tokens][heads][D] in 64 bits."""
    n = x if weight is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * weight
    y, tol = n.copy(), 12 * U * np.abs(n)
    if rotary:
        a = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
        b = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
        angle = positions[:, None, None] * inv_freq
        c, s = np.cos(angle), np.sin(angle)
        y[..., a] = n[..., a] * c - n[..., b] * s
        y[..., b] = n[..., b] * c + n[..., a] * s
        tol[..., a] = tol[..., b] = 20 * U * (np.abs(n[..., a]) + np.abs(n[..., b]))
    return y, tol


class Call:
    """One call's buffers; `run` makes it and compares every byte it may write."""

    def __init__(self, rng, dtype="bf16", inp=None, heads=(8, 2), D=128, bs=16, rotary=None, interleaved=False,
                 norm=(True, True), tokens=5, packed=True, shift=0, pages=None, scale=1.7):
        self.dtype, self.inp = dtype, inp or dtype
        self.Hq, self.H = heads
        self.D, self.bs, self.tokens = D, bs, tokens
        self.rotary = D if rotary is None else rotary
        self.interleaved = interleaved
        self.pages = pages or max(3, -(-tokens // bs) + 2)
        Hq, H = heads
        self.x = (rng.standard_normal((tokens, Hq + 2 * H, D)) * scale).astype(np.float32)
        bits = to_bits(self.x, self.inp)
        self.x = from_bits(bits, self.inp)
        self.value_bits = bits[:, Hq + H:]
        item = bits.itemsize
        # `shift`: elements that the whole input is moved up by (misaligned vectors).
        self.input = device.DeviceBuffer(bits.nbytes + (shift + 8) * item)
        if packed:
            self.input.upload(bits, shift * item)
            self.strides = [(Hq + 2 * H) * D] * 3
            self.at = [shift, shift + Hq * D, shift + (Hq + H) * D]
        else:
            parts = [bits[:, :Hq], bits[:, Hq:Hq + H], bits[:, Hq + H:]]
            self.at = [shift, shift + parts[0].size, shift + parts[0].size + parts[1].size]
            for at, part in zip(self.at, parts):
                self.input.upload(np.ascontiguousarray(part), at * item)
            self.strides = [Hq * D, H * D, H * D]
        self.item = item
        self.norm = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if on else None for on in norm]
        self.norm_dev = [None if w is None else device.to_device(w) for w in self.norm]
        self.inv_freq = 10000.0 ** (-np.arange(0, self.rotary, 2) / max(1, self.rotary))
        self.inv_dev = device.to_device(self.inv_freq) if self.rotary else None
        shape = (self.pages, H, bs, D)
        self.cache = [rng.integers(0, 1 << 15, shape).astype(STORAGE[dtype]) for _ in range(2)]
        self.cache_dev = [device.to_device(c) for c in self.cache]
        self.out0 = np.full((tokens, Hq, D), 777.0, np.float32)
        self.out_dev = device.to_device(self.out0)

    def head(self):
        ptr = [None if w is None else w.ptr for w in self.norm_dev]
        return (self.cache_dev[0].ptr, self.cache_dev[1].ptr, self.pages, self.H, self.bs, self.D, CODE[self.dtype],
                *(self.input.ptr + a * self.item for a in self.at), CODE[self.inp], *self.strides, self.Hq, *ptr, EPS,
                self.inv_dev.ptr if self.inv_dev else None, self.rotary, int(self.interleaved))

    def listed(self, positions, slots, stream=0):
        self.positions, self.slots = np.asarray(positions, np.uint64), np.asarray(slots, np.uint64)
        self.meta = device.to_device(self.positions), device.to_device(self.slots)
        capi.call("kvflux_norm_rope_write", *self.head(), self.meta[0].ptr, self.meta[1].ptr, self.tokens,
                  self.out_dev.ptr, stream)

    def tail(self, table, lens, stream=0):
        self.table, self.lens = np.asarray(table, np.uint64), np.asarray(lens, np.uint64)
        self.meta = device.to_device(self.table), device.to_device(self.lens)
        capi.call("kvflux_norm_rope_write_tail", *self.head(), self.meta[0].ptr, self.table.shape[1],
                  self.meta[1].ptr, self.tokens, self.out_dev.ptr, stream)

    def check(self, positions, slots, live=None):
        """positions, slots per token (slot None: not written); live: tokens whose query is written."""
        Hq, H, D, bs = self.Hq, self.H, self.D, self.bs
        positions = np.asarray(positions, np.float64)
        live = np.ones(self.tokens, bool) if live is None else np.asarray(live)
        want, tol = reference(self.x[:, :Hq], self.norm[0], positions, self.inv_freq, self.rotary, self.interleaved)
        out = self.out_dev.download(np.float32).reshape(self.out0.shape)
        assert np.array_equal(out[~live], self.out0[~live])
        assert (np.abs(out[live] - want[live]) <= tol[live]).all(), np.abs(out[live] - want[live]).max()
        key, key_tol = reference(self.x[:, Hq:Hq + H], self.norm[1], positions, self.inv_freq, self.rotary,
                                 self.interleaved)
        key_tol = key_tol * (1 + HALF_STEP[self.dtype]) + np.abs(key) * HALF_STEP[self.dtype] + HALF_LEAST[self.dtype]
        got = [d.download(STORAGE[self.dtype]).reshape(c.shape) for d, c in zip(self.cache_dev, self.cache)]
        if self.dtype == self.inp:
            values = self.value_bits
        else:
            values = to_bits(self.x[:, Hq + H:], self.dtype)
        untouched = np.ones((self.pages, bs), bool)
        for n, slot in enumerate(slots):
            if slot is None:
                continue
            page, off = int(slot) // bs, int(slot) % bs
            untouched[page, off] = False
            k = from_bits(np.ascontiguousarray(got[0][page, :, off]), self.dtype)
            assert (np.abs(k - key[n]) <= key_tol[n]).all(), (n, np.abs(k - key[n]).max())
            assert np.array_equal(got[1][page, :, off], values[n]), n
        for g, c in zip(got, self.cache):
            assert np.array_equal(g.transpose(0, 2, 1, 3)[untouched], c.transpose(0, 2, 1, 3)[untouched])


def slots_for(rng, c):
    return rng.permutation(c.pages * c.bs)[:c.tokens]


SHAPES = [  # heads, head size, page, rotated dims: the fast kernel's head sizes, and ones it leaves to the other
    ((8, 2), 128, 16, 128), ((4, 4), 64, 16, 64), ((7, 1), 256, 8, 128), ((3, 1), 512, 4, 512), ((6, 2), 80, 16, 80),
    ((2, 1), 96, 5, 32), ((4, 2), 64, 16, 24), ((3, 3), 4, 2, 4), ((2, 1), 3, 3, 2), ((5, 1), 128, 1, 0),
    ((8, 2), 112, 16, 56), ((4, 1), 40, 16, 40), ((2, 2), 8, 16, 8), ((1, 1), 1, 4, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0][0]}x{s[0][1]}x{s[1]}r{s[3]}b{s[2]}")
def test_shapes(gpu, shape, dtype, interleaved):
    rng = np.random.default_rng(11)
    c = Call(rng, dtype, heads=shape[0], D=shape[1], bs=shape[2], rotary=shape[3], interleaved=interleaved, tokens=7)
    slots = slots_for(rng, c)
    positions = rng.integers(0, 5000, 7)
    c.listed(positions, slots)
    c.check(positions, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("inp", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_input_types(gpu, dtype, inp):
    rng = np.random.default_rng(12)
    for D, shift in ((128, 0), (128, 1)):
        c = Call(rng, dtype, inp, D=D, tokens=9, shift=shift, packed=shift == 0)
        slots = slots_for(rng, c)
        c.listed(np.arange(9), slots)
        c.check(np.arange(9), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [(False, False), (True, False), (False, True)])
def test_without_norms(gpu, norm):
    rng = np.random.default_rng(13)
    for rotary in (0, 64, 128):
        c = Call(rng, "bf16", norm=norm, rotary=rotary, tokens=4)
        slots = slots_for(rng, c)
        c.listed([0, 1, 2, 3], slots)
        c.check([0, 1, 2, 3], slots)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 63, 257, 1000])
@pytest.mark.parametrize("heads", [(32, 8), (28, 4), (1, 1), (71, 1), (3, 9)])
def test_token_counts(gpu, tokens, heads):
    rng = np.random.default_rng(14)
    c = Call(rng, "bf16", heads=heads, D=64, tokens=tokens)
    slots = slots_for(rng, c)
    positions = np.arange(tokens) + 17
    c.listed(positions, slots)
    c.check(positions, slots)


@pytest.mark.gpu
def test_far_positions(gpu):
    """Angles of a million radians: FP32 angles would be off by 2^-5."""
    rng = np.random.default_rng(15)
    positions = [0, 1, 131071, 131072, 1 << 20, (1 << 20) + 1]
    for interleaved in (False, True):
        c = Call(rng, "f32", D=128, tokens=6, interleaved=interleaved)
        slots = slots_for(rng, c)
        c.listed(positions, slots)
        c.check(positions, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 80])
def test_skipped_slots(gpu, D):
    """A slot past the pool, and the largest number, leave the caches alone; the queries are written."""
    rng = np.random.default_rng(16)
    c = Call(rng, "bf16", D=D, tokens=4, rotary=D)
    slots = [5, c.pages * c.bs, 2 ** 64 - 1, 0]
    c.listed([3, 4, 5, 6], slots)
    c.check([3, 4, 5, 6], [5, None, None, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 80])
def test_tail(gpu, D):
    """Slots and positions from the table; empty rows, a missing page and a short table."""
    rng = np.random.default_rng(17)
    bs = 4
    c = Call(rng, "bf16", D=D, bs=bs, tokens=6, pages=10, rotary=D)
    lens = [1, 0, 8, 9, 5, 30]  # the last: block 7 of a table of 3
    none = 2 ** 64 - 1
    table = [[7, none, none], [2, 2, 2], [0, 3, none], [1, 4, 6], [8, 10, 8], [5, 9, 5]]  # page 10 is past the pool
    c.tail(table, lens)
    c.check([0, 0, 7, 8, 4, 29], [7 * bs, None, 3 * bs + 3, 6 * bs, None, None], [True, False, True, True, True, True])


@pytest.mark.gpu
def test_rows_of_zeros(gpu):
    """A row of zeros norms to zeros (eps keeps the scale finite)."""
    rng = np.random.default_rng(18)
    c = Call(rng, "bf16", heads=(2, 1), D=64, tokens=3)
    bits = to_bits(c.x, "bf16").reshape(3, 4, 64)
    bits[1] = 0
    c.input.upload(bits)
    c.x = from_bits(bits, "bf16")
    c.value_bits = bits[:, 3:]
    slots = slots_for(rng, c)
    c.listed([1, 2, 3], slots)
    c.check([1, 2, 3], slots)


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_rows(gpu):
    rng = np.random.default_rng(19)
    c = Call(rng, "f32", heads=(2, 1), D=128, tokens=3)
    bits = to_bits(c.x, "f32").reshape(3, 4, 128)
    bits[1, 0, 5] = 0x7fc00000  # NaN in a query
    bits[2, 2, 9] = 0x7f800000  # infinity in a key
    bits[0, 3, 1] = 0x7fc12345  # NaN payload in a value: bits
    c.input.upload(bits)
    slots = [0, 1, 2]
    c.listed([1, 2, 3], slots)
    out = c.out_dev.download(np.float32).reshape(3, 2, 128)
    assert np.isnan(out[1, 0]).all()
    finite = np.ones((3, 2), bool)
    finite[1, 0] = False
    assert np.isfinite(out[finite]).all()
    key = c.cache_dev[0].download(np.float32).reshape(c.cache[0].shape)
    value = c.cache_dev[1].download(np.uint32).reshape(c.cache[1].shape)
    assert np.isfinite(key[0, 0, :2]).all() and np.isnan(key[0, 0, 2]).any()
    assert np.array_equal(value[0, 0, 0], bits[0, 3])


@pytest.mark.gpu
def test_large_slots(gpu):
    """Pages behind 2^32 elements: the last pages of a cache of over 8 GiB a tensor."""
    H, D, bs = 8, 128, 16
    pages = (1 << 32) // (H * D * bs) + 40
    k, v = device.DeviceBuffer(pages * H * D * bs * 2), device.DeviceBuffer(pages * H * D * bs * 2)
    rng = np.random.default_rng(20)
    c = Call(rng, "bf16", heads=(8, H), D=D, bs=bs, tokens=3)
    c.cache_dev, small, c.pages = [k, v], c.pages, pages
    slots = [pages * bs - 1, (pages - 1) * bs, (pages - 39) * bs + 3]
    c.listed([1, 2, 3], slots)
    key, tol = reference(c.x[:, 8:16], c.norm[1], np.array([1.0, 2.0, 3.0]), c.inv_freq, D, False)
    for n, s in enumerate(slots):
        for h in range(H):
            at = ((s // bs * H + h) * bs + s % bs) * D * 2
            got = from_bits(k.download(np.uint16, D, at), "bf16")
            assert (np.abs(got - key[n, h]) <= tol[n, h] * 1.01 + np.abs(key[n, h]) * HALF_STEP["bf16"]).all()
            assert np.array_equal(v.download(np.uint16, D, at), c.value_bits[n, h])
    assert small > 0


def test_refusals():
    """Checked on the host before anything is launched (no GPU needed)."""
    ok = dict(kc=4096, vc=4096, blocks=4, H=2, bs=16, D=64, dtype=1, q=4096, k=4096, v=4096, inp=1, qs=512, ks=512,
              vs=512, Hq=4, qn=4096, kn=4096, eps=1e-6, inv=4096, rot=64, inter=0, pos=4096, slots=4096, n=3, out=4096)

    def status(fn="kvflux_norm_rope_write", **change):
        a = {**ok, **change}
        args = [a[x] for x in ("kc", "vc", "blocks", "H", "bs", "D", "dtype", "q", "k", "v", "inp", "qs", "ks", "vs",
                               "Hq", "qn", "kn", "eps", "inv", "rot", "inter")]
        if fn.endswith("tail"):
            args += [a["pos"], change.get("width", 4), a["slots"], a["n"], a["out"], None]
        else:
            args += [a["pos"], a["slots"], a["n"], a["out"], None]
        return getattr(capi.lib(), fn)(*args)

    for fn in ("kvflux_norm_rope_write", "kvflux_norm_rope_write_tail"):
        assert status(fn, n=0) == capi.OK
        for name in ("kc", "vc", "q", "k", "v", "out", "pos", "slots", "inv"):
            assert status(fn, **{name: None}) == capi.ERR_INVALID, name
        for name in ("blocks", "H", "bs", "D", "Hq"):
            assert status(fn, **{name: 0}) == capi.ERR_INVALID, name
        for change in ({"dtype": 3}, {"inp": -1}, {"rot": 63}, {"rot": 66}, {"eps": -1.0}, {"eps": float("nan")},
                       {"eps": float("inf")}, {"qs": 255}, {"ks": 127}, {"vs": 127}, {"q": 4097}, {"out": 4098},
                       {"inv": 4100}, {"kc": 4097}, {"qn": 4097}):
            assert status(fn, **change) == capi.ERR_INVALID, change
        assert status(fn, D=520, rot=64, qs=4096, ks=4096, vs=4096) == capi.ERR_UNSUPPORTED
        assert status(fn, n=1 << 26) == capi.ERR_UNSUPPORTED
        assert status(fn, blocks=1 << 62, bs=64) == capi.ERR_OVERFLOW
    assert status("kvflux_norm_rope_write_tail", width=0) == capi.ERR_INVALID
    assert "norm, rotation" in capi.last_error()
