"""An 8-bit paged cache in 64 bits (numpy), and its copy on the GPU."""
from __future__ import annotations

import math

import numpy as np

from kvflux_amd import capi, device

FORMAT = {"e4m3": capi.QUANT_E4M3, "int8": capi.QUANT_INT8}
TOP = {"e4m3": 448.0, "int8": 127.0}
CODE = {"f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16, "f32": capi.DTYPE_F32}
ITEM = {"f16": 2, "bf16": 2, "f32": 4}


def _e4m3_values():
    b = np.arange(256)
    e, m = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b > 127, -v, v)


#: What each byte stands for.
VALUES = {"e4m3": _e4m3_values(), "int8": np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)}


def hold(y, fmt):
    """Bytes of the values (at most TOP in size): the nearest, ties to even."""
    if fmt == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    mag = np.abs(y)
    _, e = np.frexp(mag)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    byte = np.searchsorted(VALUES["e4m3"][:127], np.rint(mag / step) * step).astype(np.uint8)
    return byte | (np.signbit(y).astype(np.uint8) << 7)


def scale_of(largest, fmt):
    if not np.isfinite(largest):
        return np.nan
    k = -110
    if largest > 0:
        m, e = math.frexp(largest / TOP[fmt])  # largest / 448 or / 127 as a power of two's bound
        k = max(-110, e - 3)
        while largest > TOP[fmt] * 2.0 ** k:
            k += 1
    return 2.0 ** k


def to_bits(x, name):
    x = np.ascontiguousarray(x, np.float32)
    if name == "f32":
        return x.view(np.uint32).copy()
    if name == "f16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bits(b, name):
    if name == "f32":
        return b.view(np.float32).astype(np.float64)
    if name == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Cache:
    """bytes [2][blocks][H][bs][D] and scales [2][blocks][H] of K and V, here and on the GPU."""

    def __init__(self, fmt, blocks, H, bs, D, shift=0):
        self.fmt, self.blocks, self.H, self.bs, self.D = fmt, blocks, H, bs, D
        self.bytes = np.full((2, blocks, H, bs, D), 0xff, np.uint8)  # e4m3: NaN where nothing was written
        self.scales = np.full((2, blocks, H), np.nan, np.float32)
        self.shift = shift  # bytes that the caches are moved up by
        self.dev = [device.DeviceBuffer(self.bytes[0].nbytes + 64) for _ in range(2)]
        self.dev_scales = [device.DeviceBuffer(self.scales[0].nbytes) for _ in range(2)]
        self.upload()

    def upload(self):
        for i in range(2):
            self.dev[i].upload(self.bytes[i], self.shift)
            self.dev_scales[i].upload(self.scales[i])

    def download(self):
        b = [self.dev[i].download(np.uint8, self.bytes[0].size, self.shift).reshape(self.bytes[0].shape) for i in range(2)]
        s = [self.dev_scales[i].download(np.float32).reshape(self.scales[0].shape) for i in range(2)]
        return np.stack(b), np.stack(s)

    def args(self):
        return (self.dev[0].ptr + self.shift, self.dev[1].ptr + self.shift, self.dev_scales[0].ptr,
                self.dev_scales[1].ptr, self.blocks, self.H, self.bs, self.D, FORMAT[self.fmt])

    def values(self):
        return VALUES[self.fmt][self.bytes] * self.scales[..., None, None].astype(np.float64)

    def fill(self, rng, size=1.0, spread=2.0, scales=None):
        """Every page and head written, values of a size of its own; `scales`: powers of two by default."""
        x = rng.standard_normal(self.bytes.shape) * size * np.exp2(rng.uniform(-spread, spread, self.scales.shape))[..., None, None]
        top = np.abs(x).max((3, 4))
        s = np.vectorize(lambda a: scale_of(a, self.fmt))(top) if scales is None else top / TOP[self.fmt] * scales
        self.scales = s.astype(np.float32)
        self.bytes = hold(np.clip(x / self.scales[..., None, None].astype(np.float64), -TOP[self.fmt], TOP[self.fmt]), self.fmt)
        self.upload()

    def write(self, which, table, lens, new, offsets, rows):
        """The definition of kvflux_quant_write; rows [tokens][H][D] in 64 bits."""
        for r, (n, m) in enumerate(zip(lens, new)):
            n, m = int(n), int(min(m, n))
            for page in range((n - m) // self.bs, -(-n // self.bs) if m else 0):
                if page >= table.shape[1] or table[r, page] >= self.blocks:
                    continue
                at, i = page * self.bs, int(table[r, page])
                first, last = max(0, n - m - at), min(self.bs, n - at)
                x = rows[int(offsets[r]) + at + first - (n - m):][:last - first]
                for h in range(self.H):
                    before = float(self.scales[which, i, h])
                    with np.errstate(invalid="ignore"):
                        s = scale_of(np.abs(x[:, h]).max(), self.fmt)
                    if first and not np.isnan(s) and (np.isnan(before) or before > s):
                        s = before
                    if not np.isnan(s):
                        if first and s != before:
                            self.bytes[which, i, h, :first] = hold(VALUES[self.fmt][self.bytes[which, i, h, :first]] * (before / s), self.fmt)
                        self.bytes[which, i, h, first:last] = hold(x[:, h] / s, self.fmt)
                    self.scales[which, i, h] = s


def random_table(rng, lens, bs, blocks, width=None):
    """Distinct random pages for every sequence; ~0 behind a row's pages."""
    counts = [-(-int(n) // bs) for n in lens]
    width = width or max(1, max(counts))
    order = rng.permutation(blocks)
    assert sum(counts) <= blocks
    table = np.full((len(counts), width), 2 ** 64 - 1, np.uint64)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    return table


def u64(x):
    return device.to_device(np.ascontiguousarray(x).astype(np.uint64))


def attention(cache, table, n, q, visible=None):
    """Outputs [rows][Hq][D] in 64 bits of queries [rows][Hq][D] over the first n tokens of a
    table row (row i sees visible[i] of them, all by default; missing pages drop out)."""
    Hq, D = q.shape[1:]
    G = Hq // cache.H
    pages = np.asarray(table[:-(-n // cache.bs)], np.uint64)
    n = min(n, len(pages) * cache.bs)  # a table row may end before its tokens
    ok = np.repeat(pages < cache.blocks, cache.bs)[:n]
    ids = np.where(pages < cache.blocks, pages, 0).astype(np.int64)
    values = VALUES[cache.fmt][cache.bytes[:, ids]] * cache.scales[:, ids][..., None, None].astype(np.float64)
    k, v = values.transpose(0, 2, 1, 3, 4).reshape(2, cache.H, -1, D)[:, :, :n]
    out = np.zeros(q.shape)
    for i in range(q.shape[0]):
        see = ok & (np.arange(n) < (n if visible is None else int(visible[i])))
        if not see.any():
            continue
        for h in range(cache.H):
            s = q[i, h * G:(h + 1) * G].astype(np.float64) @ k[h][see].T / math.sqrt(D)
            w = np.exp(s - s.max(-1, keepdims=True))
            out[i, h * G:(h + 1) * G] = w @ v[h][see] / w.sum(-1, keepdims=True)
    return out
