"""What the calls on an 8-bit cache refuse, before any GPU call (so on the CPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from kvflux_amd import capi

P = 0x10000  # an address that is never touched
CACHE = dict(k=P, v=P, ks=P, vs=P, blocks=8, heads=2, bs=16, D=128, fmt=capi.QUANT_E4M3)


def status(name, *args):
    return getattr(capi.lib(), name)(*args)


def cache_args(**change):
    return tuple({**CACHE, **change}.values())


def write(cache=None, **change):
    a = dict(kn=P, vn=P, dtype=capi.DTYPE_BF16, kst=256, vst=256, table=P, width=4, lens=P, new=P, off=P, seqs=3, most=5,
             stream=None) | change
    return status("kvflux_quant_write", *(cache or cache_args()), *a.values())


def tail(cache=None, **change):
    a = dict(kn=P, vn=P, dtype=capi.DTYPE_BF16, kst=256, vst=256, table=P, width=4, lens=P, rows=3, stream=None) | change
    return status("kvflux_quant_write_tail", *(cache or cache_args()), *a.values())


def gather(cache=None, **change):
    a = dict(table=P, width=4, lens=P, off=P, starts=P, seqs=3, pages=5, ko=P, vo=P, dtype=capi.DTYPE_BF16,
             stream=None) | change
    return status("kvflux_quant_gather", *(cache or cache_args()), *a.values())


def attend(cache=None, **change):
    a = dict(table=P, width=4, lens=P, kv_len=400, rows=3, Hq=8, q=P, o=P, ws=P, bytes=1 << 40, stream=None) | change
    return status("kvflux_quant_attention", *(cache or cache_args()), *a.values())


def prefill(cache=None, **change):
    a = dict(table=P, width=40, lens=P, ql=P, qo=P, seqs=3, most=7, kv_len=400, Hq=8, q=P, o=P, ws=P, bytes=1 << 60,
             stream=None) | change
    return status("kvflux_quant_prefill", *(cache or cache_args()), *a.values())


CALLS = [write, tail, gather, attend, prefill]
BAD_CACHES = [
    (dict(fmt=2), capi.ERR_INVALID), (dict(fmt=-1), capi.ERR_INVALID), (dict(k=None), capi.ERR_INVALID),
    (dict(v=None), capi.ERR_INVALID), (dict(ks=None), capi.ERR_INVALID), (dict(vs=None), capi.ERR_INVALID),
    (dict(blocks=0), capi.ERR_INVALID), (dict(heads=0), capi.ERR_INVALID), (dict(bs=0), capi.ERR_INVALID),
    (dict(D=0), capi.ERR_INVALID), (dict(ks=P + 2), capi.ERR_INVALID), (dict(vs=P + 1), capi.ERR_INVALID),
    (dict(heads=1 << 16), capi.ERR_UNSUPPORTED), (dict(bs=1 << 30), capi.ERR_UNSUPPORTED),
    (dict(blocks=1 << 60), capi.ERR_OVERFLOW), (dict(blocks=2 ** 64 - 1), capi.ERR_OVERFLOW)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,want", BAD_CACHES)
def test_caches(call, change, want):
    assert call(cache_args(**change)) == want
    assert capi.last_error()


@pytest.mark.parametrize("change,want", [
    (dict(kn=None), capi.ERR_INVALID), (dict(vn=None), capi.ERR_INVALID), (dict(table=None), capi.ERR_INVALID),
    (dict(lens=None), capi.ERR_INVALID), (dict(width=0), capi.ERR_INVALID), (dict(dtype=3), capi.ERR_INVALID),
    (dict(kn=P + 1), capi.ERR_INVALID), (dict(kst=255), capi.ERR_INVALID), (dict(vst=0), capi.ERR_INVALID),
    (dict(table=P + 4), capi.ERR_INVALID)])
def test_writes(change, want):
    assert write(**change) == want
    assert tail(**change) == want


def test_sizes_of_writes():
    assert write(new=None) == capi.ERR_INVALID and write(off=None) == capi.ERR_INVALID
    assert write(seqs=1 << 31) == capi.ERR_UNSUPPORTED and write(most=1 << 40) == capi.ERR_UNSUPPORTED
    assert write(seqs=1 << 23, most=1) == capi.ERR_UNSUPPORTED and gather(pages=1 << 24) == capi.ERR_UNSUPPORTED
    assert write(most=2 ** 64 - 1) == capi.ERR_UNSUPPORTED and tail(rows=1 << 31) == capi.ERR_UNSUPPORTED
    assert write(seqs=0, kn=None) == capi.OK and write(most=0, kn=None) == capi.OK and tail(rows=0, kn=None) == capi.OK


@pytest.mark.parametrize("change,want", [
    (dict(ko=None), capi.ERR_INVALID), (dict(vo=None), capi.ERR_INVALID), (dict(table=None), capi.ERR_INVALID),
    (dict(lens=None), capi.ERR_INVALID), (dict(off=None), capi.ERR_INVALID), (dict(starts=None), capi.ERR_INVALID),
    (dict(width=0), capi.ERR_INVALID), (dict(dtype=7), capi.ERR_INVALID), (dict(ko=P + 1), capi.ERR_INVALID),
    (dict(seqs=1 << 31), capi.ERR_UNSUPPORTED), (dict(pages=1 << 31), capi.ERR_UNSUPPORTED)])
def test_reads(change, want):
    assert gather(**change) == want


def test_nothing_to_read():
    assert gather(seqs=0, table=None) == capi.OK and gather(pages=0, table=None) == capi.OK


@pytest.mark.parametrize("change,want", [
    (dict(table=None), capi.ERR_INVALID), (dict(lens=None), capi.ERR_INVALID), (dict(q=None), capi.ERR_INVALID),
    (dict(o=None), capi.ERR_INVALID), (dict(width=0), capi.ERR_INVALID), (dict(Hq=0), capi.ERR_INVALID),
    (dict(Hq=7), capi.ERR_INVALID), (dict(q=P + 2), capi.ERR_INVALID), (dict(o=P + 1), capi.ERR_INVALID),
    (dict(table=P + 4), capi.ERR_INVALID), (dict(Hq=1 << 20), capi.ERR_UNSUPPORTED),
    (dict(kv_len=1 << 32), capi.ERR_UNSUPPORTED), (dict(rows=1 << 32), capi.ERR_UNSUPPORTED),
    (dict(kv_len=5000, ws=None), capi.ERR_INVALID), (dict(kv_len=5000, bytes=100), capi.ERR_INVALID),
    (dict(kv_len=5000, ws=P + 4), capi.ERR_INVALID)])
def test_attention(change, want):
    assert attend(**change) == want


def test_head_sizes_of_attention():
    assert attend(cache_args(D=513)) == capi.ERR_UNSUPPORTED
    assert attend(rows=0, table=None) == capi.OK


def test_workspace_sizes_of_attention():
    size = C.c_size_t(7)

    def ask(rows=4, kv_len=2000, H=2, Hq=8, bs=16, D=128):
        return status("kvflux_quant_attention_workspace_size", rows, kv_len, H, Hq, bs, D, C.byref(size))

    assert ask() == capi.OK and size.value > 0
    assert ask(kv_len=512) == capi.OK and size.value == 0
    assert ask(rows=0) == capi.OK and size.value == 0
    assert ask(D=96) == capi.OK and size.value > 0
    assert ask(D=100) == capi.OK and size.value == 0 and ask(D=272) == capi.OK and size.value == 0
    assert ask(Hq=7) == capi.ERR_INVALID and ask(H=0) == capi.ERR_INVALID and ask(kv_len=1 << 32) == capi.ERR_UNSUPPORTED
    assert status("kvflux_quant_attention_workspace_size", 1, 1, 1, 1, 1, 64, None) == capi.ERR_INVALID


@pytest.mark.parametrize("change,want", [
    (dict(table=None), capi.ERR_INVALID), (dict(lens=None), capi.ERR_INVALID), (dict(ql=None), capi.ERR_INVALID),
    (dict(qo=None), capi.ERR_INVALID), (dict(q=None), capi.ERR_INVALID), (dict(o=None), capi.ERR_INVALID),
    (dict(width=0), capi.ERR_INVALID), (dict(Hq=0), capi.ERR_INVALID), (dict(Hq=7), capi.ERR_INVALID),
    (dict(q=P + 2), capi.ERR_INVALID), (dict(qo=P + 4), capi.ERR_INVALID), (dict(most=401), capi.ERR_INVALID),
    (dict(Hq=1 << 20), capi.ERR_UNSUPPORTED), (dict(kv_len=1 << 31), capi.ERR_UNSUPPORTED),
    (dict(seqs=1 << 16), capi.ERR_UNSUPPORTED), (dict(seqs=60000, most=30000, kv_len=30000), capi.ERR_UNSUPPORTED),
    (dict(kv_len=50000, ws=None), capi.ERR_INVALID), (dict(kv_len=50000, bytes=100), capi.ERR_INVALID),
    (dict(kv_len=50000, ws=P + 2), capi.ERR_INVALID)])
def test_prefill(change, want):
    assert prefill(**change) == want


def test_shapes_of_prefill():
    assert prefill(cache_args(D=513)) == capi.ERR_UNSUPPORTED and prefill(cache_args(blocks=1 << 31)) == capi.ERR_UNSUPPORTED
    assert prefill(seqs=0, table=None) == capi.OK and prefill(most=0, table=None) == capi.OK
    size = C.c_size_t(7)

    def ask(seqs=1, most=8, kv_len=50000, H=2, Hq=8, bs=16, D=128):
        return status("kvflux_quant_prefill_workspace_size", seqs, most, kv_len, H, Hq, bs, D, C.byref(size))

    assert ask() == capi.OK and size.value > 0
    assert ask(seqs=64, most=4096, kv_len=4096, H=8, Hq=32) == capi.OK and size.value == 0
    assert ask(D=80) == capi.OK and size.value > 0
    assert ask(D=84) == capi.OK and size.value == 0
    assert ask(seqs=0) == capi.OK and size.value == 0
    assert ask(most=50001) == capi.ERR_INVALID and ask(Hq=3) == capi.ERR_INVALID and ask(kv_len=1 << 31) == capi.ERR_UNSUPPORTED
    assert status("kvflux_quant_prefill_workspace_size", 1, 1, 1, 1, 1, 1, 64, None) == capi.ERR_INVALID
