"""Prompts on an 8-bit cache whose merge would have more threads than a grid counts: refused
before any GPU call (so on the CPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from kvflux_amd import capi
from test_quant_refusals import P, cache_args, prefill, status


@pytest.mark.parametrize("D,most,group,want", [(16, 16384, 16411, capi.ERR_UNSUPPORTED), (256, 16384, 8191, capi.ERR_UNSUPPORTED),
                                               (16, 16384, 1031, None)])
def test_merges(D, most, group, want):
    """Groups that are primes past a workgroup's rows: a launch for each query head, few workgroups of each, so
    that the keys are split, and a merge over all of them."""
    size = C.c_size_t()
    got = status("kvflux_quant_prefill_workspace_size", 1, most, most, 1, group, 16, D, C.byref(size))
    if want is None:
        assert got == capi.OK and size.value > 0
        return
    assert got == want and size.value == 0
    assert prefill(cache_args(heads=1, D=D), seqs=1, most=most, kv_len=most, Hq=group, q=P, o=P) == want
