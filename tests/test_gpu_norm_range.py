"""RMS norms of rows whose squares leave FP32's range, and with eps 0.

Tolerances as in test_gpu_norm_rope_write: the steps that keep such a row in range
are products with powers of two, exact but for sums that are far below the row's.
Values below 2^-126, which only these rows have, round to FP32's least step,
2^-149, whatever their size: a normed value in up to two products, half a step
each; then y = a cos - b sin has (|cos| + |sin|) times that, at most 1.42 steps,
and half a step from each product (the sum of two such is exact). Under 3 steps.
"""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_norm_rope_write as nrw

LEAST = 2.0 ** -149


@pytest.fixture(autouse=True)
def least_steps(monkeypatch):
    plain = nrw.reference

    def reference(*args):
        y, tol = plain(*args)
        return y, tol + 3 * LEAST

    monkeypatch.setattr(nrw, "reference", reference)


# head size, rotated dims, elements the input is moved up by: the fast kernel (16 lanes a row, 10 of 16, one), the other
SHAPES = [(128, 128, 0), (80, 80, 0), (8, 8, 0), (80, 20, 0), (128, 64, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary,shift", SHAPES)
@pytest.mark.parametrize("inp", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-20, 1e-15, 1.0, 1e15, 1e19, 1e30, 5e37])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-5])
def test_sizes(gpu, monkeypatch, eps, size, inp, D, rotary, shift):
    """Means from 1e-76 to 1e75 (FP32: 1e-45 to 3e38), rows of ordinary size beside them in a wavefront."""
    monkeypatch.setattr(nrw, "EPS", eps)
    rng = np.random.default_rng(51)
    c = nrw.Call(rng, "f32", inp, D=D, rotary=rotary, tokens=6, shift=shift, scale=size)
    rows = nrw.to_bits(c.x, inp)
    rows[::2] = nrw.to_bits(rng.standard_normal(rows[::2].shape), inp)
    c.input.upload(rows, shift * c.item)
    c.x, c.value_bits = nrw.from_bits(rows, inp), rows[:, c.Hq + c.H:]
    slots = nrw.slots_for(rng, c)
    positions = rng.integers(0, 5000, 6)
    c.listed(positions, slots)
    c.check(positions, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary,shift", SHAPES)
def test_one_large_value(gpu, monkeypatch, D, rotary, shift):
    """A value of 1e38 among ones of 1, and one of 1e-38 among zeros: the formula's other values, tiny or zero."""
    for eps in (0.0, 1e-5):
        monkeypatch.setattr(nrw, "EPS", eps)
        rng = np.random.default_rng(52)
        c = nrw.Call(rng, "f32", "f32", D=D, rotary=rotary, tokens=2, shift=shift, norm=(True, True))
        rows = nrw.to_bits(c.x, "f32").view(np.float32)
        rows[0, :, 3] = 1e38
        rows[1] = 0
        rows[1, :, 5] = 1e-38
        bits = rows.view(np.uint32)
        c.input.upload(bits, shift * c.item)
        c.x, c.value_bits = nrw.from_bits(bits, "f32"), bits[:, c.Hq + c.H:]
        slots = nrw.slots_for(rng, c)
        c.listed([3, 4], slots)
        c.check([3, 4], slots)


@pytest.mark.gpu
def test_positions_past_the_angles(gpu, v2):
    """2^53 and more have no exact FP64 value: refused, nothing written; the last that has one is taken."""
    from gpu_util import read_cache
    from test_gpu_projected_step import Model, filled
    rng = np.random.default_rng(53)
    pool, storage = filled(v2, "BFloat16", 2, 64, 16, 3, 9)
    model = Model(rng, "BFloat16", 4, 2, 64, 64, False)
    rows, form, q = model.project(v2, rng, 2), model.form(v2), nrw.device.DeviceBuffer(2 * 4 * 64 * 4)
    before = [x.copy() for x in read_cache(storage, "BFloat16")]
    for bad in (2 ** 53, 2 ** 64 - 1):
        with pytest.raises(ValueError):
            v2.norm_rope_write(storage, rows, form, 4, [0, bad], [0, 1], q.ptr)
    assert all(np.array_equal(a, b) for a, b in zip(before, read_cache(storage, "BFloat16")))
    v2.norm_rope_write(storage, rows, form, 4, [0, 2 ** 53 - 1], [0, 1], q.ptr)
    assert np.isfinite(q.download(np.float32)).all()
