"""The 8-bit cache through the C++ layer, its calls used together: prompts written and
attended to, forks, decode steps with copies of shared tails, read back; and the same calls
captured into graphs. Bytes, scales and values read back are compared bit for bit with the
64-bit model, attention within its 1e-5 (test_gpu_quant_attention.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from kvflux_amd import capi, device
from quant_util import Cache, attention, from_bits, random_table, to_bits, u64
from test_gpu_projected_step import Graph

pytestmark = pytest.mark.gpu


class Model(Cache):
    """The 64-bit cache over a v2 storage's memory."""

    def __init__(self, storage):
        layout = storage.layout()
        self.fmt = {"E4M3": "e4m3", "Int8": "int8"}[layout.format().name]
        self.blocks, self.H, self.bs, self.D = layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size()
        self.storage, self.layout = storage, layout
        self.bytes, self.scales = self.download()

    def download(self):
        s, n = self.storage, self.layout
        b = [device.memcpy_d2h(p, n.cache_bytes(), np.uint8).reshape(self.blocks, self.H, self.bs, self.D)
             for p in (s.key_base(), s.value_base())]
        c = [device.memcpy_d2h(p, n.scale_bytes(), np.float32).reshape(self.blocks, self.H)
             for p in (s.key_scales(), s.value_scales())]
        return np.stack(b), np.stack(c)


def pages(seqs):
    width = max(s.num_allocated_blocks() for s in seqs)
    table = np.full((len(seqs), width), 2 ** 64 - 1, np.uint64)
    for r, s in enumerate(seqs):
        table[r, :s.num_allocated_blocks()] = [s.physical_block_id(b) for b in range(s.num_allocated_blocks())]
    return table


def live(seqs, bs):
    """Mask of the tokens that some sequence holds: [blocks of their pages, offsets]."""
    return {(int(s.physical_block_id(t // bs)), t % bs) for s in seqs for t in range(s.num_tokens())}


class Rows:
    """Q, K and V rows side by side, as a projection leaves them."""

    def __init__(self, v2, rng, n, Hq, H, D, name, size=1.0):
        x = (rng.standard_normal((n, Hq + 2 * H, D)) * size).astype(np.float32)
        self.bits = to_bits(x, name)
        self.x = from_bits(self.bits, name)[:, Hq:].reshape(n, 2, H, D)
        self.buffer = device.to_device(self.bits)
        item = self.bits.itemsize
        at, stride = self.buffer.ptr + Hq * D * item, (Hq + 2 * H) * D
        dtype = {"bf16": v2.DType.BFloat16, "f16": v2.DType.Float16, "f32": v2.DType.Float32}[name]
        self.rows = v2.NewRows(at, at + H * D * item, dtype, stride, stride)
        self.q = rng.standard_normal((n, Hq, D)).astype(np.float32)
        self.qd = device.to_device(self.q)


@pytest.mark.parametrize("fmt,name,H,Hq,D,bs", [("E4M3", "bf16", 2, 8, 128, 16), ("Int8", "f16", 2, 14, 64, 32),
                                                ("E4M3", "f32", 1, 4, 256, 8), ("Int8", "bf16", 2, 4, 96, 6),
                                                ("E4M3", "bf16", 2, 4, 128, 5)])
def test_a_serving_loop(gpu, v2, fmt, name, H, Hq, D, bs):
    rng = np.random.default_rng(D + bs)
    pool = v2.PhysicalBlockPool(120, bs)
    holders = [pool.allocate() for _ in range(120)]
    for i in rng.permutation(120):
        pool.free(holders[i])
    storage = v2.QuantizedKVStorage(pool, H, D, getattr(v2.QuantFormat, fmt))
    model = Model(storage)

    def check_cache(seqs):
        got, scales = model.download()
        table = pages(seqs)
        for r, s in enumerate(seqs):
            ids = table[r, :s.num_allocated_blocks()].astype(np.int64)
            assert np.array_equal(scales[:, ids], model.scales[:, ids])
            a, b = (x[:, ids].transpose(0, 1, 3, 2, 4).reshape(2, -1, H, D)[:, :s.num_tokens()] for x in (got, model.bytes))
            assert np.array_equal(a, b)
        return table

    def check_attention(seqs, counts, q, out):
        table, at = pages(seqs), 0
        values = np.abs(model.values())
        for r, (s, m) in enumerate(zip(seqs, counts)):
            n = s.num_tokens()
            want = attention(model, table[r], n, q[at:at + m], visible=n - m + np.arange(m) + 1)
            top = np.nanmax(values[1, table[r, :s.num_allocated_blocks()].astype(np.int64)])
            assert np.abs(out[at:at + m] - want).max() <= 1e-5 * top
            at += m

    def prefill(seqs, counts, size):
        for s, m in zip(seqs, counts):
            s.append_tokens(m)
        n = sum(counts)
        rows = Rows(v2, rng, n, Hq, H, D, name, size)
        out = device.DeviceBuffer(n * Hq * D * 4)
        v2.write_quantized_kv(storage, seqs, counts, rows.rows)
        v2.paged_attention_prompts(storage, seqs, counts, rows.qd.ptr, out.ptr, Hq)
        table = pages(seqs)
        offsets = np.cumsum(counts) - counts
        for i in range(2):
            model.write(i, table, [s.num_tokens() for s in seqs], counts, offsets, rows.x[:, i])
        check_cache(seqs)
        check_attention(seqs, counts, rows.q, out.download(np.float32).reshape(n, Hq, D))

    seqs = [v2.SequenceState(i, pool) for i in range(4)]
    prefill(seqs, [37, 1, 2 * bs, 9], 1.0)
    prefill(seqs[:2], [20, 30], 3.0)  # the next chunk, in the middle of pages
    seqs.append(seqs[0].fork_shared(10))
    seqs.append(seqs[0].fork_shared(11))
    batch = v2.DeviceBatchTable(storage, seqs, 30)
    for step in range(2 * bs + 3):
        before = pages(seqs)
        rows = Rows(v2, rng, len(seqs), Hq, H, D, name, 2.0 ** rng.integers(-2, 3))
        out = device.DeviceBuffer(len(seqs) * Hq * D * 4)
        v2.decode_step(storage, batch, rows.rows, rows.qd.ptr, out.ptr, Hq)
        table = pages(seqs)
        for r, s in enumerate(seqs):  # copies of shared tails, then the new tokens
            b = (s.num_tokens() - 1) // bs
            if b < before.shape[1] and before[r, b] != 2 ** 64 - 1 and before[r, b] != table[r, b]:
                source, to = int(before[r, b]), int(table[r, b])
                model.bytes[:, to], model.scales[:, to] = model.bytes[:, source], model.scales[:, source]
        for i in range(2):
            model.write(i, table, [s.num_tokens() for s in seqs], [1] * len(seqs), np.arange(len(seqs)), rows.x[:, i])
        check_cache(seqs)
        check_attention(seqs, [1] * len(seqs), rows.q, out.download(np.float32).reshape(len(seqs), Hq, D))
    again = device.DeviceBuffer(out.nbytes)
    v2.paged_attention_batch(storage, seqs, rows.qd.ptr, again.ptr, Hq)
    check_attention(seqs, [1] * len(seqs), rows.q, again.download(np.float32).reshape(len(seqs), Hq, D))
    v2.paged_attention_batch(storage, batch, rows.qd.ptr, again.ptr, Hq)
    assert np.array_equal(again.download(np.uint32), out.download(np.uint32))

    total = sum(s.num_tokens() for s in seqs)
    for out_name, dtype in (("bf16", v2.DType.BFloat16), ("f32", v2.DType.Float32)):
        out = [device.DeviceBuffer(total * H * D * 4) for _ in range(2)]
        v2.read_quantized_kv(storage, seqs, dtype, out[0].ptr, out[1].ptr)
        values, table = model.values(), pages(seqs)
        for i in range(2):
            want = np.concatenate([values[i, table[r, :s.num_allocated_blocks()].astype(np.int64)].transpose(0, 2, 1, 3)
                                   .reshape(-1, H, D)[:s.num_tokens()] for r, s in enumerate(seqs)])
            want = to_bits(want, out_name)
            assert np.array_equal(out[i].download(want.dtype, want.size).reshape(want.shape), want)


def test_copied_pages_bring_their_scales(gpu, v2):
    rng = np.random.default_rng(1)
    pool = v2.PhysicalBlockPool(9, 16)
    storage = v2.QuantizedKVStorage(pool, 3, 64, v2.QuantFormat.Int8)
    held = [pool.allocate() for _ in range(6)]
    layout = storage.layout()
    data = rng.integers(0, 256, layout.total_bytes()).astype(np.uint8)
    device.memcpy_h2d(storage.key_base(), data)
    model = Model(storage)
    before = model.download()
    storage.copy_blocks([(held[0], held[3]), (held[1], held[5])])
    after = model.download()
    ids = [pool.id(h) for h in held]
    for x, y in zip(before, after):
        x = x.copy()
        x[:, [ids[3], ids[5]]] = x[:, [ids[0], ids[1]]]
        assert x.tobytes() == y.tobytes()
    with pytest.raises(ValueError):
        storage.copy_blocks([(held[0], held[3]), (held[1], held[3])])


def test_refusals(gpu, v2):
    pool, other = v2.PhysicalBlockPool(20, 16), v2.PhysicalBlockPool(20, 16)
    storage = v2.QuantizedKVStorage(pool, 2, 64, v2.QuantFormat.E4M3)
    a, b = v2.SequenceState(1, pool), v2.SequenceState(2, pool)
    a.append_tokens(20)
    b.append_tokens(5)
    foreign = v2.SequenceState(3, other)
    foreign.append_tokens(4)
    buf = device.DeviceBuffer(1 << 20)
    bf16 = v2.DType.BFloat16

    def rows(key=buf.ptr, value=buf.ptr + (1 << 19), **kw):
        return v2.NewRows(key, value, bf16, **kw)

    for seqs, counts, r in [([a, b], [1], rows()), ([a, b], [21, 1], rows()), ([a, foreign], [1, 1], rows()),
                            ([a, a], [1, 1], rows()), ([a, a.fork_shared(9)], [1, 1], rows()), ([a], [1], rows(key=0)),
                            ([a], [1], rows(value=0)), ([a], [1], rows(key=buf.ptr + 1)), ([a], [1], rows(key_stride=127)),
                            ([a], [1], rows(key=storage.key_base())), ([a], [1], rows(key=0x1000)), ([None], [1], rows())]:
        with pytest.raises(ValueError):
            v2.write_quantized_kv(storage, seqs, counts, r)
    v2.write_quantized_kv(storage, [a, a], [3, 0], rows())
    v2.write_quantized_kv(storage, [a], [0], rows(key=0))
    empty = v2.SequenceState(4, pool)
    for call in (lambda: v2.paged_attention_batch(storage, [a, empty], buf.ptr, buf.ptr + 65536, 4),
                 lambda: v2.paged_attention_batch(storage, [a], buf.ptr, buf.ptr + 65536, 3),
                 lambda: v2.paged_attention_batch(storage, [a], buf.ptr, buf.ptr, 4),
                 lambda: v2.paged_attention_batch(storage, [foreign], buf.ptr, buf.ptr + 65536, 4),
                 lambda: v2.paged_attention_batch(storage, [a], 0, buf.ptr, 4),
                 lambda: v2.paged_attention_prompts(storage, [a], [21], buf.ptr, buf.ptr + 65536, 4),
                 lambda: v2.paged_attention_prompts(storage, [a], [3, 4], buf.ptr, buf.ptr + 65536, 4),
                 lambda: v2.paged_attention_prompts(storage, [a], [3], buf.ptr, storage.value_scales(), 4),
                 lambda: v2.read_quantized_kv(storage, [a], bf16, buf.ptr, buf.ptr + 256),
                 lambda: v2.read_quantized_kv(storage, [a], bf16, storage.key_scales(), buf.ptr),
                 lambda: v2.read_quantized_kv(storage, [a], bf16, 0, buf.ptr),
                 lambda: v2.DeviceBatchTable(storage, [foreign], 4),
                 lambda: v2.DeviceBatchTable(storage, [a, a], 4)):
        with pytest.raises(ValueError):
            call()
    table = v2.DeviceBatchTable(storage, [a, b], 4)
    with pytest.raises(ValueError):
        v2.decode_step(storage, table, rows(value=0), buf.ptr, buf.ptr + 65536, 4)
    with pytest.raises(ValueError):
        v2.decode_step(storage, table, rows(value_stride=5), buf.ptr, buf.ptr + 65536, 4)
    assert a.num_tokens() == 20 and b.num_tokens() == 5  # nothing was appended
    v2.paged_attention_prompts(storage, [a, b], [0, 0], 0, 0, 4)
    v2.read_quantized_kv(storage, [empty], bf16, 0, 0)
    v2.read_quantized_kv(storage, [], bf16, 0, 0)


# ------------------------------------------------------------------ graphs
def test_captured_calls(gpu):
    """The write, the attention, a prompt's write and attention and the read in one graph, replayed with
    other lengths, pages and rows between, eager work on the same workspace among them; two graphs share
    the workspaces. Every replay is the eager calls' bits."""
    rng = np.random.default_rng(2)
    H, Hq, D, bs, rows = 2, 8, 128, 16, 12
    cache = Cache("e4m3", 260, H, bs, D)
    cache.fill(rng)
    most, chunk, width = 300, 70, 19
    lens_d, table_d = device.DeviceBuffer(rows * 8), device.DeviceBuffer(rows * width * 8)
    new_d, off_d, starts_d, read_d = (device.DeviceBuffer(rows * 8) for _ in range(4))
    x = device.DeviceBuffer(rows * chunk * 2 * H * D * 2)
    q = device.DeviceBuffer(rows * chunk * Hq * D * 4)
    out = [device.DeviceBuffer(rows * chunk * Hq * D * 4) for _ in range(2)]
    read = [device.DeviceBuffer(rows * most * H * D * 2) for _ in range(2)]
    size = C.c_size_t()
    capi.call("kvflux_quant_attention_workspace_size", rows, 2048, H, Hq, bs, D, C.byref(size))
    attend_ws = device.DeviceBuffer(size.value)
    attend_bytes = size.value
    capi.call("kvflux_quant_prefill_workspace_size", rows, chunk, 8192, H, Hq, bs, D, C.byref(size))
    prompt_ws = device.DeviceBuffer(max(1, size.value))
    prompt_bytes = size.value
    assert attend_bytes > 0 and prompt_bytes > 0
    stride = 2 * H * D
    kv = (x.ptr, x.ptr + H * D * 2, capi.DTYPE_BF16, stride, stride)
    table = (table_d.ptr, width)

    def decode(s):
        capi.call("kvflux_quant_write_tail", *cache.args(), *kv, *table, lens_d.ptr, rows, s)
        capi.call("kvflux_quant_attention", *cache.args(), *table, lens_d.ptr, 2048, rows, Hq, q.ptr, out[0].ptr,
                  attend_ws.ptr, attend_bytes, s)

    def prompt(s):
        capi.call("kvflux_quant_write", *cache.args(), *kv, *table, lens_d.ptr, new_d.ptr, off_d.ptr, rows, chunk, s)
        capi.call("kvflux_quant_prefill", *cache.args(), *table, lens_d.ptr, new_d.ptr, off_d.ptr, rows, chunk, 8192, Hq,
                  q.ptr, out[1].ptr, prompt_ws.ptr, prompt_bytes, s)
        capi.call("kvflux_quant_gather", *cache.args(), *table, lens_d.ptr, read_d.ptr, starts_d.ptr, rows, rows * width,
                  read[0].ptr, read[1].ptr, capi.DTYPE_BF16, s)

    stream = device.Stream()

    def inputs(seed):
        r = np.random.default_rng(seed)
        lens = r.integers(0, most, rows)
        lens[0] = most
        new = np.minimum(r.integers(0, chunk + 1, rows), lens)
        t = np.full((rows, width), 2 ** 64 - 1, np.uint64)
        t[:, :] = r.permutation(260)[:rows * width].reshape(rows, width)
        pages = -(-lens // bs)
        for buf, v in ((lens_d, lens), (new_d, new), (off_d, np.arange(rows) * chunk), (read_d, np.arange(rows) * most), (starts_d, np.cumsum(pages) - pages),
                       (table_d, t)):
            buf.upload(np.ascontiguousarray(v).astype(np.uint64))
        x.upload(to_bits(r.standard_normal((rows * chunk, 2 * H * D)), "bf16"))
        q.upload(r.standard_normal((rows * chunk, Hq * D)).astype(np.float32))
        cache.upload()
        for o in (*out, *read):
            o.fill(0)

    def state():
        device.synchronize()
        return [o.download(np.uint8) for o in (*out, *read, *cache.dev, *cache.dev_scales)]

    inputs(0)
    graphs = Graph(stream, lambda h: (decode(h), prompt(h))), Graph(stream, decode)
    for seed in range(1, 5):
        inputs(seed)
        decode(None)
        prompt(None)
        want = state()
        inputs(seed)
        graphs[0].replay()
        assert all(np.array_equal(a, b) for a, b in zip(state(), want)), seed
        graphs[0].replay()  # the tokens are there already: the same again, but for scales that stay raised
        inputs(seed + 10)
        decode(None)
        want = state()
        inputs(seed + 10)
        graphs[1].replay()
        assert all(np.array_equal(a, b) for a, b in zip(state(), want)), seed
    for g in graphs:
        g.close()
