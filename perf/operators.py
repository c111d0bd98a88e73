"""Performance cases of the decode step's operators, through their public entry points.

Two operators of a serving program: what comes before the attention (norms of
queries and keys for each head, the position rotation, K and V into their
pages, in one pass), and the decode attention of a batch whose rows share long
prefixes. The `kind` picks the call; the other fields are the cache's shape and
the batch. Lengths, groups and positions come from the case alone (field
`lens` seeds them), so the work of a case is the same for every set of inputs;
values and page placement come from the seed. Pages are always placed at
random in the pool, as a pool that has served requests for a while has them.

Kinds
  project         kvflux_norm_rope_write: `tokens` new tokens of prompts, at
                  their positions and slots
  project_decode  kvflux_norm_rope_write_tail: one new token for each of
                  `rows` sequences, slot and position from the batch table
  shared          kvflux_paged_attention_shared: decode attention of `rows`
                  rows in `groups` groups, the rows of a group behind the
                  same prefix of lo_prefix..hi_prefix tokens (whole pages)
                  with lo..hi tokens of their own each
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE = {"f16": 0, "bf16": 1, "f32": 2}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


def _shape(dtype, q_heads, kv_heads, head_size, block_size):
    return {"dtype": dtype, "q_heads": q_heads, "kv_heads": kv_heads, "head_size": head_size,
            "block_size": block_size}


def listed():
    gqa = _shape("bf16", 32, 8, 128, 16)
    return [
        # The next token of a few interactive requests: the smallest call of
        # a serving loop, all latency.
        {"name": "project_decode_4", "kind": "project_decode", **gqa, "input": "bf16", "rows": 4, "lo": 100,
         "hi": 1500, "rotary": 128, "interleaved": False, "theta": 5e5, "lens": 1},
        # A full decode batch far into long contexts (large angles), a
        # partial rotation over neighbouring pairs, an odd group.
        {"name": "project_decode_96", "kind": "project_decode", **_shape("f16", 28, 4, 128, 32), "input": "f16",
         "rows": 96, "lo": 1000, "hi": 130000, "rotary": 64, "interleaved": True, "theta": 1e4, "lens": 2},
        # A prefill step's tokens, the ordinary shape.
        {"name": "project_4096", "kind": "project", **gqa, "input": "bf16", "tokens": 4096, "rotary": 128,
         "interleaved": False, "theta": 5e5, "lens": 3},
        # Ragged prompts, FP32 caches fed by a 16-bit model.
        {"name": "project_1111_f32", "kind": "project", **_shape("f32", 16, 4, 64, 16), "input": "bf16",
         "tokens": 1111, "rotary": 64, "interleaved": False, "theta": 1e4, "lens": 4},
        # A large prefill batch of a model with many heads.
        {"name": "project_16384", "kind": "project", **_shape("bf16", 64, 8, 128, 16), "input": "bf16",
         "tokens": 16384, "rotary": 128, "interleaved": False, "theta": 1e6, "lens": 5},
        # A few users of one assistant, just started: the smallest call.
        {"name": "shared_4x512", "kind": "shared", **gqa, "rows": 4, "groups": 1, "lo_prefix": 512,
         "hi_prefix": 512, "lo": 10, "hi": 120, "lens": 6},
        # Two agents' instructions, several conversations each; an odd group.
        {"name": "shared_17x2000", "kind": "shared", **_shape("f16", 28, 4, 128, 16), "rows": 17, "groups": 2,
         "lo_prefix": 1500, "hi_prefix": 2500, "lo": 100, "hi": 1000, "lens": 7},
        # A full batch behind one long system prompt with tools.
        {"name": "shared_64x8192", "kind": "shared", **gqa, "rows": 64, "groups": 1, "lo_prefix": 8192,
         "hi_prefix": 8192, "lo": 64, "hi": 1024, "lens": 8},
        # Many questions about one long document: the largest.
        {"name": "shared_48x60000", "kind": "shared", **_shape("bf16", 64, 8, 128, 32), "rows": 48, "groups": 1,
         "lo_prefix": 60000, "hi_prefix": 60000, "lo": 20, "hi": 300, "lens": 9},
        # Ordinary chat: many assistants, each with some conversations whose
        # own part is the longer one.
        {"name": "shared_128x12", "kind": "shared", **gqa, "rows": 128, "groups": 12, "lo_prefix": 400,
         "hi_prefix": 4000, "lo": 200, "hi": 6000, "lens": 10},
        # Parallel samples of a few prompts on FP32 caches.
        {"name": "shared_24_f32", "kind": "shared", **_shape("f32", 16, 4, 64, 16), "rows": 24, "groups": 3,
         "lo_prefix": 300, "hi_prefix": 3500, "lo": 1, "hi": 500, "lens": 11},
        # Wide heads, small pages.
        {"name": "shared_20_wide", "kind": "shared", **_shape("bf16", 16, 2, 256, 8), "rows": 20, "groups": 1,
         "lo_prefix": 5000, "hi_prefix": 5000, "lo": 50, "hi": 700, "lens": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["project", "project_decode", "shared", "shared", "shared"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    q_heads, kv_heads = rng.choice([(32, 8), (28, 4), (64, 8), (16, 4), (16, 2), (40, 8), (24, 8), (8, 8), (12, 1)])
    head_size = rng.choice([64, 128, 128, 256] if kind != "shared" or dtype != "f32" else [64, 128, 128])
    s = _shape(dtype, q_heads, kv_heads, head_size, rng.choice([8, 16, 16, 32, 64]))
    lens = rng.randrange(1 << 20)
    if kind != "shared":
        s |= {"input": rng.choice([dtype, dtype, "bf16"]), "rotary": head_size // rng.choice([1, 1, 2]),
              "interleaved": rng.random() < 0.3, "theta": rng.choice([1e4, 5e5, 1e6]), "lens": lens}
        if kind == "project_decode":
            return {"kind": kind, **s, "rows": _log_int(rng, 1, 256), "lo": 1, "hi": _log_int(rng, 16, 131072)}
        return {"kind": kind, **s, "tokens": _log_int(rng, 2, 16384 * 64 // head_size)}
    rows = _log_int(rng, 2, 128)
    groups = min(rows, _log_int(rng, 1, 12))
    token = 2 * kv_heads * head_size * BYTES[dtype]  # K and V bytes of a token
    # No more products and K/V than the largest listed cases.
    slow = 4 if dtype == "f32" else 1
    most = min(65536, int(2.0e10 / slow / (q_heads * head_size * rows)), int(4e8 / token / groups))
    hi_prefix = _log_int(rng, s["block_size"], max(s["block_size"] + 1, most))
    own_most = max(2, min(8192, int(1.2e9 / token / rows), int(2e9 / slow / (q_heads * head_size * rows))))
    hi = _log_int(rng, 1, own_most)
    return {"kind": kind, **s, "rows": rows, "groups": groups,
            "lo_prefix": max(1, hi_prefix // rng.choice([1, 2, 8])), "hi_prefix": hi_prefix,
            "lo": max(1, hi // rng.choice([1, 4, 16])), "hi": hi, "lens": lens}


# ------------------------------------------------------------------- batch
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _u64(values):
    """uint64 metadata on the GPU (as int64 tensors: the same bytes)."""
    return torch.as_tensor(np.ascontiguousarray(values).astype(np.int64), device="cuda")


def _groups(case):
    """(first row of every group and the end, prefix tokens of every group,
    tokens of every row) of a shared batch: whole pages are shared, every
    group has a row at least and every row a token of its own."""
    r = np.random.RandomState(case["lens"])
    rows, groups, bs = case["rows"], case["groups"], case["block_size"]
    starts = np.concatenate([[0], 1 + np.sort(r.permutation(rows - 1)[:groups - 1]), [rows]]).astype(np.int64)
    prefix = r.randint(case["lo_prefix"], case["hi_prefix"] + 1, groups) // bs * bs
    own_tokens = r.randint(case["lo"], case["hi"] + 1, rows)
    return starts, prefix.astype(np.int64), (np.repeat(prefix, np.diff(starts)) + own_tokens).astype(np.int64)


def _tables(lengths, block_size, seed, shared=None):
    """Random pages for every sequence: (table [rows][width], pages of the
    pool). `shared`: (first rows of the groups, prefix tokens of each)."""
    counts = -(-lengths // block_size)
    starts, prefix = shared if shared is not None else (np.arange(len(lengths) + 1), np.zeros(len(lengths), np.int64))
    width = int(counts.max())
    common = np.repeat(prefix // block_size, np.diff(starts))
    used = int((counts - common).sum() + (prefix // block_size).sum())
    pool = used + max(8, used // 16)  # a few pages belong to nobody
    order = np.random.RandomState(seed & 0x7fffffff).permutation(pool)
    table = np.full((len(lengths), width), -1, np.int64)
    at = 0
    for g, p in enumerate(prefix // block_size):
        table[starts[g]:starts[g + 1], :p] = order[at:at + p]
        at += p
    for r, (c, n) in enumerate(zip(common, counts)):
        table[r, c:n] = order[at:at + n - c]
        at += n - c
    return table, pool


def _positions(case):
    """Position of every new token: consecutive ones of a few prompts, or the
    last one of every row."""
    r = np.random.RandomState(case["lens"])
    if case["kind"] == "project_decode":
        return r.randint(case["lo"], case["hi"] + 1, case["rows"]).astype(np.int64) - 1
    tokens, prompts = case["tokens"], min(case["tokens"], 5)
    cuts = np.concatenate([[0], 1 + np.sort(r.permutation(tokens - 1)[:prompts - 1]), [tokens]])
    first = r.randint(0, 30000, prompts)  # some continue a cached prefix
    return np.concatenate([first[i] + np.arange(cuts[i + 1] - cuts[i]) for i in range(prompts)]).astype(np.int64)


def _inputs(case, seed):
    """The inputs of a case as tensors, without any of this package's code."""
    g = _generator(seed)
    H, Hq, D, bs = case["kv_heads"], case["q_heads"], case["head_size"], case["block_size"]
    dt = TORCH[case["dtype"]]
    if case["kind"] == "shared":
        starts, prefix, lengths = _groups(case)
        table, pool = _tables(lengths, bs, seed, (starts, prefix))
        k, v = (_normal(g, (pool, H, bs, D), dt) for _ in range(2))
        return {"k": k, "v": v, "q": _normal(g, (case["rows"], Hq, D), torch.float32), "table": _u64(table),
                "lens": _u64(lengths), "starts": _u64(starts), "prefix": _u64(prefix)}
    positions = _positions(case)
    n = len(positions)
    x = {"positions": _u64(positions)}
    if case["kind"] == "project_decode":
        # The pages before the last are not read: rows share one page there.
        width = int(positions.max()) // bs + 1
        pool = n + max(8, n // 8)
        order = np.random.RandomState(seed & 0x7fffffff).permutation(pool)
        table = np.full((n, width), order[n], np.int64)
        table[np.arange(n), positions // bs] = order[:n]
        x |= {"table": _u64(table), "lens": _u64(positions + 1)}
        slots = order[:n] * bs + positions % bs
    else:
        table, pool = _tables(np.array([n]), bs, seed)
        slots = table[0][np.arange(n) // bs] * bs + np.arange(n) % bs
    x["slots"] = _u64(slots)
    x["k"], x["v"] = (_normal(g, (pool, H, bs, D), dt) for _ in range(2))
    # What the projection gives: the heads of Q, K and V side by side.
    x["qkv"] = _normal(g, (n, Hq + 2 * H, D), torch.float32).mul_(1.7).to(TORCH[case["input"]])
    x["q_norm"], x["k_norm"] = (1.0 + 0.2 * _normal(g, (D,), torch.float32) for _ in range(2))
    rotary = case["rotary"]
    x["inv_freq"] = torch.as_tensor(case["theta"] ** (-np.arange(0, rotary, 2) / rotary), device="cuda")
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, "x": x}
    rows = x["q"].shape[0] if case["kind"] == "shared" else x["positions"].shape[0]
    s["out"] = torch.empty((rows, case["q_heads"], case["head_size"]), dtype=torch.float32, device="cuda")
    if case["kind"] == "shared":
        # How the plain form lays the rows out: [groups][rows of the largest].
        starts, prefix, lengths = _groups(case)
        counts = np.diff(starts)
        at = np.minimum(starts[:-1, None] + np.arange(counts.max())[None, :], case["rows"] - 1)
        group = np.repeat(np.arange(len(counts)), counts)
        s["row_of"] = _u64(at)
        s["place"] = _u64(group * counts.max() + np.arange(case["rows"]) - starts[group])
        s["group"] = _u64(group)
        s["longest"] = (int(prefix.max()), int((lengths - prefix[group]).max()), int(lengths.max()))
    if own:
        s["call"] = _call(case, s)
    return s


def _call(case, s):
    """The framework's call, its workspace with it."""
    import ctypes as C

    from kvflux_amd import capi

    x, H, Hq, D, bs = s["x"], case["kv_heads"], case["q_heads"], case["head_size"], case["block_size"]
    cache = (x["k"].data_ptr(), x["v"].data_ptr(), x["k"].shape[0], H, bs, D, CODE[case["dtype"]])
    if case["kind"] == "shared":
        rows, width = x["table"].shape
        longest_prefix, _, longest = s["longest"]
        size = C.c_size_t()
        capi.call("kvflux_paged_attention_shared_workspace_size", rows, longest, H, Hq, bs, D, CODE[case["dtype"]],
                  case["groups"], C.byref(size))
        s["workspace"] = torch.empty(max(1, size.value), dtype=torch.uint8, device="cuda")
        return ("kvflux_paged_attention_shared", *cache, x["table"].data_ptr(), width, x["lens"].data_ptr(), longest,
                rows, Hq, x["starts"].data_ptr(), x["prefix"].data_ptr(), case["groups"], longest_prefix,
                x["q"].data_ptr(), s["out"].data_ptr(), s["workspace"].data_ptr(), size.value, None)
    n, code = x["qkv"].shape[0], CODE[case["input"]]
    stride = (Hq + 2 * H) * D
    first = x["qkv"].data_ptr()
    head = D * BYTES[case["input"]]
    rows = (first, first + Hq * head, first + (Hq + H) * head, code, stride, stride, stride, Hq)
    form = (x["q_norm"].data_ptr(), x["k_norm"].data_ptr(), EPS, x["inv_freq"].data_ptr(), case["rotary"],
            int(case["interleaved"]))
    if case["kind"] == "project_decode":
        return ("kvflux_norm_rope_write_tail", *cache, *rows, *form, x["table"].data_ptr(), x["table"].shape[1],
                x["lens"].data_ptr(), n, s["out"].data_ptr(), None)
    return ("kvflux_norm_rope_write", *cache, *rows, *form, x["positions"].data_ptr(), x["slots"].data_ptr(), n,
            s["out"].data_ptr(), None)


# --------------------------------------------------------------------- run
def _plain_project(case, s):
    x, Hq, H, D, rotary = s["x"], case["q_heads"], case["kv_heads"], case["head_size"], case["rotary"]
    qkv = x["qkv"].float()
    bs = case["block_size"]
    if case["kind"] == "project_decode":
        positions = x["lens"] - 1
        page = x["table"].gather(1, (positions // bs)[:, None])[:, 0]
    else:
        positions = x["positions"]
        page = x["slots"] // bs
    offset = positions % bs if case["kind"] == "project_decode" else x["slots"] % bs
    qk = qkv[:, :Hq + H]
    weight = torch.cat([x["q_norm"].expand(Hq, D), x["k_norm"].expand(H, D)])
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * weight
    angle = positions.double()[:, None] * x["inv_freq"]
    c, n = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    rot = qk[..., :rotary]
    if case["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = rot[..., :rotary // 2], rot[..., rotary // 2:]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    qk = torch.cat([turned, qk[..., rotary:]], -1)
    x["k"][page, :, offset] = qk[:, Hq:].to(x["k"].dtype)
    x["v"][page, :, offset] = qkv[:, Hq + H:].to(x["v"].dtype)
    return [qk[:, :Hq].contiguous(), x["k"], x["v"]]


def _pages(cache, table, tokens, bs):
    """[rows][H][tokens][D] in 32 bits of the first `tokens` tokens of a table's rows."""
    got = cache[table[:, :-(-tokens // bs)].clamp(min=0)]  # [rows][pages][H][bs][D]
    return got.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :tokens].float()


def _plain_shared(case, s):
    """The prefix once for a group's rows, each row's own tokens, one softmax over both."""
    x, H, Hq, D, bs = s["x"], case["kv_heads"], case["q_heads"], case["head_size"], case["block_size"]
    rows, G = case["rows"], Hq // H
    longest_prefix, longest_own, _ = s["longest"]
    prefix, row_of, place, group = x["prefix"], s["row_of"], s["place"], s["group"]
    groups, most = row_of.shape
    q = x["q"].view(rows, H, G, D) / math.sqrt(D)
    scores, sums, tops = [], [], []
    # prefix part: [groups][H][tokens][rows of the group * G]
    if longest_prefix:
        qg = q[row_of.flatten()].view(groups, most, H, G, D).permute(0, 2, 4, 1, 3).reshape(groups, H, D, most * G)
        k = _pages(x["k"], x["table"][x["starts"][:-1]], longest_prefix, bs)
        w = torch.matmul(k, qg.contiguous())
        dead = torch.arange(longest_prefix, device=w.device)[None, :] >= prefix[:, None]
        w.masked_fill_(dead[:, None, :, None], float("-inf"))
        top = w.amax(2, keepdim=True).clamp(min=-3e38)
        w = torch.exp(w - top)
        v = _pages(x["v"], x["table"][x["starts"][:-1]], longest_prefix, bs)
        o = torch.matmul(w.transpose(2, 3).contiguous(), v)  # [groups][H][most * G][D]
        back = lambda t: t.reshape(groups, H, most, G, -1).transpose(1, 2).reshape(groups * most, H, G, -1)[place]  # noqa: E731
        scores.append(back(o))
        sums.append(back(w.sum(2)))
        tops.append(back(top[:, :, 0]))
    # own part: [rows][H][tokens][G], row r's table moved up by its prefix
    at = (prefix[group] // bs)[:, None] + torch.arange(-(-longest_own // bs), device=q.device)[None, :]
    table = x["table"].gather(1, at.clamp(max=x["table"].shape[1] - 1))
    k = _pages(x["k"], table, longest_own, bs)
    w = torch.matmul(k, q.transpose(2, 3).contiguous())
    dead = torch.arange(longest_own, device=w.device)[None, :] >= (x["lens"] - prefix[group])[:, None]
    w.masked_fill_(dead[:, None, :, None], float("-inf"))
    top = w.amax(2, keepdim=True)
    w = torch.exp(w - top)
    v = _pages(x["v"], table, longest_own, bs)
    scores.append(torch.matmul(w.transpose(2, 3).contiguous(), v))
    sums.append(w.sum(2)[..., None])
    tops.append(top[:, :, 0][..., None])
    scores, sums, tops = torch.stack(scores), torch.stack(sums), torch.stack(tops)
    f = torch.exp(tops - tops.amax(0))
    return [((scores * f).sum(0) / (sums * f).sum(0)).reshape(rows, Hq, D)]


def run(state):
    case = state["case"]
    if own:
        from kvflux_amd import capi

        name, *args = state["call"]
        capi.call(name, *args)
        return [state["out"]] + ([] if case["kind"] == "shared" else [state["x"]["k"], state["x"]["v"]])
    return _plain_shared(case, state) if case["kind"] == "shared" else _plain_project(case, state)


# -------------------------------------------------------------------- work
def work(case):
    H, Hq, D = case["kv_heads"], case["q_heads"], case["head_size"]
    token = 2 * H * D * BYTES[case["dtype"]]
    if case["kind"] == "shared":
        starts, prefix, lengths = _groups(case)
        unique = int(prefix.sum() + (lengths - np.repeat(prefix, np.diff(starts))).sum())
        return {"bytes": unique * token + unique // case["block_size"] * 8 + 8 * case["rows"] * Hq * D,
                "flops": 4 * Hq * D * int(lengths.sum())}
    n = case["rows"] if case["kind"] == "project_decode" else case["tokens"]
    rows = n * (Hq + 2 * H) * D * BYTES[case["input"]] + n * Hq * D * 4 + n * token + 16 * n
    # A norm is 4 operations a value, a rotation 3, of queries and keys.
    return {"bytes": rows + 8 * D + 4 * case["rotary"], "flops": n * (Hq + H) * (4 * D + 3 * case["rotary"])}


# ------------------------------------------------------------------- exact
def _exact_project(case, x):
    Hq, H, D, bs, half = (case[k] for k in ("q_heads", "kv_heads", "head_size", "block_size", "rotary"))
    half //= 2
    qkv = x["qkv"].double()
    weights = [x["q_norm"].double()] * Hq + [x["k_norm"].double()] * H
    y = qkv.clone()
    first = [2 * j if case["interleaved"] else j for j in range(half)]
    second = [2 * j + 1 if case["interleaved"] else j + half for j in range(half)]
    angle = torch.outer(x["positions"].double(), x["inv_freq"])
    c, n = torch.cos(angle), torch.sin(angle)
    for h, w in enumerate(weights):
        t = qkv[:, h]
        t = t / torch.sqrt(t.square().sum(-1, keepdim=True) / D + EPS) * w
        y[:, h] = t
        y[:, h, first] = t[:, first] * c - t[:, second] * n
        y[:, h, second] = t[:, first] * n + t[:, second] * c
    k, v = x["k"].double(), x["v"].double()
    page, offset = x["slots"] // bs, x["slots"] % bs
    for h in range(H):
        k[page, h, offset], v[page, h, offset] = y[:, Hq + h], y[:, Hq + H + h]
    return [y[:, :Hq].contiguous(), k, v]


def _exact_shared(case, x):
    H, Hq, D, bs = case["kv_heads"], case["q_heads"], case["head_size"], case["block_size"]
    out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    for r, n in enumerate(x["lens"].tolist()):
        pages = x["table"][r, :-(-n // bs)]
        for h in range(H):
            k, v = (x[c][pages, h].reshape(-1, D)[:n].double() for c in ("k", "v"))
            q = x["q"][r, h * (Hq // H):(h + 1) * (Hq // H)].double()
            w = torch.softmax((k @ q.t().contiguous()).t().contiguous() / math.sqrt(D), -1)
            out[r, h * (Hq // H):(h + 1) * (Hq // H)] = w @ v
    return [out]


def exact(case, seed):
    x = _inputs(case, seed)
    return _exact_shared(case, x) if case["kind"] == "shared" else _exact_project(case, x)
