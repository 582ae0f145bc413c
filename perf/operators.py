"""Attention over a paged cache, attention over selected pages and low-rank adapters: the calls a
serving program makes of them, in their plain form (elementary torch operations) and through
models_amd.attention, with the sizes it makes them at.

Three kinds of case:

* ``paged``    a layer's new tokens of many sessions in one call: RoPE, append to the pages, causal
               attention of every new token over its session's pages;
* ``sparse``   the same, each new token and KV head attending only to the pages whose bounds promise
               the largest scores, besides the first and the last ones;
* ``adapters`` each request's low-rank adapter added to a projection that all requests share.

A page of P slots of one KV head is stored as P / 32 tiles of 32 slots: keys as column panels
[head length / W][32][W] of 64 bytes a row, values transposed [head length][32].

Lengths, rows and ranks of a case come from its ``mix`` number, so that they are the case's and not
the seed's.
"""

import math

import numpy as np
import torch

own = False

TILE = 32
NO_ADAPTER = 0xFFFFFFFF
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _shape(heads, kv_heads, dim, neox, theta, half=True):
    return {"heads": heads, "kv_heads": kv_heads, "dim": dim, "neox": neox, "theta": theta, "half": half}


# Head layouts and RoPE bases of the models that this repository's tests and benchmark use, and one
# generic one of 32 query heads over 8 KV heads of 128.
SHAPES = {
    "32x8x64": _shape(32, 8, 64, False, 5e5),
    "12x2x128": _shape(12, 2, 128, True, 1e6),
    "32x8x128": _shape(32, 8, 128, True, 5e5),
    "16x8x128_f32": _shape(16, 8, 128, True, 1e6, half=False),
    "4x1x256": _shape(4, 1, 256, True, 1e6),
}


def _paged(shape, page, sequences, low, high, rows_low, rows_high, long=0, long_rows=0, window=0, mix=1):
    return {"kind": "paged", "shape": shape, "page": page, "sequences": sequences, "low": low, "high": high,
            "rows_low": rows_low, "rows_high": rows_high, "long": long, "long_rows": long_rows,
            "window": window, "top": 0, "first": 0, "last": 0, "mix": mix}


def _sparse(shape, page, sequences, low, high, rows_low, rows_high, top, first, last, mix=1):
    return dict(_paged(shape, page, sequences, low, high, rows_low, rows_high, mix=mix), kind="sparse",
                top=top, first=first, last=last)


def _adapters(dtype, cols, outs, runs, rows_low, rows_high, slots, rank_low, rank_high, without=0, mix=1):
    return {"kind": "adapters", "dtype": dtype, "cols": cols, "outs": outs, "runs": runs, "rows_low": rows_low,
            "rows_high": rows_high, "slots": slots, "rank_low": rank_low, "rank_high": rank_high,
            "without": without, "mix": mix}


def listed():
    return [
        # One token of one short conversation: the smallest call, all latency.
        dict(_paged("32x8x64", 32, 1, 700, 700, 1, 1), name="paged_token"),
        # A serving batch: one token each of 64 sessions of 256 to 12000 positions.
        dict(_paged("12x2x128", 64, 64, 256, 12000, 1, 1, mix=2), name="paged_batch_64"),
        # A step that mixes prompts with generation: 18 sessions verify 1 to 5 drafted tokens while
        # two prompts bring 301 tokens each.
        dict(_paged("32x8x64", 32, 20, 100, 4000, 1, 5, 2, 301, mix=3), name="paged_mixed"),
        # A 2k-token chunk of a long prompt after 6001 cached positions: compute bound.
        dict(_paged("32x8x128", 64, 1, 6001, 6001, 2048, 2048), name="paged_chunk_2k"),
        # A 1000-token chunk in a sliding-window layer with heads of 256.
        dict(_paged("4x1x256", 32, 1, 3001, 3001, 1000, 1000, window=512), name="paged_window"),
        # An f32 cache: 12 sessions' tokens and one 200-token prompt chunk.
        dict(_paged("16x8x128_f32", 32, 13, 50, 3000, 1, 1, 1, 200, mix=4), name="paged_f32"),
        # One token of a 100k-position document, 64 of its 1563 pages.
        dict(_sparse("32x8x64", 64, 1, 100001, 100001, 1, 1, 56, 1, 7), name="sparse_token_100k"),
        # A batch of 32 long conversations, one token each.
        dict(_sparse("32x8x128", 64, 32, 4000, 32000, 1, 1, 28, 1, 3, mix=5), name="sparse_batch_32"),
        # The last 61 tokens of a prompt, each with pages of its own, after 20000 positions.
        dict(_sparse("12x2x128", 32, 1, 20011, 20011, 61, 61, 52, 2, 10), name="sparse_rows_61"),
        # One token of one request with an adapter.
        dict(_adapters("f16", 2048, 2048, 1, 1, 1, 4, 16, 16), name="adapters_token"),
        # A serving batch: 64 requests, 40 adapters of ranks 8 to 64, six requests without one.
        dict(_adapters("bf16", 2048, 2560, 64, 1, 1, 40, 8, 64, without=6, mix=6), name="adapters_batch_64"),
        # Three prompts of up to 900 tokens, each with an adapter of its own.
        dict(_adapters("f16", 4096, 4096, 3, 500, 900, 3, 16, 64, mix=7), name="adapters_prompts"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("paged", "paged", "paged", "sparse", "sparse", "adapters", "adapters"))
    mix = rng.randint(10, 1 << 30)
    if kind == "adapters":
        runs = _log_int(rng, 1, 80)
        rows = _log_int(rng, 1, max(1, 1800 // runs))
        low = rng.randint(1, 32)
        return _adapters(rng.choice(("f16", "bf16", "f32")), 8 * _log_int(rng, 32, 512), _log_int(rng, 100, 4096),
                         runs, 1, rows, rng.randint(1, 48), low, rng.randint(low, 64),
                         without=rng.randint(0, runs // 4), mix=mix)
    shape = rng.choice(sorted(SHAPES))
    page = rng.choice((32, 64, 128))
    if kind == "sparse":
        sequences = _log_int(rng, 1, 24)
        high = _log_int(rng, 200, 120000 // sequences + 2000)
        return _sparse(shape, page, sequences, rng.randint(0, high), high, 1,
                       1 if sequences > 4 else _log_int(rng, 1, 24), rng.randint(1, 40), rng.randint(0, 2),
                       rng.randint(1, 6), mix=mix)
    style = rng.choice(("batch", "mixed", "chunk"))
    window = 512 if rng.random() < 0.25 else 0
    if style == "chunk":
        rows = _log_int(rng, 2, 1200)
        start = rng.choice((0, _log_int(rng, 1, 6000)))
        return _paged(shape, page, 1, start, start, rows, rows, window=window, mix=mix)
    sequences = _log_int(rng, 2, 64)
    high = _log_int(rng, 50, 200000 // sequences)
    if style == "mixed":
        sequences, high = min(sequences, 16), min(high, 4000)
        return _paged(shape, page, sequences, 0, high, 1, 5, rng.randint(1, 2), _log_int(rng, 20, 300), window, mix)
    return _paged(shape, page, sequences, 0, min(high, 14000), 1, 1, window=window, mix=mix)


# ---------------------------------------------------------------- what a case holds

def _chunks(case):
    """(sequence, first position, new rows) of each chunk of the call."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    n = case["sequences"]
    start = r.randint(case["low"], case["high"] + 1, n)
    rows = r.randint(case["rows_low"], case["rows_high"] + 1, n)
    rows[:case["long"]] = case["long_rows"]
    order = r.permutation(n)  # sessions in the order their requests came
    return np.stack([order, start, rows], 1).astype(np.uint32)


def _reservations(chunks, page):
    """The sessions' growth, as (sequence, length) calls: eight pages at a time in turn, so that a
    session's pages lie among the others'."""
    ends = {int(s): int(a + n) for s, a, n in chunks}
    calls = []
    step = 8 * page
    for at in range(step, max(ends.values()) + step, step):
        for s in sorted(ends):
            if at - step < ends[s]:
                calls.append((s, min(at, ends[s])))
    return calls


def _tables(calls, page):
    """Page lists of the sessions after those calls: the lowest free page each time."""
    tables, used = {}, 0
    for s, length in calls:
        t = tables.setdefault(s, [])
        while len(t) * page < length:
            t.append(used)
            used += 1
    return tables, used


def _runs(case):
    """(adapter or NO_ADAPTER, rows) of each run, and each adapter's rank and scale."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    slot = r.randint(0, case["slots"], case["runs"]).astype(np.uint32)
    slot[r.permutation(case["runs"])[:case["without"]]] = NO_ADAPTER
    rows = r.randint(case["rows_low"], case["rows_high"] + 1, case["runs"]).astype(np.uint32)
    rank = r.randint(case["rank_low"], case["rank_high"] + 1, case["slots"])
    return np.stack([slot, rows], 1).copy(), rank, 2.0 * 16.0 / rank


class State:
    """Inputs, outputs and handles of one case."""

    def __init__(self, **fields):
        self.__dict__.update(fields)


class _Open:
    """A library handle, closed once neither its state nor a view of its memory is left."""

    def __init__(self, handle):
        self.handle = handle

    def __del__(self):
        self.handle.close()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _angles(shape, positions):
    """cos and sin of every position and pair: angles in 32 bits, as the models define them."""
    d = shape["dim"]
    freq = torch.tensor([1.0 / shape["theta"] ** (2 * i / d) for i in range(d // 2)],
                        dtype=torch.float64).float().cuda()
    angle = (torch.arange(positions, device="cuda").float()[:, None] * freq).double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _keys_of(pool):
    """[..., tiles, panels, 32, W] -> [..., slots, d]"""
    x = pool.transpose(-3, -2)
    return x.reshape(*x.shape[:-4], -1, x.shape[-2] * x.shape[-1])


def _values_of(pool):
    """[..., tiles, d, 32] -> [..., slots, d]"""
    x = pool.transpose(-2, -1)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])


def _cache_inputs(case, seed):
    """The pages as the earlier steps of these sessions left them, and the new rows."""
    shape, page = SHAPES[case["shape"]], case["page"]
    hq, hkv, d, half = (shape[k] for k in ("heads", "kv_heads", "dim", "half"))
    chunks = _chunks(case)
    calls = _reservations(chunks, page)
    tables, pages = _tables(calls, page)
    g = _gen(seed)
    t, w = page // TILE, 32 if half else 16
    kv = torch.float16 if half else torch.float32
    k = _randn(g, pages, hkv, t, d // w, TILE, w).to(kv)
    # keys differ from page to page, as those of a text do
    k += (0.5 * _randn(g, pages, hkv, 1, d // w, 1, w)).to(kv)
    v = _randn(g, pages, hkv, t, d, TILE).to(kv)
    rows = int(chunks[:, 2].sum())
    new = tuple(_randn(g, rows, h * d) for h in (hq, hkv, hkv))
    bounds = None
    if case["top"]:
        # of the slots that are filled; nothing asks for those of a session's last page
        bounds = torch.stack([_keys_of(k).amin(-2), _keys_of(k).amax(-2)], -2)
    return chunks, calls, tables, k, v, bounds, new


def _indices(case, chunks, tables):
    """Where each row and each chunk is: what an elementary form indexes with."""
    page = case["page"]
    n = chunks.shape[0]
    rows = chunks[:, 2].astype(np.int64)
    row0 = np.cumsum(rows) - rows
    chunk_of = np.repeat(np.arange(n), rows)
    inside = np.arange(rows.sum()) - row0[chunk_of]
    pos = chunks[chunk_of, 1].astype(np.int64) + inside
    width = max(len(tables[int(s)]) for s in chunks[:, 0])
    table = np.zeros((n, width), np.int64)
    for i, s in enumerate(chunks[:, 0]):
        table[i, :len(tables[int(s)])] = tables[int(s)]
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    padded = np.minimum(row0[:, None] + np.arange(max(rows.max(), 1))[None, :], rows.sum() - 1)
    return {"table": put(table), "chunk_of": put(chunk_of), "inside": put(inside), "pos": put(pos),
            "padded": put(padded), "page_of": put(table[chunk_of, pos // page])}


_program = {}


def _library():
    """One library context, as a program holds it."""
    if "lib" not in _program:
        from models_amd import attention
        _program["A"] = attention
        _program["lib"] = attention.HipAttentionLibrary(0)
    return _program["A"], _program["lib"]


def _rope(shape, positions):
    """A model's RoPE table, kept for as long as the program runs."""
    positions = -(-positions // 4096) * 4096
    key = (shape["dim"], shape["theta"], positions)
    if key not in _program:
        _program[key] = _library()[1].rotary_table(shape["dim"], shape["theta"], 1.0, max_positions=positions)
    return _program[key]


class _Memory:
    """A handle's device memory, for torch to see."""

    def __init__(self, ptr, like):
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(like.shape), "version": 2,
                                         "typestr": "<f2" if like.dtype == torch.float16 else "<f4"}


def _pages_in_library(case, chunks, calls, tables, k, v, bounds):
    """A paged cache that holds those pages, and torch's view of its memory."""
    lib = _library()[1]
    shape = SHAPES[case["shape"]]
    length = int((chunks[:, 1] + chunks[:, 2]).max())
    kv = lib.paged_kv_cache(1, length, k.shape[0], case["page"], shape["kv_heads"], shape["dim"],
                            half_precision=shape["half"], sequences=case["sequences"],
                            page_bounds=bounds is not None)
    for s, upto in calls:
        kv.reserve(s, upto)
    if any(kv.pages(s).tolist() != t for s, t in tables.items()):
        raise RuntimeError("the sessions' pages are not the lowest free ones")
    memory, opened = kv.storage(0), _Open(kv)
    views = [torch.as_tensor(_Memory(ptr, x), device="cuda").copy_(x)
             for ptr, x in zip((memory.keys, memory.values, memory.bounds), (k, v, bounds)) if x is not None]
    for view in views:
        view.opened = opened  # returned as outputs, the views may be all that is left of the state
    for s, start, _ in chunks:
        kv.set_length(0, int(s), int(start))  # the positions that the copied pages hold
    return opened, views


def prepare(case, seed):
    state = _prepare_adapters(case, seed) if case["kind"] == "adapters" else _prepare_pages(case, seed)
    torch.cuda.synchronize()
    return state


def _prepare_pages(case, seed):
    shape = SHAPES[case["shape"]]
    chunks, calls, tables, k, v, bounds, (q, kn, vn) = _cache_inputs(case, seed)
    length = int((chunks[:, 1] + chunks[:, 2]).max())
    out = torch.empty_like(q)
    budget = case["top"] + case["first"] + case["last"]
    chosen = torch.empty(q.shape[0], shape["kv_heads"], budget, dtype=torch.int32, device="cuda") if case["top"] else None
    state = State(kind=case["kind"], case=case, q=q, k=kn, v=vn, out=out, chosen=chosen)
    if own:
        A = _library()[0]
        state.opened, state.pools = _pages_in_library(case, chunks, calls, tables, k, v, bounds)
        state.layer = A.AttentionLayer(0, shape["heads"], case["window"], shape["neox"], rope=_rope(shape, length))
        state.chunks = chunks
        state.selection = A.PageSelection(case["top"], case["first"], case["last"]) if case["top"] else None
    else:
        state.pools = [x for x in (k, v, bounds) if x is not None]
        state.at = _indices(case, chunks, tables)
        state.angles = _angles(shape, length)
    return state


def _adapter_inputs(case, seed):
    runs, rank, scale = _runs(case)
    g = _gen(seed)
    r, cols, outs, slots = int(rank.max()), case["cols"], case["outs"], case["slots"]
    keep = (torch.arange(r, device="cuda")[None, :] < torch.from_numpy(rank).cuda()[:, None]).float()
    a = (_randn(g, slots, r, cols) * (keep[:, :, None] / math.sqrt(cols))).to(_TYPES[case["dtype"]])
    b = (_randn(g, slots, outs, r) * (keep[:, None, :] * 0.1)).to(_TYPES[case["dtype"]])
    rows = int(runs[:, 1].sum())
    return runs, rank, scale, a, b, _randn(g, rows, cols), _randn(g, rows, outs)


def _prepare_adapters(case, seed):
    runs, rank, scale, a, b, x, base = _adapter_inputs(case, seed)
    state = State(kind="adapters", x=x, base=base, out=torch.empty_like(base))
    if own:
        A, lib = _library()
        dtype = {"f16": A.ADAPTER_F16, "bf16": A.ADAPTER_BF16, "f32": A.ADAPTER_F32}[case["dtype"]]
        adapters = lib.adapters(case["slots"], case["cols"], case["outs"], int(rank.max()), dtype)
        state.opened = _Open(adapters)
        for s in range(case["slots"]):
            n = int(rank[s])
            sa, sb = a[s, :n].contiguous(), b[s, :, :n].contiguous()
            torch.cuda.synchronize()
            adapters.load_device(s, n, sa.data_ptr(), sa.numel(), sb.data_ptr(), sb.numel(), float(scale[s]))
            lib.synchronize()
        state.runs = runs
    else:
        n = runs[:, 1].astype(np.int64)
        row0 = np.cumsum(n) - n
        held = runs[:, 0] != NO_ADAPTER
        padded = row0[:, None] + np.arange(n.max())[None, :]
        valid = (np.arange(n.max())[None, :] < n[:, None]) & held[:, None]
        put = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()  # noqa: E731
        state.a, state.b = a, b
        state.padded, state.valid = put(np.minimum(padded, n.sum() - 1)), put(valid)
        state.slot = put(np.where(held, runs[:, 0], 0).astype(np.int64))
        state.scale = torch.from_numpy(scale).float().cuda()
    return state


# ---------------------------------------------------------------- run

def run(s):
    if s.kind == "adapters":
        if own:
            s.opened.handle.apply_device(s.runs, s.x.data_ptr(), s.x.numel(), s.base.data_ptr(),
                                         s.out.data_ptr(), s.out.numel())
            return s.out
        return _plain_adapters(s)
    if own:
        s.opened.handle.forward_device(s.layer, s.chunks, s.q.data_ptr(), s.q.numel(), s.k.data_ptr(), s.k.numel(),
                                       s.v.data_ptr(), s.v.numel(), s.out.data_ptr(), s.out.numel(), s.selection,
                                       s.chosen.data_ptr() if s.chosen is not None else 0,
                                       s.chosen.numel() if s.chosen is not None else 0)
        return [s.out] + ([s.chosen] if s.chosen is not None else []) + s.pools
    return _plain_pages(s)


def _plain_adapters(s):
    x = s.x[s.padded]  # [runs, rows, cols]
    down = torch.bmm(x, s.a[s.slot].float().transpose(1, 2).contiguous())
    up = torch.bmm(down * s.scale[s.slot][:, None, None], s.b[s.slot].float().transpose(1, 2).contiguous())
    s.out.copy_(s.base)
    s.out.index_add_(0, s.padded[s.valid], up[s.valid])
    return s.out


def _rotated(x, pos, angles, neox):
    """RoPE of x [rows, heads, d] in 32 bits, each product and sum rounded."""
    d = x.shape[-1]
    c, sn = (t[pos][:, None, :] for t in angles)
    a, b = (x[..., :d // 2], x[..., d // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, v = a * c - b * sn, a * sn + b * c
    return torch.cat([u, v], -1) if neox else torch.stack([u, v], -1).flatten(-2)


def _plain_pages(s):
    case, at = s.case, s.at
    shape, page = SHAPES[case["shape"]], case["page"]
    hq, hkv, d, neox = (shape[k] for k in ("heads", "kv_heads", "dim", "neox"))
    keys, values = s.pools[:2]
    rows, pos = s.q.shape[0], at["pos"]
    q = _rotated(s.q.reshape(rows, hq, d), pos, s.angles, neox)
    k = _rotated(s.k.reshape(rows, hkv, d), pos, s.angles, neox).to(keys.dtype)
    v = s.v.reshape(rows, hkv, d).to(values.dtype)
    slot = pos % page
    p, t, i = at["page_of"], slot // TILE, slot % TILE
    w = keys.shape[-1]
    keys[p, :, t, :, i, :] = k.reshape(rows, hkv, d // w, w)
    values[p, :, t, :, i] = v
    if case["top"]:
        return _plain_sparse(s, q)
    # Each chunk's pages side by side, and its rows padded to the longest chunk's.
    ck = _keys_of(keys[at["table"]]).transpose(1, 2).reshape(len(at["table"]), hkv, -1, d).float()
    cv = _values_of(values[at["table"]]).transpose(1, 2).reshape(len(at["table"]), hkv, -1, d).float()
    padded = at["padded"]
    n, longest = padded.shape
    cq = q[padded].reshape(n, longest, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(cq.reshape(n, hkv, -1, d), ck.transpose(2, 3).contiguous()) * float(np.float32(1 / math.sqrt(d)))
    there = torch.arange(ck.shape[2], device="cuda")[None, None, :]
    mine = pos[padded][:, :, None]
    seen = there <= mine
    if case["window"]:
        seen = seen & (there > mine - case["window"])
    scores = scores.reshape(n, hkv, hq // hkv, longest, -1).masked_fill_(~seen[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1)
    y = torch.matmul(scores.reshape(n, hkv, -1, scores.shape[-1]), cv).reshape(n, hkv, hq // hkv, longest, d)
    y = (y / total[..., None]).permute(0, 3, 1, 2, 4).reshape(n, longest, hq * d)
    s.out.copy_(y[at["chunk_of"], at["inside"]])
    return [s.out] + s.pools


def _plain_sparse(s, q):
    case, at = s.case, s.at
    shape, page = SHAPES[case["shape"]], case["page"]
    hq, hkv, d = (shape[k] for k in ("heads", "kv_heads", "dim"))
    keys, values, bounds = s.pools
    rows, pos, grp = s.q.shape[0], at["pos"], hq // hkv
    # The bounds of the pages that were written, over their filled slots.
    mine = torch.zeros(keys.shape[0], dtype=torch.long, device="cuda")
    mine.scatter_reduce_(0, at["page_of"], pos % page, "amax", include_self=True)
    written = torch.zeros(keys.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, at["page_of"], True)
    k = _keys_of(keys)
    hidden = (torch.arange(page, device="cuda")[None, :] > mine[:, None])[:, None, :, None]
    fresh = torch.stack([k.masked_fill(hidden, math.inf).amin(-2), k.masked_fill(hidden, -math.inf).amax(-2)], -2)
    bounds.copy_(torch.where(written[:, None, None, None], fresh, bounds))
    # Each page's largest possible score of any of the group's heads, in 64 bits: what is next to the
    # border of the selection has to be ordered as the exact values are.
    padded = at["padded"]
    n, longest = padded.shape
    cq = q.double()[padded].reshape(n, longest, hkv, grp, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, longest * grp, d)
    cb = bounds[at["table"]].permute(0, 2, 3, 4, 1).double()  # [chunks, hkv, 2, d, pages]
    score = torch.matmul(cq.clamp_min(0), cb[:, :, 1].contiguous()) + torch.matmul(cq.clamp_max(0), cb[:, :, 0].contiguous())
    score = score.reshape(n, hkv, longest, grp, -1).amax(3).permute(0, 2, 1, 3)[at["chunk_of"], at["inside"]]
    number = torch.arange(score.shape[-1], device="cuda")[None, None, :]
    last = (pos // page)[:, None, None]
    score = torch.where((number < case["first"]) | (number > last - case["last"]), math.inf, score)
    score = torch.where(number <= last, score, -math.inf)
    # The best pages, of equal ones the lowest, in ascending order.
    best, order = torch.sort(score, dim=-1, descending=True, stable=True)
    budget = s.chosen.shape[-1]
    none = score.shape[-1]
    chosen = torch.where(best > -math.inf, order, none)[..., :budget]
    if chosen.shape[-1] < budget:
        chosen = torch.nn.functional.pad(chosen, (0, budget - chosen.shape[-1]), value=none)
    chosen = torch.sort(chosen, -1)[0]
    s.chosen.copy_(torch.where(chosen < none, chosen, -1))
    there = (chosen[..., None] * page + torch.arange(page, device="cuda")).reshape(rows, hkv, -1)
    held = at["table"][at["chunk_of"]][:, None, :].expand(-1, hkv, -1).gather(2, chosen.clamp_max(none - 1))
    head = torch.arange(hkv, device="cuda")[None, :, None]
    ck = _keys_of(keys[held, head]).reshape(rows, hkv, -1, d).float()
    cv = _values_of(values[held, head]).reshape(rows, hkv, -1, d).float()
    scores = torch.matmul(q.reshape(rows, hkv, grp, d), ck.transpose(2, 3).contiguous()) * float(np.float32(1 / math.sqrt(d)))
    scores = scores.masked_fill((there > pos[:, None, None])[:, :, None, :], -math.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp()
    y = torch.matmul(scores, cv) / scores.sum(-1, keepdim=True)
    s.out.copy_(y.reshape(rows, hq * d))
    return [s.out, s.chosen] + s.pools


# ---------------------------------------------------------------- work

def work(case):
    if case["kind"] == "adapters":
        runs, rank, _ = _runs(case)
        e = 4 if case["dtype"] == "f32" else 2
        held = runs[runs[:, 0] != NO_ADAPTER]
        slots = np.unique(held[:, 0]).astype(int)
        rows = int(runs[:, 1].sum())
        per = (rank[held[:, 0].astype(int)] * held[:, 1]).sum()
        return {"flops": 2.0 * per * (case["cols"] + case["outs"]),
                "bytes": float(rank[slots].sum()) * e * (case["cols"] + case["outs"])
                + 4.0 * (int(held[:, 1].sum()) * case["cols"] + 2 * rows * case["outs"])}
    shape, page, window = SHAPES[case["shape"]], case["page"], case["window"]
    hq, hkv, d, e = shape["heads"], shape["kv_heads"], shape["dim"], 2 if shape["half"] else 4
    chunks = _chunks(case).astype(np.int64)
    rows = int(chunks[:, 2].sum())
    new = 4.0 * rows * d * 2 * (hq + hkv) + 2.0 * rows * hkv * d * e  # q, k, v read; out, cache written
    if case["top"]:
        budget = case["top"] + case["first"] + case["last"]
        flops = bytes_ = 0.0
        for _, start, n in chunks:
            last = (start + np.arange(n)) // page
            picked = np.minimum(last + 1, budget)
            seen = np.minimum(picked * page, start + np.arange(n) + 1)
            flops += 4.0 * hq * d * seen.sum() + 4.0 * hq * d * np.maximum(last + 1 - case["first"] - case["last"], 0).sum()
            # Rows of one session may choose the same pages: each cached position is needed once.
            bytes_ += 2.0 * hkv * d * e * min(int(seen.sum()), int(start)) + 2.0 * hkv * d * e * (start // page)
        return {"flops": flops, "bytes": bytes_ + new + 4.0 * rows * hkv * budget}
    flops = bytes_ = 0.0
    for _, start, n in chunks:
        seen = start + np.arange(n) + 1
        flops += 4.0 * hq * d * (np.minimum(seen, window) if window else seen).sum()
        bytes_ += 2.0 * hkv * d * e * (min(int(start), window - 1) if window else int(start))
    return {"flops": flops, "bytes": bytes_ + new}


# ---------------------------------------------------------------- the same in 64 bits

def _turned(x, positions, shape):
    """RoPE in 64 bits of x [rows, heads, d], at 32-bit angles."""
    cos, sin = _angles(shape, int(positions.max()) + 1)
    c, s = cos.double()[positions][:, None, :], sin.double()[positions][:, None, :]
    x = x.double()
    y = torch.empty_like(x)
    d = x.shape[-1]
    first, second = (slice(0, d // 2), slice(d // 2, d)) if shape["neox"] else (slice(0, d, 2), slice(1, d, 2))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y


def exact(case, seed):
    return _exact_adapters(case, seed) if case["kind"] == "adapters" else _exact_pages(case, seed)


def _exact_adapters(case, seed):
    runs, rank, scale, a, b, x, base = _adapter_inputs(case, seed)
    out, row = base.double(), 0
    for slot, n in runs:
        n = int(n)
        if slot != NO_ADAPTER:
            down = x[row:row + n].double() @ a[slot].double().T.contiguous()
            out[row:row + n] += float(np.float32(scale[slot])) * (down @ b[slot].double().T.contiguous())
        row += n
    return out


def _exact_pages(case, seed):
    shape, page = SHAPES[case["shape"]], case["page"]
    hq, hkv, d = shape["heads"], shape["kv_heads"], shape["dim"]
    grp = hq // hkv
    chunks, _, tables, keys, values, bounds, (q, k, v) = _cache_inputs(case, seed)
    out = torch.empty(q.shape[0], hq, d, dtype=torch.float64, device="cuda")
    budget = case["top"] + case["first"] + case["last"]
    row = 0
    for s, start, n in chunks.astype(np.int64):
        pos = torch.arange(start, start + n, device="cuda")
        mine = torch.tensor(tables[int(s)], device="cuda")
        qr = _turned(q[row:row + n].reshape(n, hq, d), pos, shape)
        kr = _turned(k[row:row + n].reshape(n, hkv, d), pos, shape)
        for at in range(int(start) // page, (int(start) + int(n) - 1) // page + 1):
            lo, hi = max(at * page, int(start)), min((at + 1) * page, int(start) + int(n))
            where, rows = mine[at], slice(lo - int(start), hi - int(start))
            flat = _keys_of(keys[where]).clone()  # [hkv, page, d]
            flat[:, lo - at * page:hi - at * page] = kr[rows].transpose(0, 1).float().to(keys.dtype)
            w = keys.shape[-1]
            keys[where] = flat.reshape(hkv, page // TILE, TILE, d // w, w).transpose(2, 3)
            if bounds is not None:
                filled = flat[:, :hi - at * page]
                bounds[where] = torch.stack([filled.amin(1), filled.amax(1)], 1)
            flat = _values_of(values[where]).clone()
            flat[:, lo - at * page:hi - at * page] = v[row:row + n].reshape(n, hkv, d)[rows].transpose(0, 1).to(values.dtype)
            values[where] = flat.reshape(hkv, page // TILE, TILE, d).transpose(2, 3)
        there = torch.arange(len(mine) * page, device="cuda")
        for h in range(hkv):
            kh = _keys_of(keys[mine, h]).reshape(-1, d).double()
            vh = _values_of(values[mine, h]).reshape(-1, d).double()
            seen = there[None, :] <= pos[:, None]
            if case["window"]:
                seen &= there[None, :] > pos[:, None] - case["window"]
            qh = qr[:, h * grp:(h + 1) * grp]
            if case["top"]:
                lo, hi = bounds[mine, h, 0].double(), bounds[mine, h, 1].double()
                q32 = qh.float().double()[:, :, None, :]  # queries are rotated in 32 bits
                bound = torch.maximum(q32 * lo, q32 * hi).sum(-1).amax(1) if q32.numel() * len(lo) < 3e8 else \
                    torch.stack([torch.maximum(r[:, None] * lo, r[:, None] * hi).sum(-1).amax(0) for r in q32[:, :, 0]])
                number = torch.arange(len(mine), device="cuda")
                last = (pos // page)[:, None]
                bound[(number < case["first"]) | (number > last - case["last"])] = math.inf
                bound[number > last] = -math.inf
                picked = torch.argsort(bound, dim=1, descending=True, stable=True)[:, :budget]
                chosen = torch.zeros_like(bound, dtype=torch.bool).scatter_(1, picked, True)
                seen &= chosen.repeat_interleave(page, 1)
            for j in range(grp):
                sc = (qh[:, j] @ kh.T.contiguous()) / math.sqrt(d)
                p = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
                out[row:row + n, h * grp + j] = p @ vh
        row += int(n)
    result = [out.reshape(q.shape[0], hq * d)]
    if case["top"]:
        result.append(None)  # the pages' numbers are not computed values
    return result + [x for x in (keys, values, bounds) if x is not None]
