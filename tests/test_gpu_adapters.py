"""Low-rank adapters against plain numpy in 64 bits, and a serving step that runs them beside the shared
projections and the paged attention.

The bound: the inputs and weights are exact in 32 bits, products and sums are rounded in 32 bits, so an
output is off by at most (cols + rank + 16) 2^-24 of the sum of its terms' magnitudes, scale |B| (|A| |x|),
plus one rounding of the whole, 2^-24 (|base| + that sum).

Runs of more than 8 rows with f16 weights carry x and A x as two f16 halves, each off by at most 2^-22 of its
value: 4 2^-24 of the terms' magnitudes for either product. A term of the first product then passes at most
min(cols, 64) + 1 + cols / 256 + min(7, cols / 32) + cols / 512 rounded sums (of its 64 columns, of its wave's
steps, of the waves and of the pieces), cols + 3 at most; one of the second at most rank + 2 with the scale's
rounding: 13 beside cols + rank, of the 16 above. (An element below 2^-17 of the largest of its 64 columns is
off by 2^-39 of that one, 2^-15 of what a 2^-24 of its term is: within the rest of the 16.)
"""

import numpy as np
import pytest

from models_amd import attention as A
from models_amd import hip_runtime as rt
from models_amd import synth
from test_gpu_paged import Session

pytestmark = pytest.mark.gpu

TYPES = {A.ADAPTER_F32: np.float32, A.ADAPTER_F16: np.float16, A.ADAPTER_BF16: np.uint16}


@pytest.fixture(scope="module")
def hip():
    with A.HipAttentionLibrary(0) as lib:
        yield lib


def weights(tag, shape, dtype):
    """(as stored, the values they stand for)"""
    x = synth.normal(21, tag, shape) * 0.3
    if dtype == A.ADAPTER_BF16:
        bits = (x.view(np.uint32) >> 16).astype(np.uint16)
        return bits, (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    y = x.astype(TYPES[dtype])
    return y, y.astype(np.float64)


class Adapters:
    def __init__(self, hip, cols, outs, ranks, dtype, max_rank=None):
        self.hip, self.cols, self.outs = hip, cols, outs
        self.set = hip.adapters(len(ranks), cols, outs, max_rank or max(ranks), dtype)
        self.plain = []
        for i, r in enumerate(ranks):
            a, pa = weights(f"a{i}/{cols}", (r, cols), dtype)
            b, pb = weights(f"b{i}/{outs}", (outs, r), dtype)
            scale = np.float32(0.7 + 0.1 * i)
            da, db = rt.DeviceArray.from_host(a), rt.DeviceArray.from_host(b)
            self.set.load_device(i, r, da.ptr, da.count, db.ptr, db.count, float(scale))
            hip.synchronize()
            self.plain.append((pa, pb, float(scale)))

    def reference(self, runs, x, base):
        out = np.zeros((len(x), self.outs)) if base is None else base.astype(np.float64)
        size = np.abs(out) * 2.0 ** -24
        row = 0
        for slot, n in runs:
            if slot != A.NO_ADAPTER:
                a, b, scale = self.plain[slot]
                xs = x[row:row + n].astype(np.float64)
                out[row:row + n] += scale * (xs @ a.T) @ b.T
                terms = scale * (np.abs(xs) @ np.abs(a).T) @ np.abs(b).T
                size[row:row + n] += terms * (self.cols + a.shape[0] + 17) * 2.0 ** -24
            row += n
        return out, size

    def check(self, runs, base="random", in_place=False):
        rows = sum(n for _, n in runs)
        x = synth.normal(22, f"x{rows}", (rows, self.cols))
        plain = synth.normal(22, f"base{rows}", (rows, self.outs)) if base else None
        dx = rt.DeviceArray.from_host(x)
        out = rt.DeviceArray(rows * self.outs + 4)
        out.upload(np.full(out.count, -7.0, np.float32))
        db = rt.DeviceArray.from_host(plain) if base and not in_place else None
        if in_place:
            out.upload(plain.reshape(-1))
        self.hip.synchronize()
        self.set.apply_device(runs, dx.ptr, dx.count, out.ptr if in_place else db.ptr if db else 0, out.ptr, rows * self.outs)
        self.hip.synchronize()
        got = out.download()
        assert (got[-4:] == -7.0).all(), "written behind the rows"
        got = got[:-4].reshape(rows, self.outs)
        want, size = self.reference(runs, x, plain)
        err = np.abs(got - want)
        assert (err <= size).all(), (err / np.maximum(size, 1e-30)).max()
        return got


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cols,outs", [(8, 1), (64, 100), (520, 257), (2048, 512), (1000, 33), (4096, 1030)])
def test_runs_of_rows(hip, dtype, cols, outs):
    """Ranks from 1 up, runs of one row and of many, runs without an adapter, empty ones, an adapter that
    comes twice."""
    ad = Adapters(hip, cols, outs, [1, 8, 16, 17, 64, 3], dtype)
    ad.check([(0, 1)])
    ad.check([(4, 1), (1, 1), (A.NO_ADAPTER, 1), (4, 1), (2, 1)])
    ad.check([(3, 7), (A.NO_ADAPTER, 3), (5, 0), (0, 2), (3, 30), (2, 17)])
    ad.check([(1, 5), (4, 8)], base=None)
    ad.check([(A.NO_ADAPTER, 2), (2, 33), (5, 1)], in_place=True)
    ad.set.close()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows", [31, 64, 129, 300])
def test_prompts(hip, dtype, rows):
    ad = Adapters(hip, 1032, 770, [16, 40, 256], dtype)
    ad.check([(1, rows)])
    ad.check([(0, rows), (2, rows + 1), (A.NO_ADAPTER, 5), (1, 3)])
    ad.check([(2, rows)], in_place=True)
    ad.set.close()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_many_prompts(hip, dtype):
    """More runs of many rows than a launch takes, of lengths around a block of rows."""
    ad = Adapters(hip, 264, 133, [4, 33, 16, 70], dtype)
    ad.check([(i % 4 if i % 9 else A.NO_ADAPTER, 9 + 5 * i % 27) for i in range(120)])
    ad.check([(i % 4, 16 * (1 + i % 2) + i % 3 - 1) for i in range(50)], base=None)
    ad.set.close()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows", [3, 40])
def test_inputs_that_are_no_numbers_stay_in_their_rows(hip, dtype, rows):
    ad = Adapters(hip, 520, 300, [5, 64], dtype)
    x = synth.normal(23, "x", (2 * rows, 520))
    x[1, 3], x[rows + 2, 519] = np.inf, np.nan
    x[rows, :] *= np.float32(1e30)
    x[rows + 1, :] *= np.float32(1e-30)
    dx, out = rt.DeviceArray.from_host(x), rt.DeviceArray(2 * rows * 300)
    hip.synchronize()
    ad.set.apply_device([(0, rows), (1, rows)], dx.ptr, dx.count, 0, out.ptr, out.count)
    hip.synchronize()
    got = out.download().reshape(2 * rows, 300)
    odd = [1, rows + 2]
    assert not np.isfinite(got[odd]).any()
    with np.errstate(invalid="ignore"):
        want, size = ad.reference([(0, rows), (1, rows)], x, None)
    rest = np.delete(np.arange(2 * rows), odd)
    assert (np.abs(got[rest] - want[rest]) <= size[rest]).all()
    ad.set.close()


def test_many_runs(hip):
    ad = Adapters(hip, 256, 96, [4, 8, 12, 16, 20], A.ADAPTER_F16)
    ad.check([(i % 5 if i % 7 else A.NO_ADAPTER, i % 4) for i in range(400)])
    ad.set.close()


def test_reloaded_slot(hip):
    """A slot's next adapter may be smaller; calls already made keep the old one."""
    ad = Adapters(hip, 128, 64, [32, 5], A.ADAPTER_F16, max_rank=40)
    x = synth.normal(23, "x", (4, 128))
    dx, out, out2 = rt.DeviceArray.from_host(x), rt.DeviceArray(256), rt.DeviceArray(256)
    a, pa = weights("again a", (7, 128), A.ADAPTER_F16)
    b, pb = weights("again b", (64, 7), A.ADAPTER_F16)
    da, db = rt.DeviceArray.from_host(a), rt.DeviceArray.from_host(b)
    hip.synchronize()
    ad.set.apply_device([(0, 4)], dx.ptr, dx.count, 0, out.ptr, 256)
    ad.set.load_device(0, 7, da.ptr, da.count, db.ptr, db.count, 1.5)
    ad.set.apply_device([(0, 4)], dx.ptr, dx.count, 0, out2.ptr, 256)
    hip.synchronize()
    for o in (out, out2):
        want, size = ad.reference([(0, 4)], x, None)
        assert (np.abs(o.download().reshape(4, 64) - want) <= size).all()
        ad.plain[0] = (pa, pb, 1.5)
    ad.set.close()


def test_replayed_graph(hip):
    ad = Adapters(hip, 512, 300, [16, 24], A.ADAPTER_BF16)
    x = rt.DeviceArray.from_host(synth.normal(24, "x", (90, 512)))
    out, other = rt.DeviceArray(90 * 300), rt.DeviceArray(90 * 300)
    runs = [(0, 1), (1, 60), (A.NO_ADAPTER, 4), (0, 25)]
    step = lambda: ad.set.apply_device(runs, x.ptr, x.count, 0, out.ptr, out.count)  # noqa: E731
    hip.synchronize()
    step()
    hip.synchronize()
    want = out.download()
    graph = rt.Graph(hip.stream(), step)
    for turn in range(4):
        out.upload(np.full(out.count, np.nan, np.float32))
        hip.synchronize()
        graph.launch()
        ad.set.apply_device([(1, 90)], x.ptr, x.count, 0, other.ptr, other.count)
        if turn % 2:
            hip.synchronize()
        hip.synchronize()
        np.testing.assert_array_equal(out.download(), want)
    graph.destroy()
    ad.set.close()


@pytest.mark.parametrize("selection", [None, A.PageSelection(2, 1, 1)])
def test_a_serving_step(hip, selection):
    """One layer's attention block for a mixed batch, as a server runs it: the shared Q8_0 Q/K/V
    projection, each request's adapters on Q and on V, append and attention over pages (all, or selected
    ones), the shared output projection with the residual added, and its adapters. Every product of the
    shared projections is taken as the library gives it (they have tests of their own); what the new
    calls make of them is held to the plain forms."""
    heads, hkv, d, dim = 8, 2, 64, 256
    s = Session(hip, heads, hkv, d, True, 32, [400, 400, 400, 400], bounds=True)
    s.run([(0, 0, 300), (1, 0, 33), (2, 0, 150)])
    chunks = [(2, 150, 1), (0, 300, 3), (3, 0, 40), (1, 33, 1)]
    runs = [(0, 1), (A.NO_ADAPTER, 3), (1, 40), (0, 1)]
    rows = 45
    sizes = [heads * d, hkv * d, hkv * d]

    def blocks(tag, outs, cols):
        q = np.clip(np.rint(synth.normal(31, tag, (outs, cols // 32, 32)) * 40), -127, 127).astype(np.int8)
        scale = np.full((outs, cols // 32, 1), 0.002, np.float16)
        return rt.DeviceArray.from_host(np.concatenate([scale.view(np.uint8), q.view(np.uint8)], -1).reshape(-1))

    w = [blocks(f"w{i}", n, dim) for i, n in enumerate(sizes)]
    wo = blocks("wo", dim, heads * d)
    aq, av = Adapters(hip, dim, sizes[0], [8, 16], A.ADAPTER_F16), Adapters(hip, dim, sizes[2], [8, 16], A.ADAPTER_BF16)
    ao = Adapters(hip, heads * d, dim, [8, 16], A.ADAPTER_F16)
    x = synth.normal(31, "x", (rows, dim))
    dx, proj = rt.DeviceArray.from_host(x), rt.DeviceArray(rows * sum(sizes))
    hip.synchronize()
    hip.quantized_grouped_matmul_device([A.WEIGHTS_Q8_0] * 3, [b.ptr for b in w], [b.nbytes for b in w], sizes, dx.ptr,
                                        dx.count, proj.ptr, proj.count, rows, dim)
    hip.synchronize()
    shared = proj.download()
    parts = np.split(shared, np.cumsum([rows * n for n in sizes])[:-1])
    q, k, v = proj.at(0), proj.at(rows * sizes[0]), proj.at(rows * (sizes[0] + sizes[1]))
    attn, out = rt.DeviceArray(rows * heads * d), rt.DeviceArray(rows * dim)
    aq.set.apply_device(runs, dx.ptr, dx.count, q, q, rows * sizes[0])
    av.set.apply_device(runs, dx.ptr, dx.count, v, v, rows * sizes[2])
    s.kv.forward_device(s.layer, chunks, q, rows * sizes[0], k, rows * sizes[1], v, rows * sizes[2], attn.ptr, attn.count, selection)
    hip.quantized_matmul_device(A.WEIGHTS_Q8_0, wo.ptr, wo.nbytes, attn.ptr, attn.count, out.ptr, out.count, rows, dim,
                                heads * d, dx.ptr, A.ADDEND_RESIDUAL)
    hip.synchronize()
    before = out.download().reshape(rows, dim)
    ao.set.apply_device(runs, attn.ptr, attn.count, out.ptr, out.ptr, out.count)
    hip.synchronize()
    # The projections with their adapters, in place.
    got = np.split(proj.download(), np.cumsum([rows * n for n in sizes])[:-1])
    for i, ad in ((0, aq), (2, av)):
        want, size = ad.reference(runs, x, parts[i].reshape(rows, -1))
        assert (np.abs(got[i].reshape(rows, -1) - want) <= size).all()
    np.testing.assert_array_equal(got[1], parts[1])
    # Attention of what they gave: the plain form's new rows are those.
    real = synth.normal
    try:
        given = iter(g.reshape(rows, -1) for g in got)
        synth.normal = lambda *a: next(given)
        _, _, _, qn = s.rows(chunks)
    finally:
        synth.normal = real
    a = attn.download()
    s.close_to(a, chunks, qn, s.selected(chunks, qn, selection) if selection else None)
    s.check_cache()
    # The output projection's adapters.
    want, size = ao.reference(runs, a.reshape(rows, -1), before)
    assert (np.abs(out.download().reshape(rows, dim) - want) <= size).all()
    for ad in (aq, av, ao):
        ad.set.close()
    s.close()
