"""The paged cache's and the adapters' host side on the CPU, under the sanitizers and the host
simulation of tests/hostsim (whose launches check every device range and page number when they
execute): page bookkeeping, refusals that change nothing, graph capture, and calls past one launch's
sizes."""

import pytest

from test_hostsim_cpu import _python, sim  # noqa: F401  (sim is the fixture)

HEAD = """
import ctypes
import numpy as np
from models_amd import attention as A, hip_runtime as rt

launches = rt.hip().hipsim_launches
launches.restype = ctypes.c_long

def refused(status, call, *args, **kw):
    before = launches()
    try:
        call(*args, **kw)
    except A.AttentionStatusError as e:
        assert e.status_name == status, e
    else:
        raise AssertionError(f"not refused as {status}: {args}")
    assert launches() == before, "a refused call launched something"

class Rows:
    # q, k, v, out and rotated q of `rows` rows
    def __init__(self, rows, heads, hkv, d):
        self.q, self.k, self.v, self.out, self.rot = (rt.DeviceArray(max(rows, 1) * h * d) for h in (heads, hkv, hkv, heads, heads))
        self.n = rows
    def forward(self, kv, layer, chunks, selection=None, pages=None):
        kv.forward_device(layer, chunks, self.q.ptr, self.q.count, self.k.ptr, self.k.count, self.v.ptr, self.v.count,
                          self.out.ptr, self.out.count, selection, pages.ptr if pages else 0, pages.count if pages else 0)
    def append(self, kv, layer, chunks):
        kv.append_device(layer, chunks, self.q.ptr, self.q.count, self.k.ptr, self.k.count, self.v.ptr, self.v.count,
                         self.rot.ptr, self.rot.count)
    def attend(self, kv, layer, chunks, pages=None, budget=0):
        kv.attend_device(layer, chunks, self.rot.ptr, self.rot.count, self.out.ptr, self.out.count,
                         pages.ptr if pages else 0, pages.count if pages else 0, budget)
    def select(self, kv, layer, chunks, selection, pages):
        kv.select_device(layer, chunks, selection, self.rot.ptr, self.rot.count, pages.ptr, pages.count)
"""


def run(env, body):
    return _python(env, HEAD + body)


def test_shapes_that_are_refused(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    good = dict(num_layers=1, max_seq_len=100, pages=8, page_slots=32, num_kv_heads=2, head_length=64)
    for wrong in (dict(page_slots=16), dict(page_slots=48), dict(page_slots=512), dict(head_length=48),
                  dict(head_length=512), dict(pages=0), dict(num_layers=0), dict(max_seq_len=0),
                  dict(num_kv_heads=0), dict(sequences=0)):
        refused("INVALID_SHAPE", hip.paged_kv_cache, **{**good, **wrong})
    out = ctypes.c_void_p()
    create = hip.lib.jmodels_attn_paged_kv_create
    assert create(hip.ctx, 1, 1, 100, 8, 32, 2, 64, 2, 0, ctypes.byref(out)) == A.INVALID_SHAPE
    assert create(hip.ctx, 1, 1, 100, 8, 32, 2, 64, 1, 2, ctypes.byref(out)) == A.INVALID_SHAPE
    assert create(hip.ctx, 1, 1, 100, 8, 32, 2, 64, 1, 0, None) == A.NULL_POINTER
    assert create(None, 1, 1, 100, 8, 32, 2, 64, 1, 0, ctypes.byref(out)) == A.NULL_POINTER
    live = rt.hip().hipsim_live_bytes
    live.restype = ctypes.c_size_t
    before = live()
    rt.hip().hipsim_largest_allocation(ctypes.c_size_t(1 << 20))
    refused("DEVICE_ERROR", hip.paged_kv_cache, **{**good, "pages": 1000, "head_length": 256})
    rt.hip().hipsim_largest_allocation(ctypes.c_size_t(2 ** 62))
    assert live() == before, "a cache that could not be had left memory behind"
""")


def test_pages_are_the_lowest_free_ones(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    kv = hip.paged_kv_cache(2, 300, 10, 32, 2, 64, sequences=4)
    kv.reserve(1, 33)
    kv.reserve(0, 1)
    kv.reserve(1, 70)
    kv.reserve(2, 0)
    assert [kv.pages(s).tolist() for s in range(4)] == [[2], [0, 1, 3], [], []] and kv.free_pages() == 6
    kv.reserve(1, 70)
    assert kv.free_pages() == 6
    kv.discard_from(31, 1)       # one page is still needed
    assert kv.pages(1).tolist() == [0] and kv.free_pages() == 8
    kv.reserve(3, 32 * 4)
    assert kv.pages(3).tolist() == [1, 3, 4, 5]
    refused("OUT_OF_PAGES", kv.reserve, 2, 32 * 5)
    assert kv.pages(2).tolist() == [] and kv.free_pages() == 4
    kv.reserve(2, 32 * 4)
    assert kv.free_pages() == 0
    refused("OUT_OF_PAGES", kv.reserve, 0, 33)
    kv.clear(3)
    kv.reserve(0, 33)
    assert kv.pages(0).tolist() == [2, 1]
    kv.clear()
    assert kv.free_pages() == 10 and all(kv.pages(s).size == 0 for s in range(4))
    refused("OUT_OF_RANGE", kv.reserve, 4, 1)
    refused("OUT_OF_RANGE", kv.reserve, 0, 301)
    refused("OUT_OF_RANGE", kv.discard_from, 301, 0)
    refused("OUT_OF_RANGE", kv.clear, 4)
    refused("OUT_OF_RANGE", kv.pages, 4)
    refused("OUT_OF_RANGE", kv.length, 2, 0)
    refused("OUT_OF_RANGE", kv.storage, 2)
    refused("UNAVAILABLE", kv.set_length, 0, 0, 1)
    kv.reserve(0, 40)
    kv.set_length(1, 0, 64)
    refused("UNAVAILABLE", kv.set_length, 1, 0, 65)
    assert kv.length(1, 0) == 64 and kv.length(0, 0) == 0
    small = (ctypes.c_uint32 * 1)()
    n = ctypes.c_uint32()
    assert hip.lib.jmodels_attn_paged_kv_pages(kv.handle, 0, small, 1, ctypes.byref(n)) == A.BUFFER_TOO_SMALL
    big = hip.paged_kv_cache(1, 100000, 3000, 32, 1, 32, sequences=3)
    big.reserve(2, 32 * 1000)   # more entries than one table launch takes
    assert big.pages(2).tolist() == list(range(1000))
    for c in (kv, big):
        c.close()
""")


def test_append_rules(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    kv = hip.paged_kv_cache(2, 100, 6, 32, 2, 64, sequences=4)
    rope = hip.rotary_table(64, 1e4, max_positions=90)
    l0, l1 = (A.AttentionLayer(i, 4, rope=rope) for i in range(2))
    r = Rows(200, 4, 2, 64)
    r.forward(kv, l0, [[0, 0, 40], [2, 0, 1]])
    assert (kv.length(0, 0), kv.length(1, 0), kv.length(0, 2)) == (40, 0, 1)
    assert kv.pages(0).tolist() == [0, 1] and kv.pages(2).tolist() == [2]
    # A chunk may not leave a gap; in another layer the sequence holds nothing yet.
    refused("UNAVAILABLE", r.forward, kv, l0, [[0, 41, 1]])
    refused("UNAVAILABLE", r.forward, kv, l1, [[0, 40, 1]])
    r.forward(kv, l0, [[0, 33, 2]])  # a rewind: the layer ends with the chunk
    assert kv.length(0, 0) == 35 and kv.pages(0).tolist() == [0, 1]
    refused("UNAVAILABLE", r.attend, kv, l0, [[0, 30, 6]])
    r.attend(kv, l0, [[0, 30, 5], [2, 0, 1]])
    # Nothing changes when one of the call's chunks cannot be had.
    refused("OUT_OF_PAGES", r.forward, kv, l0, [[1, 0, 32], [3, 0, 70]])
    assert kv.free_pages() == 3 and kv.pages(1).size == 0 and kv.length(0, 1) == 0
    refused("INVALID_SHAPE", r.forward, kv, l0, [[1, 0, 1], [1, 1, 1]])
    refused("OUT_OF_RANGE", r.forward, kv, l0, [[4, 0, 1]])
    refused("OUT_OF_RANGE", r.forward, kv, l0, [[1, 0, 101]])
    refused("OUT_OF_RANGE", r.forward, kv, l0, [[1, 0, 91]])   # past the rope table
    refused("OUT_OF_RANGE", r.forward, kv, l0, [[1, 0xFFFFFFFF, 2]])
    refused("OUT_OF_RANGE", r.forward, kv, A.AttentionLayer(2, 4), [[1, 0, 1]])
    refused("INVALID_SHAPE", r.forward, kv, A.AttentionLayer(0, 3), [[1, 0, 1]])
    # Chunks without rows are left out, and a call of nothing else does nothing.
    r.forward(kv, l0, [[3, 50, 0], [2, 1, 1], [3, 0, 0]])
    assert kv.length(0, 2) == 2 and kv.length(0, 3) == 0 and kv.pages(3).size == 0
    before = launches()
    r.forward(kv, l0, [[3, 50, 0]])
    assert launches() == before
    for bad in ([], [[1, 2]], [[0.5, 0, 1]], [[-1, 0, 1]]):
        try:
            r.forward(kv, l0, bad)
            raise AssertionError(bad)
        except ValueError:
            pass
    # Sizes, pointers, alignment.
    args = lambda **kw: [kw.get(k, v) for k, v in dict(q=r.q.ptr, qn=256, k=r.k.ptr, kn=128, v=r.v.ptr, vn=128, o=r.out.ptr, on=256).items()]
    ok = [[1, 0, 1]]
    for kw, status in ((dict(qn=255), "BUFFER_TOO_SMALL"), (dict(kn=127), "BUFFER_TOO_SMALL"), (dict(vn=127), "BUFFER_TOO_SMALL"),
                       (dict(on=255), "BUFFER_TOO_SMALL"), (dict(q=0), "NULL_POINTER"), (dict(k=0), "NULL_POINTER"),
                       (dict(v=0), "NULL_POINTER"), (dict(o=0), "NULL_POINTER"), (dict(q=r.q.ptr + 4), "INVALID_SHAPE"),
                       (dict(o=r.out.ptr + 8), "INVALID_SHAPE")):
        refused(status, kv.forward_device, l0, ok, *args(**kw))
    other = A.HipAttentionLibrary(0)
    refused("INVALID_SHAPE", r.forward, kv, A.AttentionLayer(0, 4, rope=other.rotary_table(64, 1e4)), ok)
    for c in (kv, rope):
        c.close()
""")


def test_fork_shares_whole_pages(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    kv = hip.paged_kv_cache(2, 200, 8, 32, 2, 64, sequences=4)
    layers = [A.AttentionLayer(i, 4) for i in range(2)]
    r = Rows(100, 4, 2, 64)
    for l in layers:
        r.forward(kv, l, [[0, 0, 70]])
    refused("INVALID_SHAPE", kv.fork, 0, 1, 33)
    refused("UNAVAILABLE", kv.fork, 0, 1, 96)
    refused("INVALID_SHAPE", kv.fork, 0, 0, 32)
    refused("OUT_OF_RANGE", kv.fork, 0, 4, 32)
    kv.fork(0, 1, 64)
    assert kv.pages(1).tolist() == [0, 1] and kv.free_pages() == 5 and kv.length(1, 1) == 64
    refused("INVALID_SHAPE", kv.fork, 0, 1, 32)  # the target has pages
    # A shared page is read, and not written by either sequence.
    r.attend(kv, layers[0], [[1, 60, 4]])
    refused("UNAVAILABLE", r.forward, kv, layers[0], [[1, 63, 1]])
    refused("UNAVAILABLE", r.forward, kv, layers[0], [[0, 40, 30]])
    r.forward(kv, layers[0], [[1, 64, 1], [0, 70, 1]])
    assert kv.pages(1).tolist() == [0, 1, 3]
    kv.clear(0)
    assert kv.free_pages() == 5, "the forked sequence's pages were freed"
    r.forward(kv, layers[0], [[1, 63, 1]])  # now its own
    kv.clear(1)
    assert kv.free_pages() == 8
    kv.close()
""")


def test_selection_rules(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    plain = hip.paged_kv_cache(1, 2000, 64, 32, 2, 64, sequences=2)
    kv = hip.paged_kv_cache(1, 2000, 64, 32, 2, 64, sequences=2, page_bounds=True)
    layer, r = A.AttentionLayer(0, 4), Rows(1500, 4, 2, 64)
    sel = A.PageSelection(3, 1, 2)
    pages = rt.DeviceArray(1500 * 2 * 6, np.uint32)
    refused("INVALID_SHAPE", r.forward, plain, layer, [[0, 0, 4]], sel)
    assert plain.storage(0).bounds is None and kv.storage(0).bounds
    refused("INVALID_SHAPE", r.forward, kv, layer, [[0, 0, 4]], A.PageSelection(3, 1, 0))
    refused("INVALID_SHAPE", r.forward, kv, layer, [[0, 0, 4]], A.PageSelection(65536, 0, 1))
    refused("INVALID_SHAPE", r.forward, kv, A.AttentionLayer(0, 4, sliding_window=64), [[0, 0, 4]], sel)
    refused("INVALID_SHAPE", r.forward, kv, layer, [[0, 0, 4]], None, pages)  # pages without a selection
    r.forward(kv, layer, [[0, 0, 1000]], sel)
    r.forward(kv, layer, [[0, 1000, 500], [1, 0, 3]], sel, pages)
    small = rt.DeviceArray(500 * 2 * 6 - 1, np.uint32)
    refused("BUFFER_TOO_SMALL", r.forward, kv, layer, [[0, 1000, 500]], sel, small)
    assert kv.length(0, 0) == 1500
    r.select(kv, layer, [[0, 1000, 500]], sel, pages)
    refused("UNAVAILABLE", r.select, kv, layer, [[0, 1499, 2]], sel, pages)
    refused("BUFFER_TOO_SMALL", r.select, kv, layer, [[0, 1000, 500]], sel, small)
    r.attend(kv, layer, [[0, 1000, 500]], pages, 6)
    refused("BUFFER_TOO_SMALL", r.attend, kv, layer, [[0, 1000, 500]], small, 6)
    refused("INVALID_SHAPE", r.attend, kv, layer, [[0, 1000, 5]], pages, 0)
    refused("NULL_POINTER", r.attend, kv, layer, [[0, 1000, 5]], None, 6)
    refused("INVALID_SHAPE", r.attend, kv, A.AttentionLayer(0, 4, sliding_window=64), [[0, 1000, 5]], pages, 6)
    for c in (kv, plain):
        c.close()
""")


def test_capture(sim):  # noqa: F811
    """A captured call that would need pages or scratch is refused with nothing changed; one that has
    them is recorded, and its replays check their ranges again."""
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    kv = hip.paged_kv_cache(1, 5000, 400, 32, 2, 64, sequences=2, page_bounds=True)
    layer, r, sel = A.AttentionLayer(0, 4), Rows(64, 4, 2, 64), A.PageSelection(2, 1, 1)
    def captured(chunks, selection=None):
        g = rt.Graph(hip.stream(), lambda: r.forward(kv, layer, chunks, selection))
        for _ in range(3):
            g.launch()
            hip.synchronize()
        g.destroy()
    def not_captured(chunks, selection=None):
        state = kv.length(0, 0), kv.pages(0).tolist(), kv.free_pages()
        try:
            captured(chunks, selection)
        except A.AttentionStatusError as e:
            assert e.status_name == "NOT_CAPTURABLE", e
        else:
            raise AssertionError("captured")
        assert (kv.length(0, 0), kv.pages(0).tolist(), kv.free_pages()) == state
    kv.reserve(0, 64)
    not_captured([[0, 0, 64]])          # no scratch yet
    r.forward(kv, layer, [[0, 0, 64]])
    not_captured([[0, 64, 1]])          # the page is missing
    kv.reserve(0, 4000)
    captured([[0, 64, 1]])
    not_captured([[0, 65, 1]], sel)     # the selection's scratch is
    kv.set_length(0, 0, 3900)
    r.forward(kv, layer, [[0, 3900, 1]], sel)
    r.forward(kv, layer, [[0, 3901, 1]])
    captured([[0, 3902, 1]], sel)
    captured([[0, 3903, 1]])
    kv.close()
    ad = hip.adapters(2, 64, 32, 8)
    w = rt.DeviceArray(64 * 64, np.float16)
    ad.load_device(0, 8, w.ptr, 512, w.ptr, 256)
    x, y = rt.DeviceArray(64 * 64), rt.DeviceArray(64 * 32)
    def apply(n):
        ad.apply_device([[0, n]], x.ptr, x.count, 0, y.ptr, y.count)
    try:
        rt.Graph(hip.stream(), lambda: ad.load_device(1, 8, w.ptr, 512, w.ptr, 256))
        raise AssertionError("captured")
    except A.AttentionStatusError as e:
        assert e.status_name == "NOT_CAPTURABLE", e
    apply(64)
    g = rt.Graph(hip.stream(), lambda: apply(64))
    g.launch()
    g.destroy()
    ad.close()
""")


def test_calls_past_one_launch(sim):  # noqa: F811
    """More chunks than one launch takes, and chunks of more rows than a grid holds."""
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    n = 300
    kv = hip.paged_kv_cache(1, 4000, 3000, 32, 2, 32, sequences=n, page_bounds=True)
    layer, r = A.AttentionLayer(0, 2), Rows(3 * n, 2, 2, 32)
    start = np.zeros((n, 3), np.uint32)
    start[:, 0], start[:, 2] = np.arange(n), 3
    r.forward(kv, layer, start)
    one = np.stack([np.arange(n), np.full(n, 3), np.ones(n, int)], 1)
    r.forward(kv, layer, one, A.PageSelection(1, 0, 1))
    for i in range(0, n, 7):
        kv.reserve(i, 10 + 9 * i)
        kv.set_length(0, i, 10 + 8 * i)
    ragged = np.array([[i, kv.length(0, i), 1 + 40 * (i % 50 == 0)] for i in range(n)])
    big = Rows(int(ragged[:, 2].sum()), 2, 2, 32)
    big.forward(kv, layer, ragged)
    big.forward(kv, layer, ragged, A.PageSelection(9, 1, 2))
    kv.close()
    kv = hip.paged_kv_cache(1, 20000, 700, 32, 32, 32, sequences=1, page_bounds=True)
    layer, r = A.AttentionLayer(0, 64), Rows(17000, 64, 32, 32)
    r.forward(kv, layer, [[0, 0, 17000]])
    r.forward(kv, layer, [[0, 10000, 7000]], A.PageSelection(4, 1, 2))
    kv.close()
    ad = hip.adapters(3, 8, 1, 4, A.ADAPTER_F32)
    w = rt.DeviceArray(64)
    for s in range(3):
        ad.load_device(s, 4, w.ptr, 32, w.ptr, 4)
    x, y = rt.DeviceArray(600000 * 8), rt.DeviceArray(600000)
    ad.apply_device([[0, 600000]], x.ptr, x.count, 0, y.ptr, y.count)
    ad.apply_device([[i % 3, i % 5] for i in range(500)], x.ptr, x.count, y.ptr, y.ptr, y.count)
    ad.close()
""")


def test_adapter_refusals(sim):  # noqa: F811
    run(sim, """
with A.HipAttentionLibrary(0) as hip:
    for wrong in ((0, 64, 32, 8), (2, 60, 32, 8), (2, 0, 32, 8), (2, 64, 0, 8), (2, 64, 32, 0), (2, 64, 32, 257)):
        refused("INVALID_SHAPE", hip.adapters, *wrong)
    refused("INVALID_SHAPE", hip.adapters, 2, 64, 32, 8, 3)
    ad = hip.adapters(2, 64, 32, 8)
    w, x, y = rt.DeviceArray(1024, np.float16), rt.DeviceArray(10 * 64), rt.DeviceArray(10 * 32)
    refused("OUT_OF_RANGE", ad.load_device, 2, 8, w.ptr, 512, w.ptr, 256)
    refused("INVALID_SHAPE", ad.load_device, 0, 9, w.ptr, 1024, w.ptr, 1024)
    refused("INVALID_SHAPE", ad.load_device, 0, 0, w.ptr, 512, w.ptr, 256)
    refused("BUFFER_TOO_SMALL", ad.load_device, 0, 8, w.ptr, 511, w.ptr, 256)
    refused("BUFFER_TOO_SMALL", ad.load_device, 0, 8, w.ptr, 512, w.ptr, 255)
    refused("NULL_POINTER", ad.load_device, 0, 8, None, 512, w.ptr, 256)
    refused("INVALID_SHAPE", ad.load_device, 0, 8, w.ptr + 1, 512, w.ptr, 256)
    refused("INVALID_SHAPE", ad.load_device, 0, 8, w.ptr, 512, w.ptr, 256, float("nan"))
    call = lambda runs, xn=640, yn=320, xp=x.ptr, yp=y.ptr, b=0: ad.apply_device(runs, xp, xn, b, yp, yn)
    refused("UNAVAILABLE", call, [[0, 1]])
    ad.load_device(0, 8, w.ptr, 512, w.ptr, 256)
    ad.load_device(1, 3, w.ptr, 192, w.ptr, 96)
    call([[0, 3], [A.NO_ADAPTER, 2], [1, 0], [0, 5]])
    refused("OUT_OF_RANGE", call, [[0, 1], [2, 1]])
    refused("BUFFER_TOO_SMALL", call, [[0, 11]])
    refused("BUFFER_TOO_SMALL", call, [[0, 10]], 639)
    refused("BUFFER_TOO_SMALL", call, [[0, 10]], 640, 319)
    refused("INVALID_SHAPE", call, [[0, 1]], xp=x.ptr + 4)
    refused("INVALID_SHAPE", call, [[0, 1]], b=x.ptr + 4)
    refused("NULL_POINTER", call, [[0, 1]], yp=0)
    ad.unload(0)
    refused("UNAVAILABLE", call, [[0, 1]])
    before = launches()
    call([[1, 0]])
    assert launches() == before
    ad.close()
""")
