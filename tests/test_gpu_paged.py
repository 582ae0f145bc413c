"""The paged cache's kernels against plain numpy in 64 bits: stored keys, values and bounds bit for
bit, the selected pages exactly, and attention within a bound derived from the kernels' roundings.

The bound. A score is a sum of d products of 32-bit operands (an f16 cache's queries are carried as
two f16 halves, 2^-22 of the element lost at most), accumulated in 32 bits: its error is at most
(2^-21 + (d + 8) 2^-24) |q| |k| scale, by Cauchy-Schwarz. An error e of every score changes each
probability by a factor within exp(+-2 e), and an output, an average of values, by 2 e max|v| to first
order. The exponentials (2 ulp), the halves of a probability (2^-22) and the 32-bit sums over the n
positions, whose terms are all of one sign or weighted by probabilities, add (2^-20 + n 2^-24) max|v|.
"""

import numpy as np
import pytest

from models_amd import attention as A
from models_amd import hip_runtime as rt
from models_amd import synth
from gpu_support import rope_rows

pytestmark = pytest.mark.gpu

THETA = 1e4


@pytest.fixture(scope="module")
def hip():
    with A.HipAttentionLibrary(0) as lib:
        yield lib


def stored(x, half):
    return x.astype(np.float16).astype(np.float64) if half else x.astype(np.float64)


class Session:
    """A paged cache of one layer beside its plain counterpart: per sequence, the rotated keys and the
    values that it should hold."""

    def __init__(self, hip, heads, hkv, d, half, page, lengths, max_len=None, bounds=False, neox=True, rotary=None,
                 window=0, scale=0.0, norm=None, value_rms=False, poison=True, spare=0):
        self.hip, self.heads, self.hkv, self.d, self.half, self.page = hip, heads, hkv, d, half, page
        self.max_len = max_len or max(lengths) + 64
        pages = sum(-(-self.max_len // page) for _ in lengths) + spare
        self.kv = hip.paged_kv_cache(1, self.max_len, pages, page, hkv, d, half, len(lengths), bounds)
        if poison:  # what no append wrote is no number
            st = self.kv.storage(0)
            for p in (st.keys, st.values):
                rt.check(rt.hip().hipMemset(p, 0xFF, st.bytes), "hipMemset")
            rt.device_synchronize()
        self.rotary, self.neox, self.window = rotary if rotary is not None else d, neox, window
        self.rope = hip.rotary_table(self.rotary, THETA, max_positions=self.max_len) if self.rotary else None
        self.scale = scale or A.default_scale(d)
        self.norm = None
        if norm is not None:
            self.qw, self.kw, self.eps = norm
            self.norm = hip.qk_norm(d, self.qw, self.kw, self.eps, value_rms)
        self.value_rms = value_rms
        self.layer = A.AttentionLayer(0, heads, window, neox, scale, self.rope, self.norm)
        self.keys = [np.zeros((0, hkv, d), np.float32) for _ in lengths]
        self.values = [np.zeros((0, hkv, d), np.float32) for _ in lengths]
        self.count = 0

    def close(self):
        self.kv.close()
        for h in (self.rope, self.norm):
            if h is not None:
                h.close()

    def _normed(self, x, w):
        """TensorOps.rmsNorm per head: sums in order, in 32 bits."""
        ss = np.zeros(x.shape[:-1], np.float32)
        for e in range(self.d):
            ss = ss + x[..., e] * x[..., e]
        rms = np.sqrt((ss / np.float32(self.d) + np.float32(self.eps)).astype(np.float64))
        if w is None:
            return x * (1.0 / rms).astype(np.float32)[..., None]
        return x * (np.float32(1) / rms.astype(np.float32))[..., None] * np.asarray(w, np.float32)

    def rows(self, chunks, tag="x", spread=1.0):
        """New q, k, v of the chunks, and their plain form: rotated queries, keys and values appended."""
        self.count += 1
        n = sum(c[2] for c in chunks)
        q, k, v = (spread * synth.normal(11, f"{tag}/{self.count}/{name}", (n, h * self.d))
                   for name, h in (("q", self.heads), ("k", self.hkv), ("v", self.hkv)))
        pos = np.concatenate([np.arange(s, s + r) for _, s, r in chunks])
        qn, kn, vn = (x.reshape(n, -1, self.d) for x in (q, k, v))
        if self.norm is not None:
            qn = self._normed(qn, self.qw) if self.qw is not None else qn
            kn = self._normed(kn, self.kw) if self.kw is not None else kn
            vn = self._normed(vn, None) if self.value_rms else vn
        if self.rope is not None:
            qn, kn = (rope_rows(x, pos, h, self.d, self.rotary, THETA, self.neox, check_against_oracle=False)
                      .reshape(n, h, self.d) for x, h in ((qn, self.heads), (kn, self.hkv)))
        at = 0
        for s, start, r in chunks:
            self.keys[s] = np.concatenate([self.keys[s][:start], kn[at:at + r]])
            self.values[s] = np.concatenate([self.values[s][:start], vn[at:at + r]])
            at += r
        return q, k, v, qn

    def visible(self, p):
        return max(0, p - self.window + 1) if self.window else 0

    def reference(self, chunks, qn, chosen=None):
        """(out, bound) in 64 bits; chosen: per row and kv head, page numbers."""
        out = np.zeros((qn.shape[0], self.heads, self.d))
        bound = np.zeros(qn.shape[0])
        row = 0
        for s, start, r in chunks:
            grp = self.heads // self.hkv
            for j in range(self.hkv):
                k, v = (np.ascontiguousarray(stored(x[s][:, j], self.half)) for x in (self.keys, self.values))
                norms, tops = np.linalg.norm(k, axis=1), np.abs(v).max(1)
                for i in range(r):
                    p, heads = start + i, slice(j * grp, (j + 1) * grp)
                    at = slice(self.visible(p), p + 1)
                    if chosen is not None:
                        at = np.flatnonzero(np.isin(np.arange(p + 1) // self.page, chosen[row + i][j]))
                    q = qn[row + i, heads].astype(np.float64)
                    x = q @ k[at].T * self.scale
                    w = np.exp(x - x.max(1, keepdims=True))
                    out[row + i, heads] = w @ v[at] / w.sum(1, keepdims=True)
                    e = (2.0 ** -21 + (self.d + 8) * 2.0 ** -24) * np.linalg.norm(q, axis=1).max() * norms[at].max() * self.scale
                    bound[row + i] = max(bound[row + i], (2 * e + 2.0 ** -20 + x.shape[1] * 2.0 ** -24) * tops[at].max())
            row += r
        return out, bound

    def run(self, chunks, tag="x", selection=None, spread=1.0):
        """forward_device on new rows; checks out (and the pages) against the plain form."""
        q, k, v, qn = self.rows(chunks, tag, spread)
        dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
        out = rt.DeviceArray(q.size + 8)
        out.upload(np.full(q.size + 8, -7.0, np.float32))
        n = q.shape[0]
        budget = selection.budget if selection else 0
        pages = rt.DeviceArray(n * self.hkv * budget + 4, np.uint32) if selection else None
        if selection:
            pages.upload(np.full(pages.count, 12345, np.uint32))
        self.hip.synchronize()
        self.kv.forward_device(self.layer, chunks, dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, out.ptr,
                               q.size, selection, pages.ptr if selection else 0, n * self.hkv * budget if selection else 0)
        self.hip.synchronize()
        got = out.download()
        assert (got[q.size:] == -7.0).all(), "written behind the rows"
        chosen = None
        if selection:
            lists = pages.download()
            assert (lists[-4:] == 12345).all(), "written behind the lists"
            lists = lists[:-4].reshape(n, self.hkv, budget)
            chosen = self.selected(chunks, qn, selection)
            for i in range(n):
                for j in range(self.hkv):
                    want = np.full(budget, A.NO_PAGE, np.uint32)
                    want[:len(chosen[i][j])] = chosen[i][j]
                    np.testing.assert_array_equal(lists[i, j], want, f"row {i}, kv head {j}")
        self.close_to(got[:q.size], chunks, qn, chosen)
        return got[:q.size].reshape(n, self.heads, self.d), qn, chosen

    def fill(self, chunks, tag="fill"):
        """append_device alone."""
        _, k, v, _ = self.rows(chunks, tag)
        dk, dv = rt.DeviceArray.from_host(k), rt.DeviceArray.from_host(v)
        self.hip.synchronize()
        self.kv.append_device(self.layer, chunks, 0, 0, dk.ptr, dk.count, dv.ptr, dv.count)
        self.hip.synchronize()

    def close_to(self, got, chunks, qn, chosen=None):
        want, bound = self.reference(chunks, qn, chosen)
        err = np.abs(got.reshape(want.shape).astype(np.float64) - want).max((1, 2))
        assert np.isfinite(got).all() and (err <= bound).all(), (err / bound).max()

    def check_cache(self):
        for s in range(len(self.keys)):
            n = len(self.keys[s])
            k, v = self.kv.read(0, 0, n, s)
            np.testing.assert_array_equal(k.reshape(-1, self.hkv, self.d), stored(self.keys[s], self.half), f"keys of {s}")
            np.testing.assert_array_equal(v.reshape(-1, self.hkv, self.d), stored(self.values[s], self.half), f"values of {s}")

    def bounds_of(self, s):
        """Plain bounds of sequence s: [pages][2][hkv][d]."""
        k = stored(self.keys[s], self.half)
        return [np.stack([k[i:i + self.page].min(0), k[i:i + self.page].max(0)]) for i in range(0, len(k), self.page)]

    def selected(self, chunks, qn, sel):
        lists, row = [], 0
        grp = self.heads // self.hkv
        for s, start, r in chunks:
            bounds = self.bounds_of(s)
            for i in range(r):
                n = (start + i) // self.page + 1
                per = []
                for j in range(self.hkv):
                    if n <= sel.budget:
                        per.append(np.arange(n))
                        continue
                    score = np.empty(n)
                    for p in range(n):
                        lo, hi = bounds[p][:, j]
                        score[p] = max(np.maximum(x * lo, x * hi).sum() for x in qn[row, j * grp:(j + 1) * grp].astype(np.float64))
                    score[:sel.first] = np.inf
                    score[n - sel.last:] = np.inf
                    per.append(np.sort(np.argsort(-score, kind="stable")[:sel.budget]))
                lists.append(per)
                row += 1
        return lists


# heads, kv heads, head length, f16, page
SHAPES = [(4, 2, 64, True, 32), (32, 8, 64, True, 64), (12, 2, 128, True, 32), (5, 5, 128, True, 128), (3, 1, 256, True, 256),
          (16, 2, 32, True, 64), (20, 1, 64, True, 32), (33, 1, 128, True, 64), (4, 2, 64, False, 32), (16, 8, 128, False, 64),
          (6, 2, 256, False, 32), (3, 3, 32, False, 128), (40, 2, 128, False, 32)]
IDS = [f"{h}x{k}x{d}_{'f16' if f else 'f32'}_p{p}" for h, k, d, f, p in SHAPES]


@pytest.mark.parametrize("heads,hkv,d,half,page", SHAPES, ids=IDS)
def test_chunks_of_many_sequences(hip, heads, hkv, d, half, page):
    """Prompts, rewinds and single tokens mixed, pages handed out in turn, lengths around tile and page
    ends; the stored cache bit for bit."""
    s = Session(hip, heads, hkv, d, half, page, [330, 300, 1, 66])
    s.run([(0, 0, 1), (1, 0, 37)], "start")
    s.run([(1, 37, 27), (0, 1, 31), (3, 0, 65)], "tiles")        # to 64, 32, 65
    s.run([(0, 32, 1), (1, 64, 1), (2, 0, 1), (3, 65, 1)], "tokens")
    s.run([(1, 65, 200), (0, 33, 3), (3, 64, 2)], "mixed")       # sequence 3 rewinds
    s.run([(1, 265, 5), (0, 20, 290)], "rewound")                # so does sequence 0
    s.run([(2, 1, 1), (0, 310, 1), (1, 270, 1)], "tokens again")
    s.check_cache()
    s.close()


@pytest.mark.parametrize("heads,hkv,d,half", [(8, 2, 64, True), (6, 2, 32, False), (4, 4, 128, True)])
@pytest.mark.parametrize("sel", [None, A.PageSelection(2, 1, 1)])
def test_more_chunks_than_a_launch_holds(hip, heads, hkv, d, half, sel):
    """150 sequences of 1 to 20 new rows, whose blocks of rows lie one after another in the launches' grids,
    single tokens beside prompts that need several blocks."""
    n = 150
    s = Session(hip, heads, hkv, d, half, 32, [200] * n, bounds=True)
    s.fill([(i, 0, 1 + 37 * i % 150) for i in range(n)])
    rows = [1 if i % 3 else 1 + 7 * i % 20 for i in range(n)]
    s.run([(i, 1 + 37 * i % 150, rows[i]) for i in reversed(range(n))], "many", sel)
    s.close()


@pytest.mark.parametrize("neox,rotary", [(False, None), (True, 32), (False, 16), (True, 0)])
def test_rotations(hip, neox, rotary):
    for half in (True, False):
        s = Session(hip, 4, 2, 64, half, 32, [100], neox=neox, rotary=rotary)
        s.run([(0, 0, 40)])
        s.run([(0, 40, 1)])
        s.check_cache()
        s.close()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("window", [1, 5, 32, 33, 100])
def test_windows(hip, half, window):
    s = Session(hip, 6, 2, 64, half, 32, [300, 300], window=window)
    s.run([(0, 0, 150), (1, 0, 33)])
    s.run([(0, 150, 1), (1, 33, 4)])
    s.run([(0, 151, 70), (1, 37, 1)])
    s.close()


@pytest.mark.parametrize("heads,hkv,d,half,page", [SHAPES[i] for i in (0, 2, 4, 8, 10)], ids=[IDS[i] for i in (0, 2, 4, 8, 10)])
def test_norms_and_scale(hip, heads, hkv, d, half, page):
    """QK-norm on both sides, one side or none, the value norm, and a scale of one."""
    w = [1.0 + 0.1 * synth.normal(5, t, (d,)) for t in "qk"]
    for qw, kw, value in ((w[0], w[1], False), (None, w[1], True), (w[0], None, False)):
        s = Session(hip, heads, hkv, d, half, page, [90], norm=(qw, kw, 1e-6), value_rms=value, scale=0.25)
        s.run([(0, 0, 45)])
        s.run([(0, 45, 1)])
        s.run([(0, 46, 34)])
        s.check_cache()
        s.close()


@pytest.mark.parametrize("half", [True, False])
def test_long_contexts_are_split(hip, half):
    """One token far back, cut over many workgroups, and several of different lengths beside it."""
    s = Session(hip, 4, 2, 64, half, 64, [9000, 700, 40], max_len=9100)
    for at in range(0, 9000, 3000):
        s.fill([(0, at, 3000)])
    s.run([(1, 0, 699), (2, 0, 39)])
    first, *_ = s.run([(0, 9000, 1)])
    s.run([(2, 39, 1), (0, 9001, 1), (1, 699, 1)])
    s.run([(0, 9002, 3)])
    s.close()


@pytest.mark.parametrize("factor", [1e-4, 300.0])
def test_small_and_large_queries(hip, factor):
    """Queries near f16's ends: scores that hardly differ, and scores of which one takes all."""
    s = Session(hip, 4, 2, 64, True, 32, [200], scale=1.0 / factor / 8)
    q, k, v, qn = s.rows([(0, 0, 150)])
    q, qn = q * np.float32(factor), qn * np.float32(factor)
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
    rot, out = rt.DeviceArray(q.size), rt.DeviceArray(q.size)
    s.kv.append_device(s.layer, [(0, 0, 150)], dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, rot.ptr, rot.count)
    s.kv.attend_device(s.layer, [(0, 0, 150)], rot.ptr, rot.count, out.ptr, out.count)
    hip.synchronize()
    qr = rot.download().reshape(qn.shape)
    assert np.abs(qr - qn).max() <= np.abs(qn).max() * 2.0 ** -22  # the factor is no power of two
    s.close_to(out.download(), [(0, 0, 150)], qr)
    s.close()


def put(s, position, keys=None, values=None, sequence=0):
    """Overwrites one position's stored row."""
    st, page = s.kv.storage(0), s.kv.pages(sequence)[position // s.page]
    es, w = (2, 32) if s.half else (4, 16)
    dt = np.float16 if s.half else np.float32
    slot = position % s.page
    for base, x in ((st.keys, keys), (st.values, values)):
        if x is None:
            continue
        for j in range(s.hkv):
            for e in range(s.d):
                at = (int(page) * s.hkv + j) * s.page * s.d + slot // 32 * 32 * s.d
                at += e // w * 32 * w + slot % 32 * w + e % w if base == st.keys else e * 32 + slot % 32
                a = np.full(1, x, dt)
                rt.check(rt.hip().hipMemcpy(base + at * es, a.ctypes.data, es, rt.H2D), "hipMemcpy")


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rows", [4, 70])
def test_masked_rows_may_hold_anything(hip, half, rows):
    """An infinite value at one row of a chunk reaches that row's output and the later ones' (as no finite
    number: an f16 cache's probabilities come in two halves, whose products with it differ in sign), and
    not the earlier ones'; what lies behind the last row is never seen."""
    s = Session(hip, 4, 2, 64, half, 32, [200])
    chunk = [(0, 50, rows)]
    s.run([(0, 0, 50)])
    q, k, v, qn = s.rows(chunk)
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
    rot, out = rt.DeviceArray(q.size), rt.DeviceArray(q.size)
    s.kv.append_device(s.layer, chunk, dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, rot.ptr, rot.count)
    hip.synchronize()
    bad = 2
    put(s, 50 + bad, values=np.inf)
    s.kv.attend_device(s.layer, chunk, rot.ptr, rot.count, out.ptr, out.count)
    hip.synchronize()
    got = out.download().reshape(rows, 4, 64)
    assert not np.isfinite(got[bad:]).any()
    s.close_to(got[:bad], [(0, 50, bad)], qn[:bad])
    # A key that is no number: the rows that see it report it, the others are as they were.
    put(s, 50 + bad, keys=np.nan, values=1.0)
    s.kv.attend_device(s.layer, [(0, 50, bad)], rot.ptr, rot.count, out.ptr, out.count)
    hip.synchronize()
    s.close_to(out.download()[:bad * 256], [(0, 50, bad)], qn[:bad])
    s.kv.attend_device(s.layer, chunk, rot.ptr, rot.count, out.ptr, out.count)
    with pytest.raises(A.AttentionStatusError, match="NON_FINITE"):
        hip.synchronize()
    s.close_to(out.download()[:bad * 256], [(0, 50, bad)], qn[:bad])
    s.close()


def test_forked_sequences_share_their_prefix(hip):
    s = Session(hip, 8, 2, 64, True, 32, [150, 150, 150], bounds=True)
    s.run([(0, 0, 100)])
    s.kv.fork(0, 1, 96)
    s.kv.fork(0, 2, 32)
    for t, n in ((1, 96), (2, 32)):
        s.keys[t], s.values[t] = s.keys[0][:n], s.values[0][:n]
    s.run([(1, 96, 1), (0, 100, 1), (2, 32, 40)], "forked")
    s.kv.clear(0)
    s.keys[0], s.values[0] = s.keys[0][:0], s.values[0][:0]
    s.run([(0, 0, 70), (1, 97, 20), (2, 72, 1)], "after")
    s.check_cache()
    s.close()


SELECTIONS = [A.PageSelection(3, 1, 2), A.PageSelection(0, 0, 1), A.PageSelection(5, 0, 1), A.PageSelection(40, 2, 3)]


@pytest.mark.parametrize("heads,hkv,d,half,page", SHAPES, ids=IDS)
def test_selected_pages(hip, heads, hkv, d, half, page):
    """The pages' bounds, the chosen pages and the attention over them, with fewer pages than a
    selection takes, as many, and more."""
    s = Session(hip, heads, hkv, d, half, page, [12 * page, 300], bounds=True)
    n = 11 * page + page // 2
    s.run([(0, 0, page + 3)], "few", SELECTIONS[0])
    s.fill([(0, page + 3, n - page - 3), (1, 0, 65)])
    for i, sel in enumerate(SELECTIONS):
        s.run([(1, 65 + i, 1), (0, n + i, 1)], "token", sel)
    s.run([(0, n + 3, 5)], "rows", SELECTIONS[0])
    es, dt = (2, np.float16) if half else (4, np.float32)
    for t in (0, 1):
        want = s.bounds_of(t)
        for i, p in enumerate(s.kv.pages(t)[:len(want)]):
            got = np.empty((hkv, 2, d), dt)
            rt.check(rt.hip().hipMemcpy(got.ctypes.data, s.kv.storage(0).bounds + int(p) * got.nbytes, got.nbytes, rt.D2H), "copy")
            np.testing.assert_array_equal(got.transpose(1, 0, 2), want[i], f"bounds of page {i} of {t}")
    s.close()


@pytest.mark.parametrize("pages", [129, 1100, 5000])
def test_selection_of_many_pages(hip, pages):
    """Page counts past one workgroup's and past a round of the final pick; the oracle takes the stored
    bounds as they are."""
    hkv, d, n = 2, 32, pages * 32
    kv = hip.paged_kv_cache(1, n, pages, 32, hkv, d, True, 1, True)
    kv.reserve(0, n)
    bounds = synth.normal(3, "bounds", (pages, hkv, 2, d)).astype(np.float16)
    bounds = np.sort(bounds, axis=2)
    bounds[pages // 2] = bounds[pages // 3]          # equal scores: the lower page is taken
    bounds[pages // 2 + 1] = bounds[pages // 3]
    rt.check(rt.hip().hipMemcpy(kv.storage(0).bounds, bounds.ctypes.data, bounds.nbytes, rt.H2D), "copy")
    kv.set_length(0, 0, n)
    layer = A.AttentionLayer(0, 6)
    q = synth.normal(3, "q", (2, 6 * d))
    dq = rt.DeviceArray.from_host(q)
    b = bounds.astype(np.float64)
    for top in (1, 7, 64, pages // 3 + 5, pages - 4):
        sel = A.PageSelection(top, 1, 2)
        out = rt.DeviceArray(2 * hkv * sel.budget, np.uint32)
        hip.synchronize()
        kv.select_device(layer, [(0, n - 2, 2)], sel, dq.ptr, dq.count, out.ptr, out.count)
        hip.synchronize()
        got = out.download().reshape(2, hkv, sel.budget)
        for r in range(2):
            for j in range(hkv):
                x = q.reshape(2, 6, d)[r, 3 * j:3 * j + 3].astype(np.float64)
                score = np.maximum(x[:, None] * b[None, :, j, 0], x[:, None] * b[None, :, j, 1]).sum(-1).max(0)
                score[:1] = score[-2:] = np.inf
                np.testing.assert_array_equal(got[r, j], np.sort(np.argsort(-score, kind="stable")[:sel.budget]))
    kv.close()


def test_selection_in_several_launches(hip):
    """A prompt whose rows' scores take more than one launch may hold, and whose rows see page counts below,
    at and above what a selection takes."""
    hkv, d, pages, rows = 2, 32, 5000, 1000
    n = pages * 32
    kv = hip.paged_kv_cache(1, n, pages, 32, hkv, d, True, 1, True)
    kv.reserve(0, n)
    bounds = np.sort(synth.normal(4, "bounds", (pages, hkv, 2, d)).astype(np.float16), axis=2)
    rt.check(rt.hip().hipMemcpy(kv.storage(0).bounds, bounds.ctypes.data, bounds.nbytes, rt.H2D), "copy")
    kv.set_length(0, 0, n)
    q = synth.normal(4, "q", (rows, 6 * d))
    dq, sel = rt.DeviceArray.from_host(q), A.PageSelection(9, 2, 3)
    out = rt.DeviceArray(rows * hkv * sel.budget, np.uint32)
    b = bounds.astype(np.float64)
    for start in (0, n - rows):
        hip.synchronize()
        kv.select_device(A.AttentionLayer(0, 6), [(0, start, rows)], sel, dq.ptr, dq.count, out.ptr, out.count)
        hip.synchronize()
        got = out.download().reshape(rows, hkv, sel.budget)
        for r in (0, 1, 4, 5, 200, 447, 448, 449, 479, 480, 511, 512, 653, 654, 655, 816, 998, 999):
            seen = (start + r) // 32 + 1
            for j in range(hkv):
                want = np.full(sel.budget, A.NO_PAGE, np.uint32)
                if seen <= sel.budget:
                    want[:seen] = np.arange(seen)
                else:
                    x = q.reshape(rows, 6, d)[r, 3 * j:3 * j + 3].astype(np.float64)
                    score = np.maximum(x[:, None] * b[None, :seen, j, 0], x[:, None] * b[None, :seen, j, 1]).sum(-1).max(0)
                    score[:2] = score[seen - 3:] = np.inf
                    want = np.sort(np.argsort(-score, kind="stable")[:sel.budget])
                np.testing.assert_array_equal(got[r, j], want, f"row {r} at {start}, kv head {j}")
    kv.close()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("case", ["zero", "tiny", "small", "large", "one", "nan", "inf", "equal", "near", "infinite"])
@pytest.mark.parametrize("rows", [1, 3])
def test_selection_does_not_depend_on_rounding(hip, rows, half, case):
    """Scores that are equal, that differ in their last bits, that underflow or overflow 32 bits or are no
    numbers: the pages are those of scores in 64 bits, ties to the lowest."""
    hkv, d, n = 2, 64, 300
    kv = hip.paged_kv_cache(1, n * 32, n, 32, hkv, d, half, 1, True)
    kv.reserve(0, n * 32)
    dt = np.float16 if half else np.float32
    bounds = np.sort(synth.normal(5, "bounds", (n, hkv, 2, d)).astype(dt), axis=2)
    q = synth.normal(5, "q", (3, 6, d)).astype(np.float32)
    if case == "zero":
        q[1] = 0.0
    elif case in ("tiny", "small", "large"):
        q = (q * np.float32({"tiny": 1e-38, "small": 1e-30, "large": 1e37}[case])).astype(np.float32)
    elif case == "one":
        q[:, :, 1:] = 0.0
    elif case in ("nan", "inf"):
        q[1, 4, 3] = np.float32(case)
    elif case == "equal":
        bounds[20:200] = bounds[20]
    elif case == "infinite":                   # no number among a page's keys, and keys that overflowed
        bounds[50, :, 0, 5], bounds[50, :, 1, 5] = np.inf, -np.inf
        bounds[60, :, 0, 6] = bounds[70, 0, 0, 7] = -np.inf
        bounds[80, :, 1, 8] = np.inf
        q[0, :, 6] = q[1, :, 8] = 0.0
    else:
        bounds[20:200] = bounds[20]
        for i in range(20, 200):
            bounds[i, :, 1, i % d] += dt(2.0 ** -9 if half else 2.0 ** -22) * dt(i % 7)
    rt.check(rt.hip().hipMemcpy(kv.storage(0).bounds, bounds.ctypes.data, bounds.nbytes, rt.H2D), "copy")
    kv.set_length(0, 0, n * 32)
    q = q[1:2] if rows == 1 else q
    dq, sel = rt.DeviceArray.from_host(q.reshape(-1)), A.PageSelection(23, 2, 1)
    out = rt.DeviceArray(rows * hkv * sel.budget, np.uint32)
    hip.synchronize()
    kv.select_device(A.AttentionLayer(0, 6), [(0, n * 32 - rows, rows)], sel, dq.ptr, dq.count, out.ptr, out.count)
    hip.synchronize()
    got, b = out.download().reshape(rows, hkv, sel.budget), bounds.astype(np.float64)
    for r in range(rows):
        for j in range(hkv):
            x = q[r, 3 * j:3 * j + 3].astype(np.float64)
            with np.errstate(invalid="ignore"):
                score = np.maximum(x[:, None] * b[None, :, j, 0], x[:, None] * b[None, :, j, 1]).sum(-1).max(0)
            score[np.isnan(score)] = np.inf
            score[:2] = score[-1:] = np.inf
            want = np.argsort(-score[2:n - 1], kind="stable")[:23] + 2
            np.testing.assert_array_equal(got[r, j], np.concatenate([[0, 1], np.sort(want), [n - 1]]))
    kv.close()


def test_infinite_bounds_are_chosen(hip):
    """A page with an overflowed key counts as the highest, also where a zero of the query meets it."""
    s = Session(hip, 4, 2, 64, True, 32, [400], bounds=True)
    s.run([(0, 0, 300)])
    q, k, v, _ = s.rows([(0, 300, 1)])
    st, page = s.kv.storage(0), int(s.kv.pages(0)[4])
    inf = np.full(1, np.inf, np.float16)
    rt.check(rt.hip().hipMemcpy(st.bounds + (page * 2 * 2 * 64 + 64) * 2, inf.ctypes.data, 2, rt.H2D), "copy")
    q[:, 0] = 0.0
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (np.abs(q), k, v))
    out, pages = rt.DeviceArray(q.size), rt.DeviceArray(2 * 3, np.uint32)
    layer = A.AttentionLayer(0, 4)
    s.kv.append_device(layer, [(0, 300, 1)], 0, 0, dk.ptr, dk.count, dv.ptr, dv.count)
    s.kv.select_device(layer, [(0, 300, 1)], A.PageSelection(1, 1, 1), dq.ptr, dq.count, pages.ptr, pages.count)
    hip.synchronize()
    assert pages.download().reshape(2, 3)[0].tolist() == [0, 4, 9]
    s.close()


def test_wrong_page_lists_are_reported(hip):
    """Pages past the row's own, and lists that do not ascend, are left out and reported; the rest of the
    list is attended to."""
    s = Session(hip, 4, 1, 64, True, 32, [200])
    s.run([(0, 0, 150)])
    q, k, v, qn = s.rows([(0, 150, 1)])
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
    rot, out = rt.DeviceArray(q.size), rt.DeviceArray(q.size)
    s.kv.append_device(s.layer, [(0, 150, 1)], dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, rot.ptr, rot.count)
    for lists, used, wrong in (([0, 2, 4], [0, 2, 4], False), ([1, 3, A.NO_PAGE], [1, 3], False), ([0, 5, 9], [0], True),
                               ([2, 2, 4], [2, 4], True), ([3, 1, 4], [3, 4], True), ([1, 1 << 20, A.NO_PAGE], [1], True)):
        pages = rt.DeviceArray.from_host(np.array(lists, np.uint32))
        hip.synchronize()
        s.kv.attend_device(s.layer, [(0, 150, 1)], rot.ptr, rot.count, out.ptr, out.count, pages.ptr, 3, 3)
        if wrong:
            with pytest.raises(A.AttentionStatusError, match="OUT_OF_RANGE"):
                hip.synchronize()
        else:
            hip.synchronize()
        s.close_to(out.download(), [(0, 150, 1)], qn, [[used]])
    s.close()


def test_host_buffers(hip):
    s = Session(hip, 8, 2, 64, True, 32, [300, 300], bounds=True)
    for chunks, sel in (([(0, 0, 200), (1, 0, 7)], None), ([(1, 7, 1), (0, 200, 3)], A.PageSelection(2, 1, 1))):
        q, k, v, qn = s.rows(chunks)
        got = s.kv.forward(s.layer, chunks, q, k, v, sel)
        chosen = s.selected(chunks, qn, sel) if sel else None
        if sel:
            got, pages = got
            for i in range(len(chosen)):
                for j in range(2):
                    assert pages[i, j][:len(chosen[i][j])].tolist() == chosen[i][j].tolist()
        s.close_to(got, chunks, qn, chosen)
    s.close()


@pytest.mark.parametrize("selection", [None, A.PageSelection(4, 1, 2)])
def test_replayed_graphs(hip, selection):
    """A captured step is replayed several times, with eager calls of other shapes (which use the same
    scratch) and waits between, and gives the eager bits each time."""
    s = Session(hip, 8, 2, 128, True, 32, [4000, 600, 90], max_len=4100, bounds=True)
    for at in range(0, 3900, 1300):
        s.fill([(0, at, 1300)] if at else [(0, 0, 1300), (1, 0, 555), (2, 0, 77)])
    chunks = [(2, 77, 1), (0, 3900, 1), (1, 555, 4)]
    q, k, v, _ = s.rows(chunks)
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
    out = rt.DeviceArray(q.size)
    budget = selection.budget if selection else 0
    pages = rt.DeviceArray(6 * 2 * max(budget, 1), np.uint32)

    def step():
        s.kv.forward_device(s.layer, chunks, dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, out.ptr, out.count,
                            selection, pages.ptr if selection else 0, pages.count if selection else 0)

    step()
    hip.synchronize()
    want, want_pages = out.download(), pages.download()
    graph = rt.Graph(hip.stream(), step)
    for turn in range(4):
        out.upload(np.full(q.size, np.nan, np.float32))
        hip.synchronize()
        graph.launch()
        if turn % 2:
            hip.synchronize()
        other, rot = rt.DeviceArray(q.size), rt.DeviceArray.from_host(q)
        s.kv.attend_device(s.layer, [(1, 100, 3), (0, 3000, 1)], rot.ptr, rot.count, other.ptr, other.count)
        hip.synchronize()
        np.testing.assert_array_equal(out.download(), want)
        if selection:
            np.testing.assert_array_equal(pages.download(), want_pages)
    graph.destroy()
    s.close()


def test_results_do_not_depend_on_what_runs_beside(hip):
    """A sequence's tokens give the same bits alone and in a batch of the same split."""
    s = Session(hip, 4, 2, 64, True, 32, [500, 500], max_len=600)
    s.run([(0, 0, 400), (1, 0, 400)])
    q, k, v, _ = s.rows([(0, 400, 1), (1, 400, 1)])
    dq, dk, dv = (rt.DeviceArray.from_host(x) for x in (q, k, v))
    out, alone = rt.DeviceArray(q.size), rt.DeviceArray(q.size)
    for _ in range(3):
        s.kv.forward_device(s.layer, [(0, 400, 1), (1, 400, 1)], dq.ptr, dq.count, dk.ptr, dk.count, dv.ptr, dv.count, out.ptr, out.count)
        for i in range(2):
            s.kv.forward_device(s.layer, [(i, 400, 1)], dq.at(256 * i), 256, dk.at(128 * i), 128, dv.at(128 * i), 128,
                                alone.at(256 * i), 256)
        hip.synchronize()
        np.testing.assert_array_equal(out.download(), alone.download())
    s.close()
