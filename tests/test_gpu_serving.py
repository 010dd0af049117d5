"""The serving operators (include/vitna_serve.h) against plain implementations in 64 bits.

Attention's bound, element by element. The kernels may take a product of float32 operands from two bfloat16 parts of each
(a part rounds by at most 2^-8 of its value, so hi + lo leaves 2^-16, and the product of the two lo parts, dropped, is
2^-16 again): 3 2^-16 of |q_d k_d|, and HD adds of 2^-24. A score is then off by es = scale sum|q_d k_d| (3 2^-16 + HD
2^-24) + |s| 2^-22 (its scaling and the exponential's argument), a softmax weight by a factor within exp(2 max es), and
the weighted values by 3 2^-16 of the sum of p|v|, plus 2^-23 a position for the sums: the bound is
(2.2 max es + 3 2^-16 + (N + 8) 2^-23) sum p|v|.
The same roundings at random (a part's error has a root mean square of 1.6e-3 = 0.4 2^-8) leave 4.2e-6 of a product, so
6.3e-6 of the scores' 1.5 units and 4.2e-6 of the values: 7.6e-6 of the outputs' 2-norm; 2e-5 is asked for.
Which positions a row sees is tested apart from these, exactly: with queries of zero every weight is the same, and
values of whole numbers then count the positions (float32 holds the counts, and the division by the number of positions
leaves less than half a count).
"""
import ctypes as C

import numpy as np
import pytest

import vitna_amd as va
from test_zz_no_alloc import DeviceBuffer

pytestmark = pytest.mark.gpu

U = 2.0 ** -16
DT = {"f32": va.F32, "f16": va.F16, "bf16": va.BF16}


def to_bytes(x, dtype):
    """float32 x as dtype's bits, and the values those hold."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x
    if dtype == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    with np.errstate(invalid="ignore"):
        b = x.view(np.uint32)
        r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(x), np.uint16(0x7fc0), r)
    return r, (r.astype(np.uint32) << 16).view(np.float32)


class Device:
    """Buffers of one test, freed at its end."""

    def __init__(self):
        self.all = []

    def __enter__(self):
        return self

    def __exit__(self, *_):
        for b in self.all:
            b.free()

    def empty(self, nbytes):
        b = DeviceBuffer(max(int(nbytes), 16))
        self.all.append(b)
        return b

    def put(self, a):
        b = self.empty(a.nbytes)
        b.put(a)
        return b


def runtime():
    rt = C.CDLL("libamdhip64.so.7")
    rt.hipStreamCreateWithFlags.argtypes = [C.POINTER(C.c_void_p), C.c_uint]
    rt.hipStreamSynchronize.argtypes = [C.c_void_p]
    rt.hipStreamDestroy.argtypes = [C.c_void_p]
    rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    rt.hipGraphExecDestroy.argtypes = [C.c_void_p]
    rt.hipGraphDestroy.argtypes = [C.c_void_p]
    return rt


def visible(pos, window, sinks):
    t = np.arange(pos + 1)
    return t[(t > pos - window) | (t < sinks)] if window else t


class Cache:
    """Keys and values [seqs][ctx][kv][hd] as given values, on the device in a layout of one of three kinds."""

    def __init__(self, dev, dtype, seqs, ctx, kv, hd, layout="plain", seed=1, k=None, v=None):
        r = np.random.RandomState(seed)
        self.dtype, self.seqs, self.ctx, self.kv, self.hd = dtype, seqs, ctx, kv, hd
        k = r.standard_normal((seqs, ctx, kv, hd)) if k is None else k
        v = r.standard_normal((seqs, ctx, kv, hd)) if v is None else v
        kb, self.k = to_bytes(k, dtype)
        vb, self.v = to_bytes(v, dtype)
        if layout == "plain":
            self.strides = dict()
            lay = lambda b: b  # noqa: E731
        elif layout == "heads":  # [seq][head][pos][dim]
            self.strides = dict(seq_stride=kv * ctx * hd, pos_stride=hd, head_stride=ctx * hd)
            lay = lambda b: b.transpose(0, 2, 1, 3)  # noqa: E731
        else:  # the second of three layers, with gaps between positions
            self.strides = dict(seq_stride=3 * ctx * (kv * hd + 32), pos_stride=kv * hd + 32)

            def lay(b):
                full = np.full((seqs, 3, ctx, kv * hd + 32), np.nan, np.float32)
                full, _ = to_bytes(full, dtype)
                full[:, 1, :, :kv * hd] = b.reshape(seqs, ctx, kv * hd)
                return full
        self.kd = dev.put(np.ascontiguousarray(lay(kb)))
        self.vd = dev.put(np.ascontiguousarray(lay(vb)))
        skip = ctx * (kv * hd + 32) * (4 if dtype == "f32" else 2) if layout == "gaps" else 0
        self.at = (self.kd.p.value + skip, self.vd.p.value + skip)

    def view(self, heads, window=0, sinks=0, scale=0.0):
        return va.kv_view(*self.at, DT[self.dtype], heads, self.kv, self.hd, self.ctx, self.seqs, window=window, sinks=sinks, scale=scale,
                          **self.strides)

    def attend(self, q, rows, window, sinks, scale=0.0):
        """(out, bound) in 64 bits of queries [n][heads][hd]; rows (seq, pos, base, shared)."""
        n, heads, hd = q.shape
        G = heads // self.kv
        out, bound = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
        scale = scale or 1.0 / np.sqrt(hd)
        for i, (seq, pos, base, shared) in enumerate(rows):
            if not (0 <= seq < self.seqs and 0 <= pos < self.ctx and shared >= 0 and (shared == 0 or 0 <= base < self.seqs)):
                continue
            t = visible(pos, window, sinks)
            src = np.where(t < shared, base if shared else seq, seq)
            K, V = self.k[src, t].astype(np.float64), self.v[src, t].astype(np.float64)
            for h in range(heads):
                k, v, x = K[:, h // G], V[:, h // G], q[i, h].astype(np.float64)
                s = scale * (k @ x)
                es = np.max(scale * (np.abs(k) @ np.abs(x)) * (3 * U + hd * 2.0 ** -24) + np.abs(s) * 2.0 ** -22)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = p @ v
                bound[i, h] = (2.2 * es + 3 * U + (len(t) + 8) * 2.0 ** -23) * (p @ np.abs(v))
        return out, bound


def check(got, want, bound, what=""):
    over = np.abs(got - want) - bound
    assert np.all(over <= 0), (what, "worst", float(over.max()), np.unravel_index(int(over.argmax()), over.shape))
    norm = np.linalg.norm(want)
    if norm:
        rel = np.linalg.norm(got - want) / norm
        assert rel <= 2e-5, (what, "2-norm", rel)
        return rel
    return 0.0


def rows_call(dev, cache, q, rows, window=0, sinks=0, own_max=0, shared_max=0, q_gap=0, out_gap=0, scale=0.0, stream=0, in_place=False):
    n, heads, hd = q.shape
    qs, os_ = heads * hd + q_gap, heads * hd + out_gap
    flat = np.full((n, qs), np.nan, np.float32)
    flat[:, :heads * hd] = q.reshape(n, -1)
    qd = dev.put(flat)
    od = qd if in_place else dev.put(np.full((n + 1, os_), 7.0, np.float32))
    rd = dev.put(np.array(rows, np.int32).reshape(-1, 4))
    view = cache.view(heads, window, sinks, scale)
    need = va.attention_rows_work(view, n, own_max, shared_max)
    wd = dev.put(np.full(need // 4 + 4, np.nan, np.float32))
    va.attention_rows(view, qd.p.value, rd.p.value, n, od.p.value, wd.p.value, need, own_max=own_max, shared_max=shared_max, q_stride=qs,
                      out_stride=qs if in_place else os_, stream=stream)
    if in_place:
        return od.get((n, qs), np.float32)[:, :heads * hd].reshape(n, heads, hd)
    out = od.get((n + 1, os_), np.float32)
    assert np.all(out[n] == 7.0) and np.all(out[:n, heads * hd:] == 7.0), "written outside the rows"
    assert np.all(np.isnan(wd.get((need // 4 + 4,), np.float32)[need // 4:])), "written behind the workspace"
    return out[:n, :heads * hd].reshape(n, heads, hd)


def run_call(dev, cache, q, seq, pos0, window=0, sinks=0, q_gap=0, out_gap=0, stream=0):
    n, heads, hd = q.shape
    qs, os_ = heads * hd + q_gap, heads * hd + out_gap
    flat = np.full((n, qs), np.nan, np.float32)
    flat[:, :heads * hd] = q.reshape(n, -1)
    qd, od = dev.put(flat), dev.put(np.full((n + 1, os_), 7.0, np.float32))
    view = cache.view(heads, window, sinks)
    need = va.attention_run_work(view, pos0, n)
    wd = dev.put(np.full(need // 4 + 4, np.nan, np.float32))
    va.attention_run(view, seq, pos0, qd.p.value, n, od.p.value, wd.p.value, need, q_stride=qs, out_stride=os_, stream=stream)
    out = od.get((n + 1, os_), np.float32)
    assert np.all(out[n] == 7.0) and np.all(out[:n, heads * hd:] == 7.0), "written outside the rows"
    assert np.all(np.isnan(wd.get((need // 4 + 4,), np.float32)[need // 4:])), "written behind the workspace"
    return out[:n, :heads * hd].reshape(n, heads, hd)


def queries(n, heads, hd, seed=5):
    return (1.5 * np.random.RandomState(seed).standard_normal((n, heads, hd))).astype(np.float32)


SHAPES = [("f32", 32, 4, 128, "plain"), ("f32", 16, 16, 128, "heads"), ("f32", 8, 2, 64, "gaps"), ("f32", 6, 2, 128, "plain"),
          ("f32", 16, 1, 64, "heads"), ("f16", 16, 2, 128, "plain"), ("f16", 12, 4, 64, "gaps"), ("bf16", 16, 4, 128, "gaps"),
          ("bf16", 5, 1, 64, "plain"), ("bf16", 4, 4, 128, "heads")]
IDS = ["%s-%d-%d-%d-%s" % s for s in SHAPES]


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 4), (100, 70), (1000, 3)])
def test_rows_of_their_own(shape, window, sinks):
    """Ragged rows, from one position to several tiles, with and without a window; padding and rows outside the cache."""
    dtype, heads, kv, hd, layout = shape
    with Device() as dev:
        cache = Cache(dev, dtype, 7, 330, kv, hd, layout)
        pos = [0, 1, 63, 64, 65, 200, 329, -1, 330, 17, 18]
        rows = [(i % 7, p, 0, 0) for i, p in enumerate(pos)]
        rows[9], rows[10] = (7, 17, 0, 0), (-1, 18, 0, 0)
        q = queries(len(rows), heads, hd)
        want, bound = cache.attend(q, rows, window, sinks)
        for own_max in (0, 5):
            check(rows_call(dev, cache, q, rows, window, sinks, own_max=own_max, q_gap=8, out_gap=4), want, bound, own_max)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5), (1, 1)])
def test_rows_that_share(shape, window, sinks):
    """Groups of rows behind prefixes of several lengths, in no order of tiles; rows of a group at different positions, one
    inside the prefix, rows without a prefix, padding between; the prefix as its own part (shared_max 0) and apart."""
    dtype, heads, kv, hd, layout = shape
    with Device() as dev:
        cache = Cache(dev, dtype, 9, 400, kv, hd, layout, seed=2)
        rows = []
        for base, shared, many in ((0, 130, 5), (4, 64, 1), (4, 1, 3), (5, 300, 18), (0, 0, 2), (2, 399, 4), (2, 63, 3)):
            rows += [((base + j) % 9, min(399, shared + (j * j) % 90), base, shared) for j in range(many)]
        rows += [(1, 100, 3, 250), (1, 250, 3, 250), (1, 249, 3, 250)]  # the first and last inside the prefix
        rows.insert(7, (0, -1, 0, 0))
        rows.insert(20, (0, 390, 9, 200))   # no such prefix
        rows.insert(21, (0, 390, 5, -3))
        rows.insert(22, (0, 390, -1, 0))    # nothing shared: the base does not matter
        q = queries(len(rows), heads, hd, 6)
        want, bound = cache.attend(q, rows, window, sinks)
        for own_max, shared_max in ((0, 0), (90, 399), (1, 1), (400, 400)):
            check(rows_call(dev, cache, q, rows, window, sinks, own_max, shared_max, out_gap=12), want, bound, (own_max, shared_max))


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_many_groups_in_a_tile(shape, window, sinks):
    """More groups than a short prefix is cut into parts; several groups of many columns next to each other and between
    those of few; a group that two tiles share."""
    dtype, heads, kv, hd, layout = shape
    G = heads // kv
    with Device() as dev:
        cache = Cache(dev, dtype, 11, 260, kv, hd, layout, seed=15)
        many = -(-33 // G)  # rows of just more than 32 columns
        sizes = [2] * 17 + [1, many, many, many + 1, 1, many, 3, 1, 1, 1, 2 * many, 1, many]
        rows = []
        for i, size in enumerate(sizes):
            base, shared = (3 * i) % 11, (40 + i if i % 3 else 200 - 5 * i)
            rows += [((base + 1 + j) % 11, min(259, shared + (7 * j) % 50), base, shared) for j in range(size)]
        q = queries(len(rows), heads, hd, 16)
        want, bound = cache.attend(q, rows, window, sinks)
        for own_max, shared_max in ((60, 200), (260, 260), (60, 40)):
            check(rows_call(dev, cache, q, rows, window, sinks, own_max, shared_max), want, bound, (own_max, shared_max))


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("n,pos0,window,sinks", [(1, 0, 0, 0), (1, 399, 33, 2), (2, 63, 1, 0), (37, 0, 0, 0), (37, 5, 20, 3), (130, 270, 64, 100),
                                                 (301, 99, 128, 1), (400, 0, 90, 4)])
def test_runs(shape, n, pos0, window, sinks):
    dtype, heads, kv, hd, layout = shape
    with Device() as dev:
        cache = Cache(dev, dtype, 2, 400, kv, hd, layout, seed=3)
        q = queries(n, heads, hd, 7)
        some = sorted(set([0, n - 1, n // 2, n // 3, min(n - 1, 31), min(n - 1, 32), min(n - 1, 127), min(n - 1, 128)]))
        want, bound = cache.attend(q[some], [(1, pos0 + i, 0, 0) for i in some], window, sinks)
        check(run_call(dev, cache, q, 1, pos0, window, sinks, q_gap=4, out_gap=4)[some], want, bound)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (513, 5), (1000, 0), (7, 64), (2, 1)])
def test_which_positions_are_seen(dtype, window, sinks):
    """Queries of zero: out = the mean of the values of the positions seen. Values count them: dimension d of position t is
    1 where t mod 61 = d (d < 61), so out times the number of positions is how many of each remainder were seen."""
    heads, kv, hd, ctx = 8, 1, 64, 3000
    t = np.arange(ctx)
    v = np.zeros((2, ctx, 1, hd), np.float32)
    v[0, t, 0, t % 61] = 1.0
    v[1, t, 0, t % 61] = 1.0
    v[:, :, 0, 63] = [[1.0], [0.0]]  # and whose they were
    with Device() as dev:
        cache = Cache(dev, dtype, 2, ctx, kv, hd, v=v, k=np.zeros_like(v))

        def count(out, pos, shared=0):
            seen = visible(pos, window, sinks)
            many = np.bincount(seen % 61, minlength=63)
            for h in range(heads):
                got = out[h].astype(np.float64) * len(seen)
                assert np.all(np.abs(got[:63] - many) < 0.4), (pos, shared, np.abs(got[:63] - many).max())
                assert abs(got[63] - np.sum(seen < shared)) < 0.4, (pos, shared)

        pos = [0, 1, 4, 63, 64, 127, 512, 513, 1000, 1063, 1064, 2047, 2999]
        out = rows_call(dev, cache, np.zeros((len(pos), heads, hd), np.float32), [(1, p, 0, 0) for p in pos], window, sinks)
        for i, p in enumerate(pos):
            count(out[i], p)
        rows = [(1, p, 0, s) for s in (1, 64, 65, 1000, 2900) for p in pos]
        for limits in ((0, 0), (3000, 2900), (100, 2900)):
            out = rows_call(dev, cache, np.zeros((len(rows), heads, hd), np.float32), rows, window, sinks, *limits)
            for i, (_, p, _, s) in enumerate(rows):
                count(out[i], p, s)
        for n, pos0 in ((1100, 1900), (130, 0)):
            out = run_call(dev, cache, np.zeros((n, heads, hd), np.float32), 1, pos0, window, sinks)
            for i in range(n):
                count(out[i], pos0 + i)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_does_not_matter(dtype, bad):
    """NaN and infinities in keys and values behind a row, before its window and in other sequences leave it as it is; the
    rows that see one are not finite."""
    heads, kv, hd, ctx = 16, 2, 128, 300
    r = np.random.RandomState(8)
    k, v = r.standard_normal((3, ctx, kv, hd)), r.standard_normal((3, ctx, kv, hd))
    clean_k, clean_v = k.copy(), v.copy()
    for at in (30, 150, 299):  # all heads, some dimensions
        k[1, at, :, 5] = bad
        v[1, at, :, 77] = bad
    k[2], v[2] = bad, bad
    with Device() as dev:
        cache = Cache(dev, dtype, 3, ctx, kv, hd, k=k, v=v)
        clean = Cache(dev, dtype, 3, ctx, kv, hd, k=clean_k, v=clean_v)
        for window, sinks in ((0, 0), (50, 8)):
            bads = lambda p: any(t in visible(p, window, sinks) for t in (30, 150, 299))  # noqa: E731
            # a prompt's chunk: rows before and behind the bad positions in one tile
            q = queries(ctx, heads, hd, 9)
            out = run_call(dev, cache, q, 1, 0, window, sinks)
            good = [p for p in range(ctx) if not bads(p)]
            want, bound = clean.attend(q[good], [(1, p, 0, 0) for p in good], window, sinks)
            check(out[good], want, bound, "run")
            for p in set(range(ctx)) - set(good):
                assert not np.isfinite(out[p]).all(), p
            # rows behind a shared prefix that holds one, each with its own window
            rows = [(0, p, 1, 200) for p in range(120, 300, 9)] + [(0, p, 1, 20) for p in range(30, 60)]
            q = queries(len(rows), heads, hd, 10)
            out = rows_call(dev, cache, q, rows, window, sinks, 100, 200)
            sees = [any(t in visible(p, window, sinks) for t in (30, 150, 299) if t < s) for _, p, _, s in rows]
            good = [i for i in range(len(rows)) if not sees[i]]
            want, bound = clean.attend(q[good], [rows[i] for i in good], window, sinks)
            check(out[good], want, bound, "rows")
            for i in range(len(rows)):
                assert sees[i] == (not np.isfinite(out[i]).all()), rows[i]


@pytest.mark.parametrize("dtype,hd,huge", [("f32", 128, 1e30), ("f32", 64, -3e38), ("bf16", 128, -3e38), ("bf16", 64, 1e30), ("f16", 128, 65504.0)])
@pytest.mark.parametrize("window,sinks", [(70, 5), (70, 0), (3, 64), (64, 70), (200, 1)])
def test_large_numbers_that_no_row_sees(dtype, hd, huge, window, sinks):
    """Numbers of the type's largest size where no row looks: before the first row's window, behind the last row, in the
    pieces that a block reads of either side; a query of them leaves the other rows as they are."""
    heads, kv, ctx = 16, 2, 600
    r = np.random.RandomState(21)
    k, v = r.standard_normal((2, ctx, kv, hd)), r.standard_normal((2, ctx, kv, hd))
    with Device() as dev:
        clean = Cache(dev, dtype, 2, ctx, kv, hd, k=k.copy(), v=v.copy())
        for pos0, n in ((303, 200), (257, 20), (64, 130)):
            seen = np.zeros(ctx, bool)
            for p in (pos0, pos0 + n - 1):
                seen[visible(p, window, sinks)] = True
            seen[pos0:pos0 + n] = True
            dirty_k, dirty_v = k.copy(), v.copy()
            dirty_k[:, ~seen], dirty_v[:, ~seen] = huge, huge
            cache = Cache(dev, dtype, 2, ctx, kv, hd, k=dirty_k, v=dirty_v)
            q = queries(n, heads, hd, 22)
            some = sorted({0, 1, n // 2, n - 2, n - 1})
            want, bound = clean.attend(q[some], [(1, pos0 + i, 0, 0) for i in some], window, sinks)
            q[3] = np.float32(1e30)
            q[5] = np.nan
            check(run_call(dev, cache, q, 1, pos0, window, sinks)[some], want, bound, ("run", pos0, n))
            rows = [(0, pos0 + i, 1, pos0 + 1) for i in range(min(n, 40))]
            q = queries(len(rows), heads, hd, 23)
            want, bound = clean.attend(q, rows, window, sinks)
            check(rows_call(dev, cache, q, rows, window, sinks, 100, 600), want, bound, ("rows", pos0, n))


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (2300, 3)])
def test_groups_behind_long_prefixes(shape, window, sinks):
    """Groups of one to fifty rows behind prefixes long enough for every way to take them, several in a tile."""
    dtype, heads, kv, hd, layout = shape
    with Device() as dev:
        cache = Cache(dev, dtype, 7, 2600, kv, hd, layout, seed=28)
        rows = []
        for g, many in enumerate((5, 5, 1, 6, 18, 2, 2, 9, 50, 1, 13, 8)):
            base, shared = g % 7, 2500 - 61 * g
            rows += [((base + 1 + j) % 7, min(2599, shared - 3 + (11 * j) % 80), base, shared) for j in range(many)]
        q = queries(len(rows), heads, hd, 29)
        some = list(range(0, len(rows), 7)) + [len(rows) - 1]
        want, bound = cache.attend(q[some], [rows[i] for i in some], window, sinks)
        check(rows_call(dev, cache, q, rows, window, sinks, 90, 2500)[some], want, bound)


@pytest.mark.parametrize("dtype,heads,kv,hd", [("f32", 16, 1, 64), ("bf16", 2, 2, 128), ("f16", 8, 1, 128)])
def test_thousands_of_rows(dtype, heads, kv, hd):
    """Hundreds of tiles of rows, alone, in groups of one to forty and as one run."""
    n, ctx, seqs = 3001, 3100, 6
    r = np.random.RandomState(24)
    with Device() as dev:
        cache = Cache(dev, dtype, seqs, ctx, kv, hd, seed=25)
        q = queries(n, heads, hd, 26)
        some = sorted(set(r.randint(0, n, 40)) | {0, n - 1})
        rows = [(i % seqs, int(r.randint(-1, 60)), 0, 0) for i in range(n)]
        want, bound = cache.attend(q[some], [rows[i] for i in some], 20, 2)
        check(rows_call(dev, cache, q, rows, 20, 2, 60)[some], want, bound, "alone")
        rows, g = [], 0
        while len(rows) < n:
            g += 1
            rows += [((g + 1 + j) % seqs, 20 + g % 30 + j % 7, g % seqs, 20 + g % 30) for j in range(1 + (g * g) % 40)]
        rows = rows[:n]
        want, bound = cache.attend(q[some], [rows[i] for i in some], 0, 0)
        check(rows_call(dev, cache, q, rows, own_max=8, shared_max=50)[some], want, bound, "groups")
        want, bound = cache.attend(q[some], [(2, 99 + i, 0, 0) for i in some], 40, 3)
        check(run_call(dev, cache, q, 2, 99, 40, 3)[some], want, bound, "run")


def test_wide_scores_and_a_scale():
    """Scores of thousands: one position takes all the weight; and scores all alike, far below zero."""
    with Device() as dev:
        cache = Cache(dev, "f32", 1, 200, 2, 64, seed=4)
        q = queries(3, 8, 64, 11)
        rows = [(0, 199, 0, 0), (0, 100, 0, 0), (0, 64, 0, 0)]
        for scale in (0.01, 40.0):
            want, bound = cache.attend(q, rows, 0, 0, scale)
            got = rows_call(dev, cache, q, rows, scale=scale)
            assert np.all(np.abs(got - want) <= bound), scale
        k = np.full((1, 200, 2, 64), -30.0, np.float32)
        cache = Cache(dev, "f32", 1, 200, 2, 64, k=k)
        q = np.full((3, 8, 64), 30.0, np.float32)
        want, bound = cache.attend(q, rows, 0, 0)
        got = rows_call(dev, cache, q, rows)
        assert np.all(np.abs(got - want) <= bound)


def test_a_cache_past_4_gib():
    """Positions and sequences whose offsets pass 32 bits of bytes and of elements."""
    ctx, kv, hd, seqs = 1 << 21, 2, 128, 5  # 2 GiB of float32 a sequence
    with Device() as dev:
        stride = ctx * kv * hd
        kd, vd = dev.empty(seqs * stride * 4), dev.empty(seqs * stride * 4)
        r = np.random.RandomState(12)
        rows, ks, vs = [(4, ctx - 1, 0, 0), (2, ctx - 9, 4, ctx - 20)], [], []
        rt = runtime()
        rt.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        held = {}
        for seq in (2, 4):
            held[seq] = [r.standard_normal((256, kv, hd)).astype(np.float32) for _ in range(2)]
            for d, a in zip((kd, vd), held[seq]):
                assert rt.hipMemcpy(d.p.value + (seq * stride + (ctx - 256) * kv * hd) * 4, a.ctypes.data, a.nbytes, 1) == 0
        view = va.kv_view(kd.p.value, vd.p.value, va.F32, 8, kv, hd, ctx, seqs, window=100)
        q = queries(2, 8, hd, 13)
        small = Cache(dev, "f32", 5, 256, kv, hd, k=np.stack([held[4][0] if s == 4 else held[2][0] for s in range(5)]),
                      v=np.stack([held[4][1] if s == 4 else held[2][1] for s in range(5)]))
        want, bound = small.attend(q, [(4, 255, 0, 0), (2, 247, 4, 236)], 100, 0)
        qd, rd, od = dev.put(q), dev.put(np.array(rows, np.int32)), dev.empty(q.nbytes)
        for limits in ((0, 0), (100, ctx)):
            need = va.attention_rows_work(view, 2, *limits)
            wd = dev.empty(need)
            va.attention_rows(view, qd.p.value, rd.p.value, 2, od.p.value, wd.p.value, need, own_max=limits[0], shared_max=limits[1])
            check(od.get(q.shape, np.float32), want, bound, limits)
        n = 70
        q = queries(n, 8, hd, 14)
        want, bound = small.attend(q, [(4, 256 - n + i, 0, 0) for i in range(n)], 100, 0)
        qd, od = dev.put(q), dev.empty(q.nbytes)
        need = va.attention_run_work(view, ctx - n, n)
        wd = dev.empty(need)
        va.attention_run(view, 4, ctx - n, qd.p.value, n, od.p.value, wd.p.value, need)
        check(od.get(q.shape, np.float32), want, bound)


def test_in_place_and_deterministic():
    """out may be q; and the same call gives the same bits."""
    with Device() as dev:
        cache = Cache(dev, "f32", 4, 300, 4, 128)
        rows = [(i % 4, 299 - i, 1, 100) for i in range(40)]
        q = queries(40, 32, 128)
        want, bound = cache.attend(q, rows, 0, 0)
        first = rows_call(dev, cache, q, rows, own_max=200, shared_max=100)
        check(first, want, bound)
        assert np.array_equal(first, rows_call(dev, cache, q, rows, own_max=200, shared_max=100, in_place=True))
        assert np.array_equal(first, rows_call(dev, cache, q, rows, own_max=200, shared_max=100))


def test_streams_and_graphs():
    """On a stream of its own, and captured: replays follow what the rows say then; two graphs, each with a workspace."""
    rt = runtime()
    with Device() as dev:
        cache = Cache(dev, "f32", 6, 500, 2, 128)
        q = queries(12, 16, 128)
        view = cache.view(16, 90, 4)
        need = va.attention_rows_work(view, 12, 100, 400)
        qd = dev.put(q)
        s = C.c_void_p()
        assert rt.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        graphs = []
        for k in range(2):
            rd, od, wd = dev.put(np.full((12, 4), -1, np.int32)), dev.put(np.full(q.shape, np.nan, np.float32)), dev.empty(need)
            assert rt.hipStreamBeginCapture(s, 2) == 0
            va.attention_rows(view, qd.p.value, rd.p.value, 12, od.p.value, wd.p.value, need, own_max=100, shared_max=400, stream=s.value)
            g, x = C.c_void_p(), C.c_void_p()
            assert rt.hipStreamEndCapture(s, C.byref(g)) == 0
            assert rt.hipGraphInstantiate(C.byref(x), g, None, None, 0) == 0
            graphs.append((rd, od, g, x))
        for turn in range(4):
            want = []
            for k, (rd, od, g, x) in enumerate(graphs):
                rows = [(i % 6, (97 * i + 31 * turn + 11 * k) % 500, 3, (57 * (i // 4 + turn)) % 400) for i in range(12)]
                rows[turn] = (0, -1, 0, 0)
                rd.put(np.array(rows, np.int32))
                want.append(cache.attend(q, rows, 90, 4))
            for rd, od, g, x in graphs:
                assert rt.hipGraphLaunch(x, s) == 0
            assert rt.hipStreamSynchronize(s) == 0
            for (rd, od, g, x), (w, b) in zip(graphs, want):
                check(od.get(q.shape, np.float32), w, b, turn)
        for rd, od, g, x in graphs:
            assert rt.hipGraphExecDestroy(x) == 0 and rt.hipGraphDestroy(g) == 0
        assert rt.hipStreamDestroy(s) == 0


# --- selection ----------------------------------------------------------------------------------------------------------

def select_want(logits, scores, ended, end, groups, width, keep):
    """(best, parents, tokens) in 64 bits, by the definition."""
    V = logits.shape[1]
    best = np.full((groups, keep), -np.inf)
    par, tok = np.full((groups, keep), -1), np.full((groups, keep), -1)
    for g in range(groups):
        vals = np.full((width, V), -np.inf)
        for b in range(width):
            r = g * width + b
            if not scores[r] > -np.inf:
                continue
            if ended is not None and ended[r]:
                vals[b, end] = scores[r]
                continue
            x = logits[r].astype(np.float64)
            x[np.isnan(x)] = -np.inf
            m = x.max()
            if m == -np.inf:
                continue
            if m == np.inf:
                vals[b] = np.where(x == m, scores[r] - np.log(np.sum(x == m)), -np.inf)
            else:
                vals[b] = scores[r] + ((x - m) - np.log(np.sum(np.exp(x - m))))
        order = np.argsort(-vals.ravel(), kind="stable")[:keep]
        order = order[vals.ravel()[order] > -np.inf]
        best[g, :len(order)] = vals.ravel()[order]
        par[g, :len(order)], tok[g, :len(order)] = order // V, order % V
    return best, par, tok


def select_call(dev, logits, scores, ended, end, groups, width, keep, stride=0, stream=0):
    rows, V = logits.shape
    stride = stride or V
    flat = np.full((rows, stride), 1e30, np.float32)
    flat[:, :V] = logits
    ld, sd = dev.put(flat.ravel()), dev.put(np.ascontiguousarray(scores, np.float32))
    ed = dev.put(np.ascontiguousarray(ended, np.uint8)) if ended is not None else None
    bd, pd, td = (dev.put(np.full(groups * keep + 1, 77, t)) for t in (np.float32, np.int32, np.int32))
    need = va.beam_select_work(groups, width, V, keep)
    wd = dev.put(np.full(need // 4 + 4, np.nan, np.float32))
    va.beam_select(ld.p.value, V, groups, width, keep, sd.p.value, bd.p.value, pd.p.value, td.p.value, wd.p.value, need,
                   ended=ed.p.value if ed else 0, end_token=end, stride=stride, stream=stream)
    out = [d.get((groups * keep + 1,), t) for d, t in ((bd, np.float32), (pd, np.int32), (td, np.int32))]
    assert all(o[-1] == 77 for o in out)
    assert np.all(np.isnan(wd.get((need // 4 + 4,), np.float32)[need // 4:])), "written behind the workspace"
    return [o[:-1].reshape(groups, keep) for o in out]


def check_select(got, want):
    """The same continuations, and their values to float32: a value's rounding is 2^-24 of it, the exponentials' sum is
    within 2^-22 of itself (their arguments' roundings and their own)."""
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), (got[1], want[1], got[2], want[2])
    there = want[1] >= 0
    assert np.all(np.abs(got[0][there] - want[0][there]) <= np.abs(want[0][there]) * 2.0 ** -24 + 2.0 ** -22)
    assert np.all(got[0][~there] == -np.inf)


@pytest.mark.parametrize("groups,width,vocab,keep,stride", [
    (1, 1, 1, 1, 0), (1, 1, 7, 9, 0), (2, 3, 63, 64, 0), (1, 4, 64, 8, 0), (3, 5, 1000, 10, 1001), (1, 64, 1023, 64, 0), (2, 2, 4097, 1, 4099),
    (1, 4, 40000, 8, 0), (2, 32, 16385, 64, 0), (1, 2, 151936, 4, 0), (5, 1, 65537, 33, 0)])
def test_selection(groups, width, vocab, keep, stride):
    r = np.random.RandomState(groups * 1000 + width * 100 + keep)
    rows = groups * width
    logits = (2.0 * r.standard_normal((rows, vocab))).astype(np.float32)
    for i in range(rows):
        logits[i, r.randint(0, vocab, 20)] += 8.0
    scores = (-20.0 + 1.5 * r.standard_normal(rows)).astype(np.float32)
    ended = (r.randint(0, 5, rows) == 0).astype(np.uint8)
    with Device() as dev:
        for e in (None, ended):
            end = vocab // 2
            check_select(select_call(dev, logits, scores, e, end, groups, width, keep, stride),
                         select_want(logits, scores, e, end, groups, width, keep))


def test_selection_of_many_groups():
    r = np.random.RandomState(27)
    groups, width, vocab, keep = 700, 3, 257, 5
    logits = (3.0 * r.standard_normal((groups * width, vocab))).astype(np.float32)
    scores = r.standard_normal(groups * width).astype(np.float32)
    ended = (r.randint(0, 4, groups * width) == 0).astype(np.uint8)
    with Device() as dev:
        check_select(select_call(dev, logits, scores, ended, 9, groups, width, keep), select_want(logits, scores, ended, 9, groups, width, keep))


def test_selection_of_equal_values():
    """Ties, within a beam and between beams of equal logits, go to the lower beam and token; logits that are sorted
    either way; one beam that holds every result."""
    r = np.random.RandomState(3)
    V = 5000
    flat = np.zeros((3, V), np.float32)
    few = r.randint(0, 3, (1, V)).astype(np.float32).repeat(3, 0)
    up = (np.arange(V) * 1e-3 * np.array([[1.0], [1.37], [0.77]])).astype(np.float32)
    one = np.full((3, V), -50.0, np.float32)
    one[1] = np.linspace(0, 9, V)[r.permutation(V)]
    with Device() as dev:
        for logits in (flat, few, np.ascontiguousarray(up[:, ::-1]), up, one):
            for scores in (np.zeros(3, np.float32), np.array([-1, 0, 0], np.float32), np.array([0, -np.inf, -np.inf], np.float32)):
                check_select(select_call(dev, logits, scores, None, 0, 1, 3, 50), select_want(logits, scores, None, 0, 1, 3, 50))


def test_selection_with_nothing_to_choose():
    """-inf and NaN logits, whole rows of them, +inf ones, scores of -inf and NaN, and beams that have ended."""
    r = np.random.RandomState(4)
    V = 3001
    logits = r.standard_normal((8, V)).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, r.randint(0, V, 2000)] = -np.inf
    logits[3, r.randint(0, V, 2000)] = np.nan
    logits[4, [5, 77, 3000]] = np.inf
    logits[5, 4:] = -np.inf
    scores = np.array([-1, -2, -3, -4, -5, -6, np.nan, -np.inf], np.float32)
    with Device() as dev:
        for rows in ([0, 1, 2, 3, 4, 5, 6, 7], [0, 1, 6, 7], [5, 0], [4], [7], [0]):
            for ended in (None, np.array([i == rows[-1] for i in rows], np.uint8)):
                x, s = logits[rows], scores[rows]
                check_select(select_call(dev, x, s, ended, 2, 1, len(rows), 20), select_want(x, s, ended, 2, 1, len(rows), 20))


# --- reordering ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,kv,hd,layout", [("f32", 4, 128, "plain"), ("f32", 1, 64, "heads"), ("f16", 2, 64, "plain"), ("bf16", 3, 128, "heads")])
@pytest.mark.parametrize("groups,width,layers,ctx", [(1, 1, 1, 1), (1, 2, 1, 40), (3, 4, 2, 33), (2, 7, 3, 20), (1, 16, 1, 9), (2, 33, 1, 11), (1, 64, 2, 5)])
def test_reordering(dtype, kv, hd, layout, groups, width, layers, ctx):
    """Any parents, swaps and rings among them, in the order before the call; spans of every length; what is not in a span,
    and sequences that are no beams, as they were; a parent or sequence outside leaves a beam as it is."""
    r = np.random.RandomState(width * 10 + layers)
    seqs = groups * width + 2
    shape = (seqs, layers, ctx, kv, hd) if layout == "plain" else (seqs, layers, kv, ctx, hd)
    size = np.uint32 if dtype == "f32" else np.uint16
    k, v = (r.randint(0, 1 << 16, shape).astype(size) for _ in range(2))
    strides = dict() if layout == "plain" else dict(pos_stride=hd, head_stride=ctx * hd)
    one = kv * hd * ctx
    order = r.permutation(seqs)[:groups * width].astype(np.int32)
    with Device() as dev:
        kd, vd = dev.put(k), dev.put(v)
        view = va.kv_view(kd.p.value, vd.p.value, DT[dtype], kv, kv, hd, ctx, seqs, seq_stride=layers * one, **strides)
        for turn in range(4):
            parents = r.randint(0, width, (groups, width)).astype(np.int32)
            seq_list = order.copy()
            if turn == 1:
                parents[:] = np.roll(np.arange(width), 1)  # a ring
            if turn == 2 and width > 1:
                parents[0, 0], parents[-1, -1] = width, -1
                seq_list[1] = seqs
            spans = np.sort(r.randint(0, ctx + 1, (groups, 2)), 1).astype(np.int32)
            if turn == 0:
                spans[0] = [-3, ctx + 9]
            if turn == 3:
                spans[0] = [ctx, 0]
            wk, wv = k.copy(), v.copy()
            for g in range(groups):
                a, b = max(0, spans[g, 0]), min(ctx, spans[g, 1])
                for i in range(width):
                    p, to = parents[g, i], seq_list[g * width + i]
                    if not (0 <= p < width and 0 <= to < seqs) or not 0 <= seq_list[g * width + p] < seqs or b <= a:
                        continue
                    src = seq_list[g * width + p]
                    if layout == "plain":
                        wk[to, :, a:b], wv[to, :, a:b] = k[src, :, a:b], v[src, :, a:b]
                    else:
                        wk[to, :, :, a:b], wv[to, :, :, a:b] = k[src, :, :, a:b], v[src, :, :, a:b]
            sd, pd, nd = dev.put(seq_list), dev.put(parents), dev.put(spans)
            va.kv_reorder(view, layers, one, sd.p.value, pd.p.value, nd.p.value, groups, width, longest=[0, 1, ctx, 3][turn])
            k, v = kd.get(shape, size), vd.get(shape, size)
            assert np.array_equal(k, wk) and np.array_equal(v, wv), turn


def test_selection_and_reordering_captured():
    """Both in one graph, replayed with other logits: each replay as the calls by themselves."""
    rt = runtime()
    r = np.random.RandomState(9)
    groups, width, V, layers, ctx, kv, hd = 2, 4, 3000, 2, 24, 2, 64
    rows = groups * width
    shape = (rows, layers, ctx, kv, hd)
    with Device() as dev:
        k, v = (r.standard_normal(shape).astype(np.float32) for _ in range(2))
        kd, vd = dev.put(k), dev.put(v)
        view = va.kv_view(kd.p.value, vd.p.value, va.F32, kv, kv, hd, ctx, rows, seq_stride=layers * ctx * kv * hd)
        need = va.beam_select_work(groups, width, V, width)
        ld, sd, wd = dev.empty(rows * V * 4), dev.empty(rows * 4), dev.empty(need)
        bd, pd, td = (dev.empty(rows * 4) for _ in range(3))
        od, nd = dev.put(np.arange(rows, dtype=np.int32)), dev.put(np.array([[3, 20], [0, 24]], np.int32))
        s = C.c_void_p()
        assert rt.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        assert rt.hipStreamBeginCapture(s, 2) == 0
        va.beam_select(ld.p.value, V, groups, width, width, sd.p.value, bd.p.value, pd.p.value, td.p.value, wd.p.value, need, stream=s.value)
        va.kv_reorder(view, layers, ctx * kv * hd, od.p.value, pd.p.value, nd.p.value, groups, width, stream=s.value)
        g, x = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamEndCapture(s, C.byref(g)) == 0
        assert rt.hipGraphInstantiate(C.byref(x), g, None, None, 0) == 0
        for turn in range(4):
            logits = (3.0 * r.standard_normal((rows, V))).astype(np.float32)
            scores = r.standard_normal(rows).astype(np.float32)
            ld.put(logits)
            sd.put(scores)
            assert rt.hipGraphLaunch(x, s) == 0 and rt.hipStreamSynchronize(s) == 0
            want = select_want(logits, scores, None, 0, groups, width, width)
            check_select([d.get((groups, width), t) for d, t in ((bd, np.float32), (pd, np.int32), (td, np.int32))], want)
            for c in (k, v):
                old = c.copy()
                for i in range(rows):
                    a, b = [(3, 20), (0, 24)][i // width]
                    c[i, :, a:b] = old[i // width * width + want[1][i // width, i % width], :, a:b]
            assert np.array_equal(kd.get(shape, np.float32), k) and np.array_equal(vd.get(shape, np.float32), v), turn
        assert rt.hipGraphExecDestroy(x) == 0 and rt.hipGraphDestroy(g) == 0 and rt.hipStreamDestroy(s) == 0


def test_pointers_refused_on_the_gpu():
    """Host addresses among device ones, and an unknown stream's device, are refused before anything runs."""
    with Device() as dev:
        cache = Cache(dev, "f32", 1, 8, 1, 64)
        view = cache.view(1)
        b = dev.empty(1 << 16)
        host = np.zeros(4096, np.float32)
        at = (host.ctypes.data + 15) & ~15
        for q, rows, out, work in ((at, b.p.value, b.p.value, b.p.value), (b.p.value, at, b.p.value, b.p.value), (b.p.value, b.p.value, at, b.p.value),
                                   (b.p.value, b.p.value, b.p.value, at)):
            with pytest.raises(va.VitnaError, match="not device memory"):
                va.attention_rows(view, q, rows, 1, out, work, 1 << 16)
        q = queries(1, 1, 64)
        check(rows_call(dev, cache, q, [(0, 7, 0, 0)]), *cache.attend(q, [(0, 7, 0, 0)], 0, 0))
