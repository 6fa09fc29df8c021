"""Any number of new tokens a sequence over a pool of pages (pages from lengths, append of rows, attention of rows) through the
C ABI, against plain numpy forms: 64 bits for numbers, page by page for tables.

Tolerances as in test_batch_gpu, with u = 2^-24: a sum of n fp32 terms 4 sqrt(n) u times the root of the sum of their squares, a
product, an exponential or a scaling u to 2u of its value. What enters the matrix cores in fewer bits adds its own half step
e: fp32 queries and probabilities as three bf16 (2^-24 left over) or as two f16 (2^-22), probabilities in the cache's type (bf16
2^-8, f16 2^-11), each off by its own amount, so their sum by at most 4 e times the root of the sum of squares. Results in the cache's type round by
that half step once more. Selections, tables and copies are exact."""
import ctypes

import numpy as np
import pytest

from qfix import bf16_round, bf16_to_f32
from test_batch_cpu import INVALID
from test_batch_gpu import PAGE, U, Cache, Hip, from_half, same, to_half, within, workspace

pytestmark = pytest.mark.gpu
INF, NAN = np.float32(np.inf), np.float32(np.nan)


def half_step(st):
    return 2.0 ** -8 if st == 0 else 2.0 ** -11


def one_half(x, st):
    return to_half(np.full(1, x, np.float32), st)[0]


# ------------------------------------------------------------------------------------------- attention
class Rows:
    """Rows of a batch: ranges in another order than the sequences, with rows between them that no sequence names."""

    def __init__(self, c, counts, nH, io, seed=1, gap=2, pad=8, scale=1.5):
        rs = np.random.default_rng(seed)
        self.c, self.nH, self.io, self.width = c, nH, io, nH * c.D + pad
        self.count = np.array(counts, np.int32)
        self.start = np.zeros(c.B, np.int32)
        at = gap
        for b in rs.permutation(c.B):
            self.start[b] = at
            at += max(0, int(self.count[b])) + gap
        self.rows = max(1, at)
        q = np.full((self.rows, self.width), NAN, np.float32)   # nothing reads the rows between, nor the padding
        for b in range(c.B):
            n = max(0, int(self.count[b]))
            q[self.start[b]:self.start[b] + n, :nH * c.D] = rs.standard_normal((n, nH * c.D)) * scale
        self.set(q)

    def set(self, q):
        self.bits = to_half(q, self.c.st) if self.io else q
        self.q = from_half(self.bits, self.c.st) if self.io else q


def attend(mlxr, r, window=0, scale=0.09, work=None, desc=None, stream=None, in_place=False, **over):
    c = r.c
    kv = desc or c.desc()
    d = mlxr.DeviceArray.from_numpy
    before = np.full(r.bits.shape, 7, r.bits.dtype)
    dq = d(r.bits)
    do = dq if in_place else d(before)
    need = mlxr.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(kv), r.nH, r.rows, r.io)
    work = work or workspace(mlxr, need)
    ds, dc = d(over.get("start", r.start)), d(over.get("count", r.count))
    mlxr.check(mlxr.lib.mlxr_k_paged_attention_rows(ctypes.byref(kv), ds.ptr, dc.ptr, over.get("rows", r.rows), dq.ptr, r.io, r.width, r.nH, window, scale,
                                                    do.ptr, r.width, work.ptr, work.nbytes, stream))
    mlxr.synchronize()
    return do.numpy()


def reference(r, window, scale, start=None, count=None, rows=None):
    """out, its tolerance, and which rows are written."""
    c, D, st = r.c, r.c.D, r.c.st
    G = r.nH // c.nKV
    start, count, rows = r.start if start is None else start, r.count if count is None else count, rows or r.rows
    out, tol, named = np.zeros((r.rows, r.nH, D)), np.zeros((r.rows, r.nH, D)), np.zeros(r.rows, bool)
    scale = float(np.float32(scale))
    e_q = 0.0 if r.io else (2.0 ** -24 if st == 0 else 2.0 ** -22)
    e_p = half_step(st) if r.io else (2.0 ** -24 if st == 0 else 2.0 ** -22)
    for b in range(c.B):
        L, n = int(np.clip(c.lens[b], 0, c.max_len)), max(0, int(count[b]))
        mine = np.arange(n)[(start[b] + np.arange(n) >= 0) & (start[b] + np.arange(n) < rows)]
        if not len(mine):
            continue
        row, at = start[b] + mine, L - n + mine
        named[row] = True
        for h in range(c.nKV):
            (k, there), (v, _) = c.rows(c.k, b, h, L), c.rows(c.v, b, h, L)
            j = np.arange(L)
            seen = there & (j <= at[:, None])
            if window:
                seen &= j > at[:, None] - window
            any_seen = seen.any(1)
            k, v = (np.where(there[:, None], x, 0) for x in (k, v))
            used = seen.any(0)
            k, v = np.where(used[:, None], k, 0), np.where(used[:, None], v, 0)
            for g in range(h * G, h * G + G):
                x = r.q[row, g * D:(g + 1) * D].astype(np.float64)
                s = np.where(seen, scale * (x @ k.T), -np.inf)
                top = np.where(any_seen, s.max(1, initial=-np.inf), 0)[:, None]
                e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                total = e.sum(1, keepdims=True)
                p = e / np.where(total > 0, total, 1)
                root = np.sqrt((x ** 2) @ (k ** 2).T)
                size = np.where(seen, np.abs(s), 0)
                ds = scale * np.where(seen, root, 0) * (4 * np.sqrt(D) * U + 4 * e_q) + 4 * U * size + 2 * U * size.max(1, initial=0)[:, None]
                rel = 2 * ds.max(1, initial=0)[:, None] + 8 * U
                count_seen = np.maximum(seen.sum(1), 1)[:, None]
                o = p @ v
                sq = np.sqrt((p ** 2) @ (v ** 2))
                out[row, g] = o
                t = rel * (p @ np.abs(v)) + 4 * (np.sqrt(count_seen) * U + e_p) * sq + np.abs(o) * (4 * np.sqrt(count_seen) * U * np.sqrt((p ** 2).sum(1, keepdims=True)) + 2 * U)
                tol[row, g] = t * (1 + half_step(st) * r.io) + (half_step(st) * np.abs(o) + (2.0 ** -25 if st else 0)) * r.io
    return out.reshape(r.rows, -1), tol.reshape(r.rows, -1), named


def check(got, r, want, tol, named):
    n = r.nH * r.c.D
    x = from_half(got, r.c.st) if r.io else got
    assert within(np.abs(x[named, :n] - want[named]), tol[named]) <= 1
    assert same(got[~named], np.full_like(got[~named], 7)) and same(got[:, n:], np.full_like(got[:, n:], 7))


TYPES = [(128, 0, 0), (128, 0, 1), (64, 1, 1), (64, 0, 0), (128, 1, 0), (128, 1, 1), (64, 0, 1), (64, 1, 0)]   # D, cache type, q in the cache's type


@pytest.mark.parametrize("nKV,G", [(2, 1), (2, 4), (1, 5), (2, 8), (1, 17), (1, 40)])
@pytest.mark.parametrize("D,st,io", TYPES)
def test_attention_lengths(gpu, nKV, G, D, st, io):
    print(f"[case] {nKV} {G} {D} {st} {io}", flush=True)
    counts = [1, 0, 5, 33, 64, 65, 1, 130, 2, 31, 7, 0]
    lens = [1, 0, 5, 33, 64, 700, 4097, 131, 1000, 95, 65, 300]
    c = Cache(gpu, lens, nKV, D, st, seed=G).up()
    r = Rows(c, counts, nKV * G, io, seed=G)
    check(attend(gpu, r), r, *reference(r, 0, 0.09))


@pytest.mark.parametrize("count,length,nKV,G,D,st,io", [(1, 1, 8, 4, 128, 0, 0), (1, 20011, 2, 5, 128, 0, 1), (600, 600, 2, 4, 128, 0, 1), (300, 5000, 1, 8, 64, 1, 1),
                                                        (513, 3000, 1, 3, 128, 1, 0), (2, 9000, 4, 16, 64, 0, 0), (1500, 1500, 1, 1, 128, 0, 0), (129, 129, 8, 4, 128, 0, 1)])
def test_attention_sizes(gpu, count, length, nKV, G, D, st, io):
    print(f"[case] {count} {length} {nKV} {G} {D} {st} {io}", flush=True)
    c = Cache(gpu, [length], nKV, D, st, seed=count).up()
    r = Rows(c, [count], nKV * G, io, gap=0)
    check(attend(gpu, r), r, *reference(r, 0, 0.09))


@pytest.mark.parametrize("counts,lengths,G,D,st,io", [([60], [9000], 5, 128, 0, 1), ([180, 60], [1500, 9000], 5, 128, 0, 0), ([20], [5000], 4, 64, 1, 1),
                                                      ([30], [14000], 2, 64, 0, 0), ([1], [40000], 1, 128, 0, 1), ([40, 3], [33000, 100], 1, 128, 1, 0)])
def test_attention_of_many_parts(gpu, counts, lengths, G, D, st, io):
    """Few queries and many pages: an item is cut into so many runs that its parts are joined in groups, and twice the same."""
    c = Cache(gpu, lengths, 1, D, st, seed=77).up()
    r = Rows(c, counts, G, io, seed=77)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(c.desc()), r.nH, r.rows, io))
    got = attend(gpu, r, work=work)
    check(got, r, *reference(r, 0, 0.09))
    assert same(attend(gpu, r, work=work), got)


@pytest.mark.parametrize("window", [1, 2, 31, 63, 64, 65, 128, 1000, 1 << 30])
@pytest.mark.parametrize("D,st,io,G", [(128, 0, 1, 4), (64, 1, 0, 3)])
def test_attention_window(gpu, window, D, st, io, G):
    c = Cache(gpu, [1, 64, 150, 2000, 333, 900], 2, D, st, seed=3).up()
    r = Rows(c, [1, 64, 150, 200, 1, 400], 2 * G, io, seed=4)
    check(attend(gpu, r, window=window), r, *reference(r, window, 0.09))


@pytest.mark.parametrize("B,top,G", [(65, 40, 2), (300, 70, 2), (1000, 9, 1)])
def test_attention_many_sequences(gpu, B, top, G):
    rs = np.random.default_rng(B)
    lens = rs.integers(0, 150, B)
    c = Cache(gpu, lens, 1, 64, 0, seed=B).up()
    r = Rows(c, np.minimum(rs.integers(0, top, B), lens), G, 1, seed=B, gap=0)
    check(attend(gpu, r), r, *reference(r, 0, 0.09))


def test_attention_mixed_step(gpu):
    """Chunks among single tokens, far apart in length."""
    lens = [8000, 3, 5000, 64, 128, 7001, 1, 2500]
    c = Cache(gpu, lens, 2, 128, 0, seed=8).up()
    r = Rows(c, [1, 1, 500, 64, 1, 1, 1, 77], 8, 1, seed=8)
    check(attend(gpu, r), r, *reference(r, 0, 0.09))


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_attention_scales(gpu, st, io, scale):
    """Scores of both signs, all equal, and so far apart that nearly every p but the largest is 0."""
    c = Cache(gpu, [200, 70], 2, 128, st, seed=11).up()
    r = Rows(c, [100, 3], 4, io, seed=11)
    want, tol, named = reference(r, 0, abs(scale)) if scale > 0 else (None, None, None)
    if scale <= 0:
        r2 = Rows(c, [100, 3], 4, io, seed=11)
        r2.q = -r.q if scale < 0 else 0 * r.q
        want, tol, named = reference(r2, 0, abs(scale) or 1.0)
    check(attend(gpu, r, scale=scale), r, want, tol, named)


def test_attention_bounds_on_the_device(gpu):
    """Lengths, counts, starts and pages that only the device sees: held in bounds, and nothing else is touched."""
    c = Cache(gpu, [100, 40, 300, 64, 200, 30, 90, 300], 2, 128, 0, seed=21)
    c.lens = np.array([100, 40, 500, 64, -5, 30, 90, 300], np.int32)      # past max_len, negative
    c.table[0, 1], c.table[3, 0] = c.k.shape[0], -9                        # a page behind the pool; a sequence without any page
    c.up()
    r = Rows(c, [70, 45, 20, 10, 5, -3, 40, 30], 4, 0, seed=21)           # 45 rows for 40 slots; a negative count
    want = reference(r, 0, 0.09)
    zero = [r.start[1] + np.arange(5), r.start[3] + np.arange(10), r.start[4] + np.arange(5)]
    got = attend(gpu, r)
    check(got, r, *want)
    n = r.nH * c.D
    for rows in zero:
        assert same(got[rows, :n], np.zeros_like(got[rows, :n]))
    # rows in front of the array and behind it
    start = r.start.copy()
    start[0], start[6], start[7] = -25, r.rows - 11, r.rows + 5
    start[[1, 2, 3, 4]] = [60, 110, 140, 160]
    fits = r.rows - 11
    assert fits > 170
    r.set(np.where(np.isnan(r.q), np.float32(0.25), r.q))
    want = reference(r, 0, 0.09, start=start)
    check(attend(gpu, r, start=start), r, *want)
    start[7] = 2 ** 31 - 10                                                # start + count passes 32 bits
    check(attend(gpu, r, start=start), r, *reference(r, 0, 0.09, start=start.astype(np.int64)))


def test_attention_in_place_and_again(gpu):
    """Over its own queries, and the same bits in a second call with the same workspace."""
    for io in (0, 1):
        c = Cache(gpu, [2000, 64, 700, 1], 2, 128, 0, seed=31).up()
        r = Rows(c, [300, 64, 1, 1], 8, io, seed=31)
        kv = c.desc()
        work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(kv), 8, r.rows, io))
        one, two, over = attend(gpu, r, work=work), attend(gpu, r, work=work), attend(gpu, r, work=work, in_place=True)
        assert same(one, two)
        named, n = reference(r, 0, 0.09)[2], 8 * 128
        assert same(over[named, :n], one[named, :n]) and same(over[~named], r.bits[~named]) and same(over[:, n:], r.bits[:, n:])


def test_attention_shared_pages(gpu):
    """Two sequences over the same prompt's pages, with pages of their own behind."""
    c = Cache(gpu, [200, 200], 2, 128, 0, seed=41, weight=True)
    c.table[1, :3] = c.table[0, :3]
    c.up()
    r = Rows(c, [8, 70], 8, 0, seed=41)
    check(attend(gpu, r), r, *reference(r, 0, 0.09))
    assert same(c.dw.numpy(), c.weight)


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("D", [128, 64])
def test_attention_odd_values_out_of_sight(gpu, st, io, D):
    """NaN and infinities in keys and values that a row does not attend (later tokens of its own chunk, slots in front
    of its window) leave it as it is, to the bit; rows that do attend them get what the formula gives."""
    lens, counts, G, window = [300, 128, 70], [150, 128, 1], 3, 90
    for odd in (NAN, INF, -INF):
        c = Cache(gpu, lens, 1, D, st, seed=51)
        r = Rows(c, counts, G, io, seed=51)
        clean = reference(r, window, 0.09)
        c.up()
        base = attend(gpu, r, window=window)
        check(base, r, *clean)
        at = {0: 222, 1: 64, 2: 3}                       # one slot of each sequence; the third's is in front of every window
        if odd == -INF:
            at[2] = 0
        for pool in (c.k, c.v):
            for b, j in at.items():
                pool[c.table[b, j // PAGE], :, j % PAGE, 5 if odd != odd else slice(None)] = one_half(odd, st)
        c.up()
        got = attend(gpu, r, window=window)
        n = G * D
        for b, j in at.items():
            slot = lens[b] - counts[b] + np.arange(counts[b])
            sees = (slot >= j) & (slot - window < j)
            rows = r.start[b] + np.arange(counts[b])
            x = from_half(got, st) if io else got
            y = from_half(base, st) if io else base
            # a wave that meets such a slot takes all its rows another way: within twice the tolerance, where nothing is seen
            assert within(np.abs(x[rows[~sees], :n] - y[rows[~sees], :n]), 2 * clean[1][rows[~sees]]) <= 1, (odd, b)
            if odd != odd:
                assert np.isnan(x[rows[sees]][:, :n]).any(1).all()


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_attention_infinite_values(gpu, st, io):
    """An infinite value is infinite in every row that attends it, however small its share; with one of the other sign NaN."""
    c = Cache(gpu, [260], 1, 128, st, seed=61)
    put = lambda j, d, x: c.v.__setitem__((c.table[0, j // PAGE], 0, j % PAGE, d), one_half(x, st))  # noqa: E731
    put(100, 7, INF), put(200, 7, -INF), put(150, 9, -INF)
    key = (c.table[0, 100 // PAGE], 0, 100 % PAGE)
    r = Rows(c, [230], 2, io, seed=61)
    c.k[key] = to_half(np.zeros(128, np.float32), st)
    c.up()
    got = attend(gpu, r, scale=30.0)                     # every other score is far above slot 100's 0 or far below
    x = (from_half(got, st) if io else got)[r.start[0] + np.arange(230)][:, :256].reshape(230, 2, 128)
    slot = np.arange(30, 260)
    assert np.isposinf(x[(slot >= 100) & (slot < 200), :, 7]).all() and np.isnan(x[slot >= 200][:, :, 7]).all()
    assert np.isneginf(x[slot >= 150][:, :, 9]).all()
    assert np.isfinite(x[slot < 100]).all() and np.isfinite(np.delete(x, [7, 9], 2)).all()


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_attention_infinite_keys(gpu, st, io):
    """A key whose score is -infinity takes no part, rows that have no other give zeros, +infinity is NaN."""
    D, n = 128, 140
    c = Cache(gpu, [n], 1, D, st, seed=71)
    c.k[c.table[0, 0], 0, :5, 3] = one_half(-INF, st)    # the first five: rows that see no others give zeros
    c.k[c.table[0, 2], 0, 2, 3] = one_half(-INF, st)     # slot 130
    r = Rows(c, [n], 2, io, seed=71)
    q = r.q.copy()
    q[r.start[0]:r.start[0] + n, 3] = np.abs(q[r.start[0]:r.start[0] + n, 3]) + 0.5      # head 0: -infinity
    q[r.start[0]:r.start[0] + n, D + 3] = 1.0
    q[r.start[0] + 138, D + 3] = -1.0                                                      # head 1 of one row: +infinity
    r.set(q)
    c.up()
    got = attend(gpu, r)

    class Gone:   # the same without those slots
        def __getattr__(self, name):
            return getattr(c, name)

        def rows(self, pool, b, h, m):
            x, there = c.rows(pool, b, h, m)
            gone = np.isin(np.arange(m), [0, 1, 2, 3, 4, 130])
            return np.where(gone[:, None], 0, x), there & ~gone
    r.c = Gone()
    want, tol, named = reference(r, 0, 0.09)
    r.c = c
    x = (from_half(got, st) if io else got)[:, :2 * D]
    assert np.isnan(x[r.start[0] + 138, D:]).all()
    rest = named.copy()
    rest[r.start[0] + 138] = False
    assert within(np.abs(x[rest] - want[rest]), tol[rest]) <= 1
    assert within(np.abs(x[r.start[0] + 138, :D] - want[r.start[0] + 138, :D]), tol[r.start[0] + 138, :D]) <= 1
    assert (x[r.start[0] + np.arange(5)] == 0).all()


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 1)])
def test_attention_odd_queries(gpu, st, io):
    """NaN in a query is that head's alone; an infinite one has infinite scores: NaN where one is +infinity, zeros where all are -infinity."""
    D = 128
    c = Cache(gpu, [150], 1, D, st, seed=81)
    for i in range(3):                                   # dimension 6 of every key is below 0
        c.k[c.table[0, i], 0, :min(64, 150 - 64 * i), 6] = one_half(-1.0, st)
    r = Rows(c, [90], 3, io, seed=81)
    want, tol, named = reference(r, 0, 0.09)
    q, s = r.q.copy(), r.start[0]
    q[s + 10, 4], q[s + 20, D + 6], q[s + 33, 2 * D + 6] = NAN, INF, -INF
    r.set(q)
    c.up()
    x = attend(gpu, r)
    x = (from_half(x, st) if io else x)[:, :3 * D]
    assert np.isnan(x[s + 10, :D]).all() and (x[s + 20, D:2 * D] == 0).all() and np.isnan(x[s + 33, 2 * D:]).all()
    ok = np.repeat(named[:, None], 3 * D, 1)
    ok[s + 10, :D] = ok[s + 20, D:2 * D] = ok[s + 33, 2 * D:] = False
    assert within(np.abs(x - want)[ok], tol[ok]) <= 1


def test_attention_is_the_decode_step_of_one_token(gpu):
    """One row a sequence: the single-token call's results, within both tolerances."""
    lens = [1, 64, 65, 4000, 333]
    c = Cache(gpu, lens, 2, 128, 0, seed=91).up()
    r = Rows(c, [1] * 5, 8, 0, seed=91, gap=0, pad=0)
    got = attend(gpu, r)
    kv, q = c.desc(), r.q[r.start]
    dq, out = gpu.DeviceArray.from_numpy(q), gpu.DeviceArray.zeros(q.shape, np.float32)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_work(ctypes.byref(kv), 8))
    gpu.check(gpu.lib.mlxr_k_paged_attention(ctypes.byref(kv), dq.ptr, 1024, 8, 0, 0.09, out.ptr, 1024, None, 1.0, work.ptr, work.nbytes, None))
    gpu.synchronize()
    _, tol, _ = reference(r, 0, 0.09)
    assert within(np.abs(out.numpy() - got[r.start]), 2 * tol[r.start]) <= 1


# ------------------------------------------------------------------------------------------- append
def run_append(mlxr, c, qkv, seq, slot, nH, inv_freq, qn, kn, rot, traditional, positions, eps, rope_scale, io, in_place, q_pad, offset=0):
    d = mlxr.DeviceArray.from_numpy
    rows, kv = len(seq), c.desc()
    flat = np.concatenate([np.zeros(offset, np.float32), qkv.ravel()])
    dx = d(flat)
    width = qkv.shape[1] if in_place else nH * c.D + q_pad
    before = np.full((rows, width), 7, np.uint16 if io else np.float32)
    dq = dx if in_place else d(before)
    up = lambda x: None if x is None else d(x)  # noqa: E731
    di, dqn, dkn, ds, dt, dp = up(inv_freq if rot else None), up(qn), up(kn), up(seq.astype(np.int32)), up(slot.astype(np.int32)), up(positions)
    ptr = lambda x: x.ptr if x else None  # noqa: E731
    x_at = dx.ptr + 4 * offset
    mlxr.check(mlxr.lib.mlxr_k_paged_append_rows(ctypes.byref(kv), x_at, qkv.shape[1], rows, ds.ptr, dt.ptr, ptr(dp), ptr(di), rope_scale, ptr(dqn), ptr(dkn), nH, rot,
                                                 traditional, eps, x_at if in_place else dq.ptr, io, width, None))
    mlxr.synchronize()
    x = dx.numpy()[offset:].reshape(qkv.shape)
    return (x if in_place else dq.numpy()), x


@pytest.mark.parametrize("nH,nKV,D,st,io,rot,traditional,norm,positions,in_place,scale", [
    (8, 2, 128, 0, 0, 128, 0, True, False, False, 1.0), (8, 2, 128, 0, 1, 128, 0, True, True, False, 1.0), (5, 1, 64, 1, 1, 64, 1, False, True, False, 1.25),
    (16, 16, 128, 1, 0, 64, 1, True, True, False, 1.28), (4, 4, 64, 0, 0, 32, 0, True, True, True, 1.0), (3, 1, 128, 0, 1, 0, 0, False, False, False, 1.0),
    (40, 8, 128, 1, 1, 128, 1, True, True, False, 0.5), (6, 2, 64, 0, 1, 6, 0, True, True, False, 1.5), (6, 2, 128, 1, 0, 6, 1, False, True, False, 1.5),
    (2, 1, 128, 0, 0, 2, 0, True, False, True, 1.0), (7, 7, 64, 0, 0, 64, 0, False, True, False, 1.0), (32, 8, 128, 0, 0, 96, 0, True, True, True, 1.1)])
@pytest.mark.parametrize("shift", [0, 1])   # 1: rows that start off their 16 bytes
def test_append(gpu, nH, nKV, D, st, io, rot, traditional, norm, positions, in_place, scale, shift):
    print(f"[case] {nH} {nKV} {D} {st} {io} {rot} {traditional} {norm} {positions} {in_place} {shift}", flush=True)
    rs = np.random.default_rng(nH)
    lens = [1, 64, 65, 200, 0, 130]
    c = Cache(gpu, lens, nKV, D, st, seed=nH, weight=True, position=True).up()
    # rows of all sequences mixed, with rows that name none, a sequence too many and a slot too many
    pairs = [(b, j) for b, n in enumerate(lens) for j in range(n) if j >= n - 70]
    pairs = [pairs[i] for i in rs.permutation(len(pairs))]
    pairs[3:3] = [(-1, -1), (len(lens), 0), (3, c.max_len), (2, -1), (-2 ** 31, 2 ** 31 - 1)]
    seq, slot = (np.array(x) for x in zip(*pairs))
    on = (seq >= 0) & (seq < len(lens)) & (slot >= 0) & (slot < c.max_len)
    R = len(seq)
    qkv = rs.standard_normal((R, (nH + 2 * nKV) * D + (1 if shift else 4))).astype(np.float32)
    inv = (1e6 ** (-np.arange(0, rot, 2) / max(1, rot))).astype(np.float32)
    qn, kn = ((1 + 0.1 * rs.standard_normal((2, D))).astype(np.float32) if norm else (None, None))
    pos = rs.integers(0, 131072, R).astype(np.int32) if positions else None
    before = {x: getattr(c, x).numpy() for x in ("dk", "dv", "dw", "dp")}
    q, x_after = run_append(gpu, c, qkv, seq, slot, nH, inv, qn, kn, rot, traditional, pos, 1e-6, scale, io, in_place, 3 if shift else 8, offset=shift)
    x = qkv[:, :(nH + 2 * nKV) * D].astype(np.float64).reshape(R, -1, D)
    h = x[:, :nH + nKV].copy()
    if norm:
        h /= np.sqrt((h ** 2).mean(-1, keepdims=True) + 1e-6)
        h[:, :nH] *= qn
        h[:, nH:] *= kn
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if traditional else (np.arange(rot // 2), np.arange(rot // 2, rot))
    at = slot if pos is None else pos
    z = (h[..., i] + 1j * h[..., j]) * (float(np.float32(scale)) * np.exp(1j * at[:, None] * inv.astype(np.float64)))[:, None]
    size = np.abs(h)                                      # of the pair a value comes from
    size[..., i] = size[..., j] = np.abs(z) + scale * (np.abs(h[..., i]) + np.abs(h[..., j]))
    h[..., i], h[..., j] = z.real, z.imag
    # norm: a mean of D squares (half its relative error: 2 sqrt(D) u), root, quotient, two products; rotation: sine and
    # cosine to 4 u of one and their scaling, two products and a sum
    tol = size * ((2 * np.sqrt(D) + 6) * U * norm + 10 * U)
    n, step = nH * D, half_step(st)
    tiny = 2.0 ** -25 * st
    got = (from_half(q, st) if io else q)[:, :n].reshape(R, nH, D)
    q_tol = tol[:, :nH] * (1 + step * io) + io * (step * np.abs(h[:, :nH]) + tiny)
    assert within(np.abs(got - h[:, :nH])[on], q_tol[on]) <= 1
    if in_place:
        assert same(q[:, n:], qkv[:, n:]) and same(q[~on], qkv[~on])
    else:
        assert same(q[:, n:], np.full_like(q[:, n:], 7)) and same(q[~on], np.full_like(q[~on], 7)) and same(x_after, qkv)
    k, v, w, p = before["dk"], before["dv"], before["dw"], before["dp"]
    new_k = c.dk.numpy()
    for r in np.nonzero(on)[0]:
        page = c.table[seq[r], slot[r] // PAGE]
        if not 0 <= page < k.shape[0]:
            continue
        row = slot[r] % PAGE
        assert within(np.abs(from_half(new_k[page, :, row], st) - h[r, nH:]), tol[r, nH:] * (1 + step) + step * np.abs(h[r, nH:]) + tiny) <= 1
        k[page, :, row] = new_k[page, :, row]
        v[page, :, row] = to_half(x[r, nH + nKV:].astype(np.float32), st)
        w[seq[r], :, slot[r]], p[seq[r], :, slot[r]] = 0, at[r]
    assert same(new_k, k) and same(c.dv.numpy(), v) and same(c.dw.numpy(), w) and same(c.dp.numpy(), p)


def test_append_bad_pages(gpu):
    """A page outside the pool takes nothing, weights and positions neither; the query still comes."""
    c = Cache(gpu, [65, 64], 2, 128, 0, seed=9, weight=True, position=True)
    c.table[0, 1], c.table[1, 0] = c.k.shape[0], -7
    c.up()
    qkv = np.random.default_rng(1).standard_normal((2, 6 * 128)).astype(np.float32)
    q, _ = run_append(gpu, c, qkv, np.array([0, 1]), np.array([64, 5]), 2, np.zeros(0, np.float32), None, None, 0, 0, None, 1e-6, 1.0, 0, False, 0)
    assert same(q[:, :256], qkv[:, :256])
    for x, y in ((c.dk, c.k), (c.dv, c.v), (c.dw, c.weight), (c.dp, c.position)):
        assert same(x.numpy(), y)


# ------------------------------------------------------------------------------------------- pages from lengths
def reserve_reference(table, lens, want, free, n_free, rows, n_pages, max_len):
    """Page by page."""
    table, free, B = table.copy(), free.copy(), len(lens)
    lens, want, nf = (np.clip(np.asarray(x, np.int64), 0, m) for x, m in ((lens, max_len), (want, max_len), (n_free, n_pages)))
    nf = int(nf)
    pages = lambda x: -(-int(x) // PAGE)  # noqa: E731
    for b in range(B):
        for e in range(pages(want[b]), pages(lens[b])):
            if 0 <= table[b, e] < n_pages and nf < n_pages:
                free[nf] = table[b, e]
                nf += 1
    start, count, len_out, seq, slot = np.zeros(B, np.int64), np.zeros(B, np.int64), np.minimum(lens, want), np.full(rows, -1), np.full(rows, -1)
    row, asked, there = 0, 0, nf
    for b in range(B):
        start[b] = min(row, 2 ** 31 - 1)
        more = int(want[b] - lens[b])
        if more <= 0:
            continue
        entries = range(pages(lens[b]), pages(want[b]))
        asked += len(entries)
        if row + more <= rows and (not entries or asked <= there):
            for e in entries:
                nf -= 1
                table[b, e] = free[nf]
            len_out[b], count[b] = want[b], more
            seq[row:row + more], slot[row:row + more] = b, np.arange(lens[b], want[b])
        row += more
    return [np.asarray(x, np.int32) for x in (table, free, len_out, [nf], start, count, seq, slot)]


class Pool:
    """The device's side of a reservation. nothing of the pool itself is touched: its pointers are the table's."""

    def __init__(self, mlxr, table, lens, free, n_free, max_len, n_pages, rows):
        d = lambda x: mlxr.DeviceArray.from_numpy(np.asarray(x, np.int32))  # noqa: E731
        self.mlxr, self.rows = mlxr, rows
        self.table, self.len, self.free, self.n_free = d(table), d(lens), d(free), d([n_free])
        self.len_out, self.n_free_out = d(np.full(len(lens), 77)), d([77])
        self.start, self.count, self.seq, self.slot = (d(np.full(n, 77)) for n in (len(lens), len(lens), rows + 2, rows + 2))
        self.kv = mlxr.PagedKV(k=self.table.ptr // 16 * 16, v=self.table.ptr // 16 * 16, table=self.table.ptr, len=self.len.ptr, n_pages=n_pages,
                               table_stride=table.shape[1], slot_stride=0, max_len=max_len, B=len(lens), nKV=1, D=64, st=0)
        self.work = workspace(mlxr, mlxr.lib.mlxr_k_paged_reserve_work(ctypes.byref(self.kv), rows))

    def run(self, want, in_place=False, stream=None):
        dw = self.want = self.mlxr.DeviceArray.from_numpy(np.asarray(want, np.int32))
        self.out = [self.table, self.free, self.len if in_place else self.len_out, self.n_free if in_place else self.n_free_out, self.start, self.count,
                    self.seq, self.slot]
        self.mlxr.check(self.mlxr.lib.mlxr_k_paged_reserve(ctypes.byref(self.kv), dw.ptr, self.free.ptr, self.n_free.ptr, self.rows, self.out[2].ptr, self.out[3].ptr,
                                                           self.start.ptr, self.count.ptr, self.seq.ptr, self.slot.ptr, self.work.ptr, self.work.nbytes, stream))

    def check(self, expected):
        self.mlxr.synchronize()
        names = ("table", "free", "len_out", "n_free_out", "start", "count", "seq", "slot")
        for name, got, want in zip(names, self.out, expected):
            got = got.numpy()
            if name in ("seq", "slot"):
                assert (got[self.rows:] == 77).all(), name
                got = got[:self.rows]
            assert same(got, want.reshape(got.shape)), (name, np.argwhere(got != want.reshape(got.shape))[:5])


def random_pool(rs, B, top, max_len, spare):
    lens = rs.integers(0, top + 1, B)
    used = -(-lens // PAGE)
    n_pages, width = int(used.sum()) + spare, -(-max_len // PAGE) + 1
    order = rs.permutation(n_pages)
    table = np.full((B, width), -1, np.int64)
    at = 0
    for b in range(B):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    free = np.full(n_pages, -5, np.int64)
    free[:spare] = order[at:]
    return lens, table, free, n_pages


@pytest.mark.parametrize("B,top,grow,spare,rows", [(1, 0, 1, 1, 1), (1, 64, 1, 1, 1), (3, 200, 300, 20, 900), (32, 500, 1, 40, 32), (64, 300, 90, 5, 9000),
                                                   (200, 400, 200, 100, 25000), (1025, 130, 3, 700, 4000), (4095, 64, 2, 300, 4097), (4096, 100, 2, 9000, 3000), (5000, 90, 5, 2500, 20000),
                                                   (7, 20000, 30000, 3000, 200000), (9, 300, 0, 4, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve(gpu, B, top, grow, spare, rows, in_place):
    rs = np.random.default_rng(B)
    max_len = top + grow + 1
    lens, table, free, n_pages = random_pool(rs, B, top, max_len, spare)
    want = np.where(rs.random(B) < 0.3, rs.integers(0, np.maximum(lens, 1) + 1), lens + rs.integers(0, grow + 1, B))
    want[rs.random(B) < 0.1] = 0
    expected = reserve_reference(table, lens, want, free, spare, rows, n_pages, max_len)
    p = Pool(gpu, table, lens, free, spare, max_len, n_pages, rows)
    p.run(want, in_place)
    p.check(expected)
    if not in_place:                                       # separate outputs: the call repeats itself
        p.run(want)
        p.check(expected)


def test_reserve_bounds_on_the_device(gpu):
    """Lengths and wanted lengths outside [0, max_len], table entries outside the pool, stack heights outside [0, n_pages], rows that
    are too few, sums past 32 bits."""
    rs = np.random.default_rng(3)
    lens, table, free, n_pages = random_pool(rs, 40, 500, 600, 30)
    lens[[3, 4, 5]] = [-7, 10 ** 6, 2 ** 31 - 1]
    table[6, :4], table[4, :10] = [n_pages, -1, 2 ** 31 - 1, -2 ** 31], rs.integers(0, n_pages, 10)
    want = np.where(rs.random(40) < 0.5, 0, lens + 40)
    want[[1, 4, 6, 9]] = [-3, 5, 0, 2 ** 31 - 1]
    want = np.clip(want, -2 ** 31, 2 ** 31 - 1)
    for n_free in (30, 0, -4, n_pages + 9, n_pages):
        for rows in (1, 100, 5000):
            p = Pool(gpu, table, lens, free, n_free, 600, n_pages, rows)
            p.run(want)
            p.check(reserve_reference(table, lens, want, free, n_free, rows, n_pages, 600))
    # 300 sequences that ask for 2^24 slots each: 2^32 rows
    B = 300
    table, free = np.full((B, 1 << 18), -1, np.int32), np.arange(50)
    p = Pool(gpu, table, np.zeros(B, np.int64), free, 50, 1 << 24, 50, 5000)
    want = np.full(B, 1 << 24)
    want[:2] = [70, 0]
    p.run(want)
    p.check(reserve_reference(table, np.zeros(B, np.int64), want, free, 50, 5000, 50, 1 << 24))


def test_reserve_keeps_pages_apart(gpu):
    """Sixty steps of a server, in place: sequences grow, end, are cut and refused; no page is lost or had twice."""
    rs = np.random.default_rng(7)
    B, max_len, n_pages, rows = 50, 1000, 260, 1500
    table, free, lens, nf = np.full((B, 16), -1, np.int32), rs.permutation(n_pages).astype(np.int32), np.zeros(B, np.int32), n_pages
    p = Pool(gpu, table, lens, free, n_pages, max_len, n_pages, rows)
    refused = 0
    for step in range(60):
        want = lens + np.where(rs.random(B) < 0.1, rs.integers(1, 400, B), 1)
        want[rs.random(B) < 0.08] = 0
        cut = rs.random(B) < 0.05
        want[cut] = lens[cut] // 2
        want = np.minimum(want, max_len)
        expected = reserve_reference(table, lens, want, free, nf, rows, n_pages, max_len)
        p.run(want, in_place=True)
        p.check(expected)
        refused += int(((want > lens) & (expected[5] == 0)).sum())
        table, free, lens, nf = expected[0], expected[1], expected[2], int(expected[3][0])
        held = np.concatenate([table[b, :-(-lens[b] // PAGE)] for b in range(B)] + [free[:nf]])
        assert len(held) == n_pages and len(np.unique(held)) == n_pages
    assert refused > 20


# ------------------------------------------------------------------------------------------- together
class Server:
    """Sequences over one pool: a reservation, the append of its rows and their attention, from host token rows."""

    def __init__(self, gpu, B=5, nKV=2, nH=8, st=0, io=0, seed=1, max_len=512, n_pages=24, rows=300):
        d = gpu.DeviceArray
        self.gpu, self.B, self.nKV, self.nH, self.D, self.st, self.io, self.max_len, self.rows, self.n_pages = gpu, B, nKV, nH, 128, st, io, max_len, rows, n_pages
        self.rs = np.random.default_rng(seed)
        self.k, self.v = (d.from_numpy(np.full((n_pages, nKV, PAGE, 128), one_half(NAN, st), np.uint16)) for _ in range(2))
        self.table = d.from_numpy(np.full((B, max_len // PAGE), -1, np.int32))
        self.free, self.n_free = d.from_numpy(self.rs.permutation(n_pages).astype(np.int32)), d.from_numpy(np.array([n_pages], np.int32))
        self.len, self.want, self.start, self.count = (d.zeros(B, np.int32) for _ in range(4))
        self.seq, self.slot = (d.zeros(rows, np.int32) for _ in range(2))
        self.width = (nH + 2 * nKV) * 128
        self.qkv = d.zeros((rows, self.width), np.float32)
        self.inv_freq = (1e6 ** (-np.arange(0, 128, 2) / 128)).astype(np.float32)
        self.inv = d.from_numpy(self.inv_freq)
        t = np.uint16 if io else np.float32
        self.q, self.out = d.zeros((rows, nH * 128), t), d.zeros((rows, nH * 128), t)
        self.kv = gpu.PagedKV(k=self.k.ptr, v=self.v.ptr, table=self.table.ptr, len=self.len.ptr, n_pages=n_pages, table_stride=max_len // PAGE, slot_stride=0,
                              max_len=max_len, B=B, nKV=nKV, D=128, st=st)
        ref = ctypes.byref(self.kv)
        self.wr = workspace(gpu, gpu.lib.mlxr_k_paged_reserve_work(ref, rows))
        self.wa = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ref, nH, rows, io))

    def inputs(self, want, qkv):
        self.want.upload(np.asarray(want, np.int32))
        full = np.zeros((self.rows, self.width), np.float32)
        full[:len(qkv)] = qkv
        self.qkv.upload(full)

    def run(self, s=None):
        gpu, lib, ref, n = self.gpu, self.gpu.lib, ctypes.byref(self.kv), self.nH * 128
        gpu.check(lib.mlxr_k_paged_reserve(ref, self.want.ptr, self.free.ptr, self.n_free.ptr, self.rows, self.len.ptr, self.n_free.ptr, self.start.ptr, self.count.ptr,
                                           self.seq.ptr, self.slot.ptr, self.wr.ptr, self.wr.nbytes, s))
        gpu.check(lib.mlxr_k_paged_append_rows(ref, self.qkv.ptr, self.width, self.rows, self.seq.ptr, self.slot.ptr, None, self.inv.ptr, 1.0, None, None, self.nH, 128, 0, 1e-6,
                                               self.q.ptr, self.io, n, s))
        gpu.check(lib.mlxr_k_paged_attention_rows(ref, self.start.ptr, self.count.ptr, self.rows, self.q.ptr, self.io, n, self.nH, 0, 128 ** -0.5, self.out.ptr, n,
                                                  self.wa.ptr, self.wa.nbytes, s))

    def state(self):
        return [x.numpy() for x in (self.k, self.v, self.table, self.free, self.n_free, self.len, self.start, self.count, self.seq, self.slot, self.q, self.out)]


def steps(rs, B, width, n):
    """What arrives: wanted changes of length and token rows. Prompts, chunks, single tokens, an ended and a cut sequence."""
    plan = [[40, 1, 100, 0, 3], [1, 70, 1, 64, 1], [1, 1, 1, 1, 1], [-30, 1, None, 1, 1], [5, 1, 130, 1, 0], [1, 1, 1, 1, 1]]
    for i in range(n):
        yield plan[i % len(plan)], [rs.standard_normal((max(0, x or 0), width)).astype(np.float32) for x in plan[i % len(plan)]]


@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 1)])
def test_steps_together(gpu, st, io):
    """Pages, append and attention of six steps, against attention over every sequence's own tokens kept on the host."""
    s = Server(gpu, st=st, io=io)
    tokens = [np.zeros((0, s.width), np.float32) for _ in range(s.B)]
    G, n = s.nH // s.nKV, s.nH * 128
    for change, new in steps(np.random.default_rng(17), s.B, s.width, 6):
        for b, x in enumerate(change):
            tokens[b] = tokens[b][:0] if x is None else tokens[b][:x] if x < 0 else np.concatenate([tokens[b], new[b]])
        s.inputs([len(t) for t in tokens], np.concatenate(new))
        s.run()
        gpu.synchronize()
        assert same(s.len.numpy(), np.array([len(t) for t in tokens], np.int32))
        got = from_half(s.out.numpy(), st) if io else s.out.numpy()
        row = 0
        for b, t in enumerate(tokens):
            m, L = len(new[b]), len(t)
            if m == 0:
                continue
            x = t.astype(np.float64).reshape(L, -1, 128)
            z = (x[..., :64] + 1j * x[..., 64:]) * np.exp(1j * np.arange(L)[:, None] * s.inv_freq.astype(np.float64))[:, None]
            rot = np.concatenate([z.real, z.imag], -1)
            half = lambda y: from_half(to_half(y.astype(np.float32), st), st).astype(np.float64)  # noqa: E731
            for h in range(s.nH):
                k, v = half(rot[:, s.nH + h // G]), half(x[:, s.nH + s.nKV + h // G])
                q = rot[L - m:, h]
                e = (half(q) if io else q) @ k.T * 128 ** -0.5
                e[np.arange(L) > np.arange(L - m, L)[:, None]] = -np.inf
                p = np.exp(e - e.max(1, keepdims=True))
                want = p / p.sum(1, keepdims=True) @ v
                # a rotated value may lie so near the middle of two numbers of the type that it is rounded the other way: few of
                # a score's 128 terms, so some hundredths of a p (bf16); beyond that the types' roundings, on values of about one
                err = np.abs(got[row:row + m, h * 128:h * 128 + 128] - want)
                assert err.max() < (0.05 if io and st == 0 else 0.02) and err.mean() < (2.0 ** -9 if io and st == 0 else 2.0 ** -12), (b, h)
            row += m


def test_steps_captured(gpu):
    """The three calls in a HIP graph: replays with new lengths and tokens, eager work and synchronizations between them, give the
    eager calls' bits."""
    hip = Hip(gpu)
    a, b, st = Server(gpu), Server(gpu), hip.stream()
    graph = None
    for i, (change, new) in enumerate(steps(np.random.default_rng(18), a.B, a.width, 12)):
        lens = a.len.numpy()
        want = [0 if x is None else lens[j] + x for j, x in enumerate(change)]
        for s in (a, b):
            s.inputs(want, np.concatenate(new))
        a.run(st)
        hip.wait(st)
        if i == 0:
            b.run(st)
            hip.wait(st)
            graph = hip.capture(st, lambda: b.run(st))
        else:
            hip("hipGraphLaunch", graph, st)
            hip.wait(st)
        for x, y in zip(a.state(), b.state()):
            assert same(x, y), i
    hip("hipGraphExecDestroy", graph)
    hip("hipStreamDestroy", st)


def test_steps_captured_in_the_strictest_mode(gpu):
    """Nothing that the calls ask of the runtime is forbidden in a capture of mode 'global', and the first run of buffers may be a replay."""
    hip = Hip(gpu)
    a, b, st, graph, ex = Server(gpu), Server(gpu), hip.stream(), ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", st, 0)
    b.run(st)
    hip("hipStreamEndCapture", st, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
    for i, (change, new) in enumerate(steps(np.random.default_rng(20), a.B, a.width, 4)):
        lens = a.len.numpy()
        for s in (a, b):
            s.inputs([0 if x is None else lens[j] + x for j, x in enumerate(change)], np.concatenate(new))
        a.run(st)
        hip("hipGraphLaunch", ex, st)
        hip.wait(st)
        for x, y in zip(a.state(), b.state()):
            assert same(x, y), i
    hip("hipGraphExecDestroy", ex)
    hip("hipStreamDestroy", st)


def test_host_memory_is_refused(gpu):
    """Every pointer that a kernel would follow, at memory that the device does not have: an error, and nothing written."""
    s, host = Server(gpu), np.zeros(1 << 16, np.uint8)
    at = -(-host.ctypes.data // 256) * 256
    names = {"mlxr_k_paged_reserve": (1, 2, 3, 5, 6, 7, 8, 9, 10, 11), "mlxr_k_paged_append_rows": (1, 4, 5, 7, 15), "mlxr_k_paged_attention_rows": (1, 2, 4, 10, 12)}
    real = {n: getattr(gpu.lib, n) for n in names}

    class Lib:   # the server's calls, with argument `bad` of `name` replaced
        name = bad = None

        def __getattr__(self, n):
            if n not in real:
                return getattr(gpu.lib, n)
            return lambda *x: real[n](*(at if n == self.name and i == self.bad else y for i, y in enumerate(x)))

    class Gpu:
        lib, check = Lib(), staticmethod(lambda rc: seen.append(rc))
    s.inputs([3, 1, 0, 2, 70], np.ones((76, s.width), np.float32))
    s.gpu = Gpu
    for Lib.name, places in names.items():
        for Lib.bad in places:
            seen = []
            print(f"[case] {Lib.name} {Lib.bad}", flush=True)
            s.run()
            assert seen == [INVALID if n == Lib.name else 0 for n in names], (Lib.name, Lib.bad)
    gpu.synchronize()
    assert not host.any()


def test_one_workspace_for_all_sizes(gpu):
    """Calls of other batches, types and sizes take turns on a workspace of the largest one's size."""
    big, small = Cache(gpu, [3000, 700], 2, 128, 0, seed=31).up(), Cache(gpu, [90], 1, 64, 0, seed=32).up()
    runs = [Rows(big, [300, 1], 8, 1, seed=31), Rows(small, [3], 3, 0, seed=32), Rows(big, [5, 2], 8, 0, seed=33), Rows(small, [80], 1, 1, seed=34)]
    alone = [attend(gpu, r) for r in runs]
    work = workspace(gpu, max(gpu.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(r.c.desc()), r.nH, r.rows, r.io) for r in runs))
    for r, want in list(zip(runs, alone)) * 2:
        assert same(attend(gpu, r, work=work), want)


def test_two_streams_at_once(gpu):
    """Two servers on two streams, each with its own workspaces, give what they give alone."""
    hip = Hip(gpu)
    plan = list(steps(np.random.default_rng(19), 5, 12 * 128, 4))

    def go(s, st):
        lens = np.zeros(5, int)
        for change, new in plan:
            lens = np.array([0 if x is None else lens[j] + x for j, x in enumerate(change)])
            s.inputs(lens, np.concatenate(new))
            yield s.run(st)
    alone = []
    for io in (0, 1):
        s = Server(gpu, io=io)
        for _ in go(s, None):
            gpu.synchronize()
        alone.append(s.state())
    both, streams = [Server(gpu, io=io) for io in (0, 1)], [hip.stream(), hip.stream()]
    for _ in zip(*(go(s, st) for s, st in zip(both, streams))):
        for st in streams:
            hip.wait(st)
    for s, want in zip(both, alone):
        for x, y in zip(s.state(), want):
            assert same(x, y)
    for st in streams:
        hip("hipStreamDestroy", st)


def test_offsets_past_32_bits(gpu):
    """The same rows with their pages behind 2^32 elements of the pools: the same bits from append and attention."""
    from test_batch_gpu import far_pool, fetch
    nKV, D, nH = 8, 128, 16
    page_bytes = nKV * PAGE * D * 2
    c = Cache(gpu, [200, 64, 300], nKV, D, 0, seed=95).up()
    r = Rows(c, [100, 64, 1], nH, 1, seed=95)
    pools, pages, shift = far_pool(gpu, c, page_bytes)
    table = gpu.DeviceArray.from_numpy(np.where(c.table < 0, -1, c.table + shift).astype(np.int32))
    far = c.desc(k=pools[0].ptr, v=pools[1].ptr, n_pages=pages, table=table.ptr)
    assert same(attend(gpu, r), attend(gpu, r, desc=far))
    rs = np.random.default_rng(96)
    seq, slot = np.repeat([0, 2], 40), np.concatenate([np.arange(100, 140), np.arange(260, 300)])
    qkv, inv = rs.standard_normal((80, (nH + 2 * nKV) * D)).astype(np.float32), (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    near, _ = run_append(gpu, c, qkv, seq, slot, nH, inv, None, None, D, 0, None, 1e-6, 1.0, 0, False, 0)
    d = gpu.DeviceArray.from_numpy
    dx, di, ds, dt, dq = d(qkv), d(inv), d(seq.astype(np.int32)), d(slot.astype(np.int32)), gpu.DeviceArray.zeros((80, nH * D), np.float32)
    gpu.check(gpu.lib.mlxr_k_paged_append_rows(ctypes.byref(far), dx.ptr, qkv.shape[1], 80, ds.ptr, dt.ptr, None, di.ptr, 1.0, None, None, nH, D, 0, 1e-6, dq.ptr, 0, nH * D, None))
    gpu.synchronize()
    assert same(dq.numpy(), near)
    assert same(fetch(gpu, pools[0], shift * page_bytes, c.k), c.dk.numpy()) and same(fetch(gpu, pools[1], shift * page_bytes, c.v), c.dv.numpy())
