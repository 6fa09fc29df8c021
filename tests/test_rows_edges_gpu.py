"""Attention of rows where the tests of its sizes do not look.

Tolerances as in test_rows_gpu, with u = 2^-24; terms that are all alike are rounded alike, so their common error counts in full."""
import ctypes
import time

import numpy as np
import pytest

from test_batch_gpu import PAGE, U, Cache, from_half, same, to_half, within, workspace
from test_rows_gpu import INF, Rows, attend, check, half_step, one_half, reference

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- long tails
def tail_attention(gpu, n, nKV, G, D, st, io, sink, rows=64):
    """One key of a large score at slot `sink`, and about n of score 0. Rows and heads differ in what the n weigh together against
    the one: from a 64th to four times as much. Values: 0 and -1 in turn for the one, 1 and 0 for the others. All pages but the
    one key's are the same one, so a long sequence needs no memory; 256 KV heads, so a run is long too."""
    d, nH, length, rs = gpu.DeviceArray.from_numpy, nKV * G, n + rows, np.random.default_rng(n)
    kv = np.zeros((2, 2, nKV, PAGE, D), np.float32)
    kv[1, ..., ::2] = 1.0
    kv[0, 0, :, sink % PAGE, 0] = 8.0
    kv[1, 0, :, sink % PAGE, ::2], kv[1, 0, :, sink % PAGE, 1::2] = 0.0, -1.0
    k, v = (d(to_half(x, st).reshape(x.shape)) for x in kv)
    table = np.full((1, -(-length // PAGE)), 1, np.int32)
    table[0, sink // PAGE] = 0
    q = np.zeros((rows, nH, D), np.float32)
    q[..., 0] = np.log(n / 2.0 ** rs.uniform(-6, 2, (rows, nH)))      # times 8 and a scale of 1/8: the large score
    bits = to_half(q, st).reshape(q.shape) if io else q
    score = (from_half(bits, st) if io else q)[..., :1].astype(np.float64)
    w, others = np.exp(score), (n + np.arange(rows))[:, None, None].astype(np.float64)
    want = np.where(np.arange(D) % 2 == 0, others / (w + others), -w / (w + others))
    dt, dl, ds, dc, dq, out = d(table), d(np.array([length], np.int32)), d(np.zeros(1, np.int32)), d(np.array([rows], np.int32)), d(bits), d(np.zeros_like(bits))
    desc = gpu.PagedKV(k=k.ptr, v=v.ptr, table=dt.ptr, len=dl.ptr, weight=None, position=None, n_pages=2, table_stride=table.shape[1], slot_stride=0,
                       max_len=length, B=1, nKV=nKV, D=D, st=st)
    ref = ctypes.byref(desc)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ref, nH, rows, io))
    gpu.check(gpu.lib.mlxr_k_paged_attention_rows(ref, ds.ptr, dc.ptr, rows, dq.ptr, io, nH * D, nH, 0, 0.125, out.ptr, nH * D, work.ptr, work.nbytes, None))
    gpu.synchronize()
    return (from_half(out.numpy(), st) if io else out.numpy()), want, score


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_sum_of_equal_keys(gpu, D, place):
    """Keys that are each far less than the last bits of the sum that holds a large one still add up."""
    n = 131072
    got, want, score = tail_attention(gpu, n, 256, 1, D, 0, 0, {"first": 5, "middle": n // 2, "last": n - 70}[place])
    # a wave has every other page. The sum rounds once a page (u of itself, all alike), the values twelve times: four steps of 16
    # keys in three parts. A score: the query's parts, scaling, the exponential's argument (2^-24 and 6 u); a dozen roundings besides
    pages = n / PAGE / 2 + 1
    times = np.where(np.arange(D) % 2 == 0, 13, 1)
    tol = np.abs(want) * (times * pages * U + score * 7 * U + 14 * U)
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("n,G,D,io", [(32768, 4, 128, 0), (131072, 4, 64, 0), (131072, 1, 128, 0), (131072, 4, 128, 1), (3000000, 1, 64, 1)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_long_tail_in_f16(gpu, n, G, D, io, place):
    """The numbers of f16 end 2^-24 below one, and a long tail's p end further below the largest: they keep their bits."""
    print(f"[case] {n} {G} {D} {io} {place}", flush=True)
    got, want, score = tail_attention(gpu, n, 256, G, D, 1, io, {"first": 5, "middle": n // 2, "last": n - 70}[place])
    # a score: the query's parts (2^-22), scaling, the exponential's argument (6 u); a p: its rounding, all alike. A tail's p is a power of two
    # of its own page's largest, so that their sums, page by page, are exact: the large one is less than 2^28 of them. 63 of them beside the
    # large one end 2^-34 of it away, half of that off at most: 2^-29 together, 2^-23 of a tail that weighs a 64th. A dozen roundings of sums and results
    e = half_step(1) if io else 2.0 ** -22
    tol = np.abs(want) * (score * ((0 if io else e) + 6 * U) + 2 * e + 12 * U + half_step(1) * io) + 2.0 ** -25 * io
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("G,D,io", [(4, 128, 0), (1, 64, 0), (4, 64, 1), (1, 128, 1)])
def test_pages_of_two_scores_in_f16(gpu, G, D, io):
    """Pages whose scores are 6 to 29 powers of two apart, in turn: either kind keeps its bits, however often the larger comes back."""
    d, n, rows, nKV, rs = gpu.DeviceArray.from_numpy, 32768, 64, 256, np.random.default_rng(D)
    nH, length = nKV * G, n + 64
    kv = np.zeros((2, 2, nKV, PAGE, D), np.float32)
    kv[0, 1, ..., 0] = 8.0
    kv[1, 0, ..., ::2], kv[1, 1, ..., 1::2] = 1.0, -1.0
    k, v = (d(to_half(x, 1).reshape(x.shape)) for x in kv)
    table = (np.arange(length // PAGE) % 2).astype(np.int32)[None]
    q = np.zeros((rows, nH, D), np.float32)
    q[..., 0] = rs.uniform(4.3, 20.0, (rows, nH))
    bits = to_half(q, 1).reshape(q.shape) if io else q
    score = (from_half(bits, 1) if io else q)[..., :1].astype(np.float64)
    large = np.cumsum(np.arange(length) // PAGE % 2)[n:][:, None, None] * np.exp(score)
    small = np.cumsum(1 - np.arange(length) // PAGE % 2)[n:][:, None, None]
    want = np.where(np.arange(D) % 2 == 0, small, -large) / (large + small)
    dt, dl, ds, dc, dq, out = d(table), d(np.array([length], np.int32)), d(np.zeros(1, np.int32)), d(np.array([rows], np.int32)), d(bits), d(np.zeros_like(bits))
    desc = gpu.PagedKV(k=k.ptr, v=v.ptr, table=dt.ptr, len=dl.ptr, weight=None, position=None, n_pages=2, table_stride=table.shape[1], slot_stride=0,
                       max_len=length, B=1, nKV=nKV, D=D, st=1)
    ref = ctypes.byref(desc)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ref, nH, rows, io))
    gpu.check(gpu.lib.mlxr_k_paged_attention_rows(ref, ds.ptr, dc.ptr, rows, dq.ptr, io, nH * D, nH, 0, 0.125, out.ptr, nH * D, work.ptr, work.nbytes, None))
    gpu.synchronize()
    got = from_half(out.numpy(), 1) if io else out.numpy()
    # roundings all alike: one of the sum and eight of the values a page (four steps of 16 keys, two parts), two of each where the point
    # of reference moves by a power that is no whole number (queries in f16); those of a score and a p as above
    e, pages = half_step(1) if io else 2.0 ** -22, length / PAGE
    tol = np.abs(want) * (score * ((0 if io else e) + 6 * U) + 2 * e + (13 if io else 9) * pages * U + 12 * U + half_step(1) * io) + 2.0 ** -25 * io
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, worst


# ------------------------------------------------------------------------------------------- many sequences
def scattered(gpu, at, B=60000):
    """Chunks of eight sequences of a batch whose other ones are idle, and a function that runs the call."""
    lens, counts = np.zeros(B, int), np.zeros(B, int)
    lens[at], counts[at] = 700 + 37 * np.arange(8), 100
    c = Cache(gpu, lens, 1, 64, 0, seed=5).up()
    r = Rows(c, counts, 1, 1, seed=6, gap=0)
    d, kv = gpu.DeviceArray.from_numpy, c.desc()
    ds, dc, dq, do = d(r.start), d(r.count), d(r.bits), d(np.full(r.bits.shape, 7, r.bits.dtype))
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(kv), 1, r.rows, 1))

    def run():
        gpu.check(gpu.lib.mlxr_k_paged_attention_rows(ctypes.byref(kv), ds.ptr, dc.ptr, r.rows, dq.ptr, 1, r.width, 1, 0, 0.09, do.ptr, r.width, work.ptr, work.nbytes, None))
        gpu.synchronize()
        return do.numpy
    return c, r, run


def test_idle_sequences_between(gpu):
    """Thousands of idle sequences between those with rows: the same results, and they cost about what they cost behind them."""
    times = []
    for at in (np.arange(8), np.arange(8) * 7500 + 3000):
        c, r, run = scattered(gpu, at)
        check(run()(), r, *reference(r, 0, 0.09))
        best = np.inf
        for _ in range(20):
            t = time.perf_counter()
            run()
            best = min(best, time.perf_counter() - t)
        times.append(best)
    print(times)
    # the batch is looked over twice either way, 120 steps each; between two chunks lie 7500 more sequences, 30 steps. One by one they
    # would be 7500 steps
    assert times[1] < 3 * times[0], times


@pytest.mark.parametrize("B,nKV,G,D,st,io,window,idle", [(65, 2, 2, 128, 0, 0, 0, 0.1), (65, 1, 3, 64, 1, 1, 50, 0.5), (600, 1, 2, 128, 0, 0, 70, 0.9), (600, 2, 1, 64, 0, 1, 0, 0.2),
                                                         (1100, 1, 1, 128, 1, 0, 0, 0.95)])
def test_bounds_of_many_sequences(gpu, B, nKV, G, D, st, io, window, idle):
    """What only the device sees of a batch of more sequences than a wave looks over at once: lengths and counts of no use, counts
    above lengths, pages that are not there, rows in front of the array and behind it."""
    print(f"[case] {B} {nKV} {G} {D} {st} {io} {window} {idle}", flush=True)
    rs = np.random.default_rng(B + D)
    lens = rs.integers(0, 260, B)
    lens[-2:] = 259, 200
    c = Cache(gpu, lens, nKV, D, st, seed=B)
    bad = rs.permutation(np.arange(2, B - 2))[:12]
    c.lens[bad[:4]] = [-7, 5000, -2 ** 31, 2 ** 31 - 1]
    for b in bad[1], bad[3]:                                     # held at max_len: pages for that
        c.table[b, :-(-c.max_len // PAGE)] = c.table[B - 2, :-(-c.max_len // PAGE)]
    c.table[bad[4], 0], c.table[bad[5], :3] = c.k.shape[0], [-1, -2 ** 31, 2 ** 31 - 1]
    c.up()
    counts = np.where(rs.random(B) < idle, 0, np.minimum(rs.integers(1, 60, B), lens))
    counts[bad] = [5, 9, 4, 30, 20, 20, -4, -2 ** 31, lens[bad[8]] + 3, lens[bad[9]] + 70, 6, 8]
    r = Rows(c, counts, nKV * G, io, seed=B)
    r.set(np.where(np.isnan(r.q), np.float32(0.25), r.q))        # rows of no sequence have one here
    want = reference(r, window, 0.09)
    got = attend(gpu, r, window=window)
    check(got, r, *want)
    over = r.start[bad[9]] + np.arange(70)
    assert not got[over, :nKV * G * D].any()
    start = r.start.copy()
    start[bad[10]], start[bad[11]], start[bad[8]], start[bad[9]] = -5, r.rows - 1, r.rows + 1, 2 ** 31 - 2
    check(attend(gpu, r, window=window, start=start), r, *reference(r, window, 0.09, start=start.astype(np.int64)))


@pytest.mark.parametrize("B", [3, 64, 65, 700])
@pytest.mark.parametrize("D,st,io", [(128, 0, 0), (64, 1, 1)])
def test_no_sequence_has_a_slot(gpu, B, D, st, io):
    """Rows of sequences without any slot, and nothing else to do: zeros, and the workspace serves the next call."""
    c, full = Cache(gpu, [0] * B, 1, D, st, seed=1, max_len=64).up(), Cache(gpu, [40] * B, 1, D, st, seed=2).up()
    r, other = Rows(c, np.arange(B) % 4, 2, io, seed=3), Rows(full, np.arange(B) % 4, 2, io, seed=4)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(full.desc()), 2, max(r.rows, other.rows), io))
    check(attend(gpu, r, work=work), r, *reference(r, 0, 0.09))
    check(attend(gpu, other, work=work), other, *reference(other, 0, 0.09))


# ------------------------------------------------------------------------------------------- infinities
@pytest.mark.parametrize("st,io", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("odd", [INF, -INF])
@pytest.mark.parametrize("window", [0, 90])
def test_infinities_in_sight(gpu, st, io, D, odd, window):
    """Rows that attend an infinite key or value get what the formula gives, others what they get without: a key is left out where its
    score is -infinity, its infinite values too, and makes NaN where it is +infinity; an infinite value stays where it is attended."""
    lens, counts, G = [300, 128, 70], [150, 128, 1], 3
    c = Cache(gpu, lens, 1, D, st, seed=52)
    r = Rows(c, counts, G, io, seed=52)
    key, value = {0: 222, 1: 64, 2: 3}, {0: 180, 1: 30, 2: 60}
    q = r.q.copy()
    sign = np.zeros(r.rows)
    for b in range(3):
        mine = r.start[b] + np.arange(counts[b])
        sign[mine] = np.where(np.arange(counts[b]) % 3 == 1, 1, -1)    # a third of the rows have +infinity
        for g in range(G):
            q[mine, g * D + 5] = (np.abs(q[mine, g * D + 5]) + 0.25) * sign[mine] * np.sign(odd)
    r.set(q)

    class Gone:   # without the infinite keys, and with zeros for infinite values
        def __getattr__(self, name):
            return getattr(c, name)

        def rows(self, pool, b, h, m):
            x, there = c.rows(pool, b, h, m)
            gone = np.arange(m) == key[b]
            x = np.where(gone[:, None], 0, x)
            if pool is c.v:
                x[value[b], 7] = 0
            return x, there & ~gone
    spot = lambda b, j: (c.table[b, j // PAGE], 0, j % PAGE)  # noqa: E731
    for b in range(3):
        c.k[spot(b, key[b])][5], c.v[spot(b, key[b])][:], c.v[spot(b, value[b])][7] = (one_half(odd, st) for _ in range(3))
    c.up()
    got = attend(gpu, r, window=window)
    r.c = Gone()
    want, tol, named = reference(r, window, 0.09)
    r.c = c
    want, n = want.reshape(r.rows, G, D), G * D
    for b in range(3):
        rows, slot = r.start[b] + np.arange(counts[b]), lens[b] - counts[b] + np.arange(counts[b])
        sees = lambda j: (slot >= j) & ((slot - window < j) | (window == 0))  # noqa: E731
        want[rows[sees(value[b])], :, 7] = odd
        want[rows[sees(key[b]) & (sign[rows] > 0)]] = np.nan
    want = want.reshape(r.rows, n)
    x = (from_half(got, st) if io else got)[:, :n]
    finite, odd_ones = named[:, None] & np.isfinite(want), named[:, None] & ~np.isfinite(want)
    assert np.array_equal(x[odd_ones], want[odd_ones].astype(np.float32), equal_nan=True)
    assert within(np.abs(x[finite] - want[finite]), tol[finite]) <= 1
    assert same(got[~named], np.full_like(got[~named], 7))
