"""Attention of rows where the tests of its sizes do not look.

Tolerances as in test_rows_gpu, with u = 2^-24; terms that are all alike are rounded alike, so their common error counts in full."""
import ctypes
import time

import numpy as np
import pytest

from test_batch_gpu import PAGE, U, Cache, from_half, to_half, workspace
from test_rows_gpu import Rows, attend, check, half_step, reference

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
