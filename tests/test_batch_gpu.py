"""A batch's decode step (paged append, attention, eviction, sampling of rows) through the C ABI, against plain
64-bit numpy forms.

Tolerances. u = 2^-24, the half step of fp32. A sum of n fp32 terms is taken to be off by 4 sqrt(n) u times the
root of the sum of their squares (rounding errors are independent; 4 is four standard deviations and more), a
product, an exponential or a scaling by u to 2u of its value. bf16 rounds by 2^-8 of the value at most, f16 by 2^-11
(2^-25 below its normal numbers). Selections, copies and tokens are exact."""
import ctypes

import numpy as np
import pytest

from qfix import bf16_round, bf16_to_f32

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
PAGE = 64


def to_half(x, st):
    return bf16_round(x) if st == 0 else np.asarray(x, np.float32).astype(np.float16).view(np.uint16)


def from_half(x, st):
    return bf16_to_f32(x) if st == 0 else np.asarray(x).view(np.float16).astype(np.float32)


class Cache:
    """A pool of pages and the table of a batch: every page distinct, in random order, NaN in every row that holds
    no slot and in the pages that no table names; table entries behind a sequence's last page name no page."""

    def __init__(self, mlxr, lens, nKV, D, st, seed=0, extra_pages=2, max_len=None, weight=False, position=False, pad=3, room=None):
        rs = np.random.default_rng(seed)
        self.mlxr, self.rs = mlxr, rs
        self.lens = np.array(lens, np.int32)
        self.B, self.nKV, self.D, self.st = len(lens), nKV, D, st
        self.max_len = max_len or max(1, int(self.lens.max()))
        room = self.lens if room is None else np.array(room)
        used = -(-room // PAGE)
        self.width = max(1, -(-self.max_len // PAGE)) + 1
        n = int(used.sum()) + extra_pages
        order = rs.permutation(n)
        self.table = np.full((self.B, self.width), -1, np.int32)
        at = 0
        for b in range(self.B):
            self.table[b, :used[b]] = order[at:at + used[b]]
            at += used[b]
        self.free = order[at:]
        shape = (n, nKV, PAGE, D)
        nan = np.float32(np.nan)
        self.k, self.v = (np.full(shape, to_half(nan, st), np.uint16) for _ in range(2))
        for b in range(self.B):
            for i in range(int(used[b])):
                rows = min(PAGE, int(self.lens[b]) - i * PAGE)
                if rows > 0:
                    for pool in (self.k, self.v):
                        pool[self.table[b, i], :, :rows] = to_half(rs.standard_normal((nKV, rows, D)), st)
        self.stride = self.max_len + pad
        self.weight = rs.exponential(1.0, (self.B, nKV, self.stride)).astype(np.float32) if weight else None
        self.position = rs.integers(0, 1 << 30, (self.B, nKV, self.stride)).astype(np.int32) if position else None

    def up(self):
        d = self.mlxr.DeviceArray.from_numpy
        self.dk, self.dv, self.dtable, self.dlen = d(self.k), d(self.v), d(self.table), d(self.lens)
        self.dw = d(self.weight) if self.weight is not None else None
        self.dp = d(self.position) if self.position is not None else None
        return self

    def desc(self, **over):
        a = dict(k=self.dk.ptr, v=self.dv.ptr, table=self.dtable.ptr, len=self.dlen.ptr, weight=self.dw and self.dw.ptr,
                 position=self.dp and self.dp.ptr, n_pages=self.k.shape[0], table_stride=self.width, slot_stride=self.stride,
                 max_len=self.max_len, B=self.B, nKV=self.nKV, D=self.D, st=self.st)
        a.update(over)
        return self.mlxr.PagedKV(**a)

    def rows(self, pool, b, h, n):
        """Slots 0 .. n - 1 as [n][D] floats; rows of pages that are not in the pool come as None in `there`."""
        j = np.arange(n)
        page = self.table[b, j // PAGE]
        there = (page >= 0) & (page < pool.shape[0])
        return from_half(pool[np.where(there, page, 0), h, j % PAGE], self.st).astype(np.float64), there


def within(err, tol):
    """The largest error in units of its tolerance (at most 1 where all are within)."""
    err, tol = np.broadcast_arrays(err, tol)
    return float((err / (tol + 1e-37)).max()) if err.size else 0.0


def same(a, b):
    a, b = (np.ascontiguousarray(x) for x in (a, b))
    return a.dtype == b.dtype and a.tobytes() == b.tobytes()


def workspace(mlxr, n):
    assert n > 0
    return mlxr.DeviceArray.zeros(int(n), np.uint8)


# ------------------------------------------------------------------------------------------- attention
def attend(mlxr, c, q, nH, window=0, scale=0.09, weight_in=None, decay=1.0, work=None, out=None, desc=None):
    kv = desc or c.desc()
    dq = mlxr.DeviceArray.from_numpy(q)
    do = out or mlxr.DeviceArray.from_numpy(np.full((c.B, q.shape[1]), 7.0, np.float32))
    n = mlxr.lib.mlxr_k_paged_attention_work(ctypes.byref(kv), nH)
    work = work or workspace(mlxr, n)
    mlxr.check(mlxr.lib.mlxr_k_paged_attention(ctypes.byref(kv), dq.ptr, q.shape[1], nH, window, scale, do.ptr, q.shape[1],
                                               weight_in.ptr if weight_in else None, decay, work.ptr, work.nbytes, None))
    mlxr.synchronize()
    return do.numpy()


def attention_reference(c, q, nH, window, scale):
    """out, its tolerance, the weights of this step and theirs."""
    G, D = nH // c.nKV, c.D
    out, tol = np.zeros((c.B, nH, D)), np.zeros((c.B, nH, D))
    p_sum, p_tol = np.zeros((c.B, c.nKV, c.max_len)), np.zeros((c.B, c.nKV, c.max_len))
    scale = float(np.float32(scale))
    for b in range(c.B):
        L = int(np.clip(c.lens[b], 0, c.max_len))
        first = max(0, L - window) if window else 0
        for h in range(c.nKV):
            if L == 0:
                continue
            (k, there), (v, _) = c.rows(c.k, b, h, L), c.rows(c.v, b, h, L)
            seen = there & (np.arange(L) >= first)
            if not seen.any():
                continue
            k, v = k[seen], v[seen]
            for g in range(h * G, h * G + G):
                x = q[b, g * D:(g + 1) * D].astype(np.float64)
                s = scale * (k @ x)
                e = np.exp(s - s.max())
                p = e / e.sum()
                # a score's error: D products summed, then a few roundings of its own size (scale, base of the exponential)
                ds = 4 * np.sqrt(D) * U * scale * np.sqrt((k ** 2) @ (x ** 2)) + 4 * U * np.abs(s) + 2 * U * np.abs(s).max()
                rel = 2 * ds.max() + 8 * U
                n = len(p)
                out[b, g] = p @ v
                tol[b, g] = rel * (p @ np.abs(v)) + 4 * np.sqrt(n) * U * np.sqrt((p ** 2) @ (v ** 2)) + np.abs(out[b, g]) * (4 * np.sqrt(n) * U * np.sqrt((p ** 2).sum()) + 2 * U)
                p_sum[b, h, np.nonzero(seen)[0]] += p
                p_tol[b, h, np.nonzero(seen)[0]] += p * (rel + 4 * np.sqrt(n) * U * np.sqrt((p ** 2).sum()) + 2 * U)
    return out.reshape(c.B, -1), tol.reshape(c.B, -1), p_sum, p_tol


def queries(c, nH, seed=1, pad=4):
    """Rows of nH heads with a row stride wider by `pad`, NaN in the padding."""
    q = np.full((c.B, nH * c.D + pad), np.nan, np.float32)
    q[:, :nH * c.D] = np.random.default_rng(seed).standard_normal((c.B, nH * c.D)) * 1.5
    return q


def check_out(got, c, nH, out, tol):
    n = nH * c.D
    assert same(got[:, n:], np.full_like(got[:, n:], 7.0)), "padding written"
    assert within(np.abs(got[:, :n] - out), tol) <= 1


HEADS = [(1, 1), (2, 5), (8, 4), (1, 16), (1, 17), (2, 8), (4, 1)]


@pytest.mark.parametrize("nKV,G", HEADS)
@pytest.mark.parametrize("D,st", [(128, 0), (64, 0), (128, 1), (64, 1)])
def test_attention_lengths(gpu, nKV, G, D, st):
    print(f"[case] {nKV} {G} {D} {st}", flush=True)
    c = Cache(gpu, [65, 0, 1, 63, 64, 500, 0, 1025, 31, 33], nKV, D, st, seed=nKV + G).up()
    q = queries(c, nKV * G)
    out, tol, _, _ = attention_reference(c, q, nKV * G, 0, 0.09)
    check_out(attend(gpu, c, q, nKV * G), c, nKV * G, out, tol)


@pytest.mark.parametrize("B,L,nKV,G", [(1, 4096, 8, 4), (1, 1, 8, 4), (1, 20011, 2, 5), (3, 9000, 8, 5), (300, 70, 2, 2), (1, 2, 1, 1)])
def test_attention_sizes(gpu, B, L, nKV, G):
    print(f"[case] {B} {L} {nKV} {G}", flush=True)
    c = Cache(gpu, [max(1, L - 37 * b) if b % 7 else L for b in range(B)], nKV, 128, 0, seed=L).up()
    q = queries(c, nKV * G)
    out, tol, _, _ = attention_reference(c, q, nKV * G, 0, 0.09)
    check_out(attend(gpu, c, q, nKV * G), c, nKV * G, out, tol)


@pytest.mark.parametrize("window", [1, 2, 31, 63, 64, 65, 128, 1000, 1 << 30])
def test_attention_window(gpu, window):
    c = Cache(gpu, [1, 64, 65, 200, 0, 1000, 999], 2, 128, 0, seed=window % 1000).up()
    q = queries(c, 8)
    out, tol, _, _ = attention_reference(c, q, 8, window, 0.09)
    check_out(attend(gpu, c, q, 8, window=window), c, 8, out, tol)


@pytest.mark.parametrize("nKV,G,D,st", [(2, 5, 128, 0), (8, 4, 128, 1), (1, 17, 64, 0), (4, 1, 64, 1)])
@pytest.mark.parametrize("window,decay,source", [(0, 1.0, "other"), (0, 0.0, "nan"), (100, 0.5, "other"), (64, 0.9, "same"), (0, 1.0, "none")])
def test_attention_weights(gpu, nKV, G, D, st, window, decay, source):
    print(f"[case] {nKV} {G} {D} {st} {window} {decay} {source}", flush=True)
    nH = nKV * G
    c = Cache(gpu, [65, 0, 1, 500, 2049, 64], nKV, D, st, seed=11, weight=True).up()
    before = c.weight.copy()
    q = queries(c, nH)
    given = np.full_like(before, np.nan) if source == "nan" else np.random.default_rng(2).exponential(1, before.shape).astype(np.float32)
    arg = {"other": lambda: gpu.DeviceArray.from_numpy(given), "nan": lambda: gpu.DeviceArray.from_numpy(given), "same": lambda: c.dw, "none": lambda: None}[source]()
    given = {"other": given, "nan": np.zeros_like(before), "same": before, "none": np.zeros_like(before)}[source]
    out, tol, p, p_tol = attention_reference(c, q, nH, window, 0.09)
    check_out(attend(gpu, c, q, nH, window=window, weight_in=arg, decay=decay), c, nH, out, tol)
    got = c.dw.numpy()
    for b in range(c.B):
        L = int(c.lens[b])
        kept = float(np.float32(decay)) * given[b, :, :L].astype(np.float64)
        want = kept + p[b, :, :L]
        assert within(np.abs(got[b, :, :L] - want), p_tol[b, :, :L] + 2 * U * (np.abs(kept) + np.abs(want)) + (G + 2) * U * p[b, :, :L]) <= 1
        assert same(got[b, :, L:], before[b, :, L:]), "weights behind the length written"


def test_attention_scores_of_every_size(gpu):
    """Scores far apart (one key takes all), all equal, and tiny: no overflow, no NaN."""
    for size in (0.0, 1e-20, 60.0, 3000.0):
        c = Cache(gpu, [700, 1, 129], 2, 128, 0, seed=3).up()
        q = queries(c, 8) * np.float32(size)
        out, tol, _, _ = attention_reference(c, q, 8, 0, 0.09)
        got = attend(gpu, c, q, 8)
        assert np.isfinite(got[:, :8 * 128]).all()
        # where scores are thousands their rounding alone moves p: the bound grows with them, up to the values' own size
        check_out(got, c, 8, out, np.minimum(tol, 20.0))


def test_attention_odd_lengths_on_the_device(gpu):
    """Lengths outside [0, max_len] count as the bounds; pages outside the pool hold no keys."""
    c = Cache(gpu, [200, 200, 130, 64, 320], 2, 128, 0, seed=5)
    c.lens[:] = [-5, 1 << 30, 130, 64, 320]
    c.max_len = 200
    c.table[1, 3:] = -1                # slots 192 .. 199 of sequence 1
    c.table[2, 1] = c.k.shape[0]       # slots 64 .. 127 of sequence 2
    c.table[3, 0] = -2147483648        # all of sequence 3
    c.up()
    q = queries(c, 8)
    out, tol, _, _ = attention_reference(c, q, 8, 0, 0.09)
    assert not out[0].any() and not out[3].any()
    check_out(attend(gpu, c, q, 8), c, 8, out, tol)


def test_attention_shared_pages_and_minus_infinity(gpu):
    """Sequences that share pages, and keys whose scores are -infinity: they take no part; where all are, the row is zeros."""
    c = Cache(gpu, [256, 256, 64], 1, 128, 0, seed=6, weight=True)
    c.table[1] = c.table[0]
    q = queries(c, 2)
    q[:, :256] = np.abs(q[:, :256])
    c.k[c.table[0, 1], 0, 5] = to_half(np.float32(-3e38), 0)      # the score overflows to -infinity
    c.k[c.table[2, 0]] = to_half(np.float32(-3e38), 0)
    c.up()
    got = attend(gpu, c, q, 2, scale=1.0)
    assert np.isfinite(got[:, :256]).all() and not got[2, :256].any()
    skip = np.arange(256) != 69
    for b in range(2):
        (k, _), (v, _) = c.rows(c.k, 0, 0, 256), c.rows(c.v, 0, 0, 256)
        for g in range(2):
            s = k[skip] @ q[b, g * 128:(g + 1) * 128].astype(np.float64)
            p = np.exp(s - s.max())
            p /= p.sum()
            assert np.abs(got[b, g * 128:(g + 1) * 128] - p @ v[skip]).max() < 1e-3   # scores of up to 100: 2 * 100 * 45 u
    assert (c.dw.numpy()[0, 0, 69] == 0) and not c.dw.numpy()[2, 0, :64].any()


def test_attention_same_bits_again(gpu):
    """The same call gives the same bits, whatever ran in its workspace before."""
    big = Cache(gpu, [3000, 17, 900], 8, 128, 0, seed=7).up()
    small = Cache(gpu, [130, 64], 2, 128, 0, seed=8).up()
    kv = big.desc()
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_work(ctypes.byref(kv), 32))
    qb, qs = queries(big, 32), queries(small, 4)
    a = attend(gpu, big, qb, 32, work=work)
    s = attend(gpu, small, qs, 4, work=work)
    for _ in range(3):
        assert same(attend(gpu, big, qb, 32, work=work).view(np.uint32), a.view(np.uint32))
        assert same(attend(gpu, small, qs, 4, work=work).view(np.uint32), s.view(np.uint32))


def test_attention_many_sequences(gpu):
    """More sequences than a workgroup scans at once, most of them short, idle ones among them."""
    rs = np.random.default_rng(13)
    lens = rs.integers(0, 70, 1300)
    lens[::9] = 0
    lens[[5, 700, 1299]] = [700, 1, 333]
    c = Cache(gpu, lens, 1, 64, 0, seed=14).up()
    q = queries(c, 2)
    out, tol, _, _ = attention_reference(c, q, 2, 0, 0.09)
    check_out(attend(gpu, c, q, 2), c, 2, out, tol)


def test_attention_in_place(gpu):
    """The output over the queries, at their stride."""
    c = Cache(gpu, [500, 0, 2000, 64], 2, 128, 0, seed=15).up()
    q = queries(c, 8, pad=0)
    out, tol, _, _ = attention_reference(c, q, 8, 0, 0.09)
    kv, dq = c.desc(), gpu.DeviceArray.from_numpy(q)
    work = workspace(gpu, gpu.lib.mlxr_k_paged_attention_work(ctypes.byref(kv), 8))
    gpu.check(gpu.lib.mlxr_k_paged_attention(ctypes.byref(kv), dq.ptr, 1024, 8, 0, 0.09, dq.ptr, 1024, None, 1.0, work.ptr, work.nbytes, None))
    gpu.synchronize()
    assert within(np.abs(dq.numpy() - out), tol) <= 1


def far_pool(gpu, c, page_bytes):
    """The cache's pages at the far end of pools whose offsets pass 2^32 elements and more; the table goes with them."""
    pages = (1 << 32) // (page_bytes // 2) + 64 + c.k.shape[0]
    pools = [gpu.DeviceArray(pages * page_bytes, np.uint8) for _ in range(2)]
    shift = pages - c.k.shape[0]
    for pool, a in zip(pools, (c.k, c.v)):
        gpu.check(gpu.lib.mlxr_memcpy_h2d(pool.ptr + shift * page_bytes, a.ctypes.data, a.nbytes))
    return pools, pages, shift


def fetch(gpu, pool, at, like):
    a = np.empty_like(like)
    gpu.check(gpu.lib.mlxr_memcpy_d2h(a.ctypes.data, pool.ptr + at, a.nbytes))
    return a


def test_offsets_past_32_bits(gpu):
    """The same step with its pages behind 2^32 elements of the pools: the same bits from append, attention and eviction."""
    nKV, D, nH = 8, 128, 32
    page_bytes = nKV * PAGE * D * 2
    src, dst = pair(gpu, [200, 64, 300], nKV, D, 0, 100, seed=51)
    src.up(), dst.up()
    rs = np.random.default_rng(52)
    qkv, inv = rs.standard_normal((3, (nH + 2 * nKV) * D)).astype(np.float32), (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    pools, pages, shift = far_pool(gpu, src, page_bytes)
    tables = [gpu.DeviceArray.from_numpy(np.where(t < 0, -1, t + shift).astype(np.int32)) for t in (src.table, dst.table)]
    near = run_append(gpu, src, qkv, nH, inv, None, None, D, 0, None, 1e-6, False, q_pad=0)[0]
    got = [attend(gpu, src, near, nH)]
    evict(gpu, src, dst, 100, 4, 16)
    k_near, v_near = src.dk.numpy(), src.dv.numpy()
    far = dict(k=pools[0].ptr, v=pools[1].ptr, n_pages=pages)
    a, b = src.desc(table=tables[0].ptr, **far), dst.desc(table=tables[1].ptr, **far)
    dx, df, dq = gpu.DeviceArray.from_numpy(qkv), gpu.DeviceArray.from_numpy(inv), gpu.DeviceArray.zeros((3, nH * D), np.float32)
    gpu.check(gpu.lib.mlxr_k_paged_append(ctypes.byref(a), dx.ptr, qkv.shape[1], df.ptr, None, None, nH, D, 0, None, 1e-6, dq.ptr, nH * D, None))
    assert same(dq.numpy(), near)
    got.append(attend(gpu, src, near, nH, desc=a))
    assert same(got[0], got[1])
    work = workspace(gpu, gpu.lib.mlxr_k_paged_evict_work(ctypes.byref(a), 100))
    # the attention above kept weights: eviction reads them as they are now in both runs' arrays
    gpu.check(gpu.lib.mlxr_k_paged_evict(ctypes.byref(a), ctypes.byref(b), 100, 4, 16, work.ptr, work.nbytes, None))
    gpu.synchronize()
    assert same(fetch(gpu, pools[0], shift * page_bytes, src.k), k_near) and same(fetch(gpu, pools[1], shift * page_bytes, src.v), v_near)


def test_sample_far_rows(gpu):
    """Rows of logits 2^30 and more floats apart."""
    V, stride, R = 40000, (1 << 30) + 3, 4
    x = model_logits(np.random.default_rng(53), R, V)
    buf = gpu.DeviceArray((R - 1) * stride + V, np.float32)
    for r in range(R):
        gpu.check(gpu.lib.mlxr_memcpy_h2d(buf.ptr + 4 * r * stride, x[r].ctypes.data, x[r].nbytes))
    d = gpu.DeviceArray.from_numpy
    t, p, u, tok = d(np.full(R, 0.8, np.float32)), d(np.full(R, 0.9, np.float32)), d(np.array([0.1, 0.5, 0.9, 0.99], np.float32)), gpu.DeviceArray.zeros(R, np.int32)
    work = workspace(gpu, gpu.lib.mlxr_k_sample_rows_work(R, V))
    gpu.check(gpu.lib.mlxr_k_sample_rows(buf.ptr, R, V, stride, t.ptr, None, p.ptr, None, u.ptr, tok.ptr, None, work.ptr, work.nbytes, None))
    gpu.synchronize()
    assert same(tok.numpy(), sample(gpu, x, 0.8, p=0.9, u=[0.1, 0.5, 0.9, 0.99])[0])


# ------------------------------------------------------------------------------------------- append
def run_append(mlxr, c, qkv, nH, inv_freq, qn, kn, rot, traditional, positions, eps, in_place, q_pad=2):
    d = mlxr.DeviceArray.from_numpy
    dx, df = d(qkv), d(inv_freq if len(inv_freq) else np.zeros(1, np.float32))
    dq = dx if in_place else d(np.full((c.B, nH * c.D + q_pad), 7.0, np.float32))
    keep = [d(x) if x is not None else None for x in (qn, kn, positions)]
    kv = c.desc()
    mlxr.check(mlxr.lib.mlxr_k_paged_append(ctypes.byref(kv), dx.ptr, qkv.shape[1], df.ptr, keep[0] and keep[0].ptr, keep[1] and keep[1].ptr, nH, rot,
                                            traditional, keep[2] and keep[2].ptr, eps, dq.ptr, dq.shape[1], None))
    mlxr.synchronize()
    return dq.numpy(), dx.numpy()


@pytest.mark.parametrize("nH,nKV,D,st,rot,traditional,norm,positions,in_place", [
    (32, 8, 128, 0, 128, 0, True, True, False), (40, 8, 128, 1, 64, 0, False, True, True), (3, 1, 64, 0, 64, 1, True, True, False),
    (4, 4, 64, 1, 32, 1, True, False, True), (5, 5, 128, 0, 0, 0, True, True, False), (16, 2, 128, 1, 126, 1, False, False, False),
    (2, 1, 64, 0, 2, 0, False, True, False)])
def test_append(gpu, nH, nKV, D, st, rot, traditional, norm, positions, in_place):
    lens = [1, 64, 65, 0, 128, 200, 129]
    c = Cache(gpu, lens, nKV, D, st, seed=rot, weight=True, position=True)
    rs = np.random.default_rng(4)
    B, pad = len(lens), 3
    qkv = rs.standard_normal((B, (nH + 2 * nKV) * D + pad)).astype(np.float32)
    inv = (1e6 ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32)
    qn, kn = (rs.uniform(0.5, 1.5, D).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pos = np.array([0, 131071, 1, 5, 99999, 7, 12345], np.int32) if positions else None
    k, v, w, p = c.k.copy(), c.v.copy(), c.weight.copy(), c.position.copy()
    c.up()
    q, x_after = run_append(gpu, c, qkv, nH, inv, qn, kn, rot, traditional, pos, 1e-6, in_place)
    x = qkv[:, :(nH + 2 * nKV) * D].astype(np.float64).reshape(B, -1, D)
    h = x[:, :nH + nKV].copy()
    if norm:
        h /= np.sqrt((h ** 2).mean(-1, keepdims=True) + float(np.float32(1e-6)))
        h[:, :nH] *= qn
        h[:, nH:] *= kn
    at = pos if positions else np.array(lens) - 1
    ang = at[:, None] * inv.astype(np.float64)
    cos, sin = np.cos(ang)[:, None], np.sin(ang)[:, None]
    half = rot // 2
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if traditional else (np.arange(half), np.arange(half, rot))
    a, b_ = h[..., ia].copy(), h[..., ib].copy()
    size = np.abs(h)
    size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b_)
    h[..., ia], h[..., ib] = a * cos - b_ * sin, b_ * cos + a * sin
    # norm: a mean of D squares (half its relative error: 2 sqrt(D) u), root, quotient, two products; rotation: sine and
    # cosine to 4 u of one, two products and a sum
    tol = size * ((2 * np.sqrt(D) + 6) * U * norm + 8 * U)
    idle = np.array(lens) == 0
    n = nH * D
    got_q = q[:, :n].reshape(B, nH, D)
    assert within(np.abs(got_q - h[:, :nH])[~idle], tol[:, :nH][~idle]) <= 1
    if in_place:
        assert same(q[:, n:], qkv[:, n:]) and same(q[idle], qkv[idle])
    else:
        assert same(q[:, n:], np.full_like(q[:, n:], 7.0)) and same(q[idle], np.full_like(q[idle], 7.0))
        assert same(x_after, qkv)
    step = 2.0 ** -8 if st == 0 else 2.0 ** -11
    for b in range(B):
        if lens[b] == 0:
            continue
        page, row = c.table[b, (lens[b] - 1) // PAGE], (lens[b] - 1) % PAGE
        got_k = from_half(c.dk.numpy()[page, :, row], st)
        want = h[b, nH:]
        assert within(np.abs(got_k - want), tol[b, nH:] * (1 + step) + step * np.abs(want) + 2.0 ** -25 * st) <= 1
        k[page, :, row] = c.dk.numpy()[page, :, row]
        v[page, :, row] = to_half(x[b, nH + nKV:].astype(np.float32), st)
        w[b, :, lens[b] - 1] = 0
        p[b, :, lens[b] - 1] = at[b]
    assert same(c.dk.numpy(), k) and same(c.dv.numpy(), v)
    assert same(c.dw.numpy(), w) and same(c.dp.numpy(), p)


def test_append_bad_pages(gpu):
    """A page outside the pool takes nothing; the query still comes."""
    c = Cache(gpu, [65, 64], 2, 128, 0, seed=9)
    c.table[0, 1], c.table[1, 0] = c.k.shape[0], -7
    c.up()
    qkv = np.random.default_rng(1).standard_normal((2, 6 * 128)).astype(np.float32)
    q, _ = run_append(gpu, c, qkv, 2, np.zeros(0, np.float32), None, None, 0, 0, None, 1e-6, False)
    assert same(q[:, :256], qkv[:, :256])
    assert same(c.dk.numpy(), c.k) and same(c.dv.numpy(), c.v)


# ------------------------------------------------------------------------------------------- eviction
def evict(mlxr, src, dst, budget, sink, window, work=None):
    a, b = src.desc(), dst.desc(k=src.dk.ptr, v=src.dv.ptr, n_pages=src.k.shape[0]) if dst.k is src.k else dst.desc()
    n = mlxr.lib.mlxr_k_paged_evict_work(ctypes.byref(a), budget)
    work = work or workspace(mlxr, n)
    mlxr.check(mlxr.lib.mlxr_k_paged_evict(ctypes.byref(a), ctypes.byref(b), budget, sink, window, work.ptr, work.nbytes, None))
    mlxr.synchronize()


def kept_slots(w, n, budget, sink, window):
    if n <= budget:
        return np.arange(n)
    w = np.where(np.isnan(w), -np.inf, w).astype(np.float64) + 0.0
    nan = np.isnan(w)
    mid = np.arange(sink, n - window)
    mid = mid[np.lexsort((mid, nan[mid], -w[mid]))][:budget - sink - window]
    return np.sort(np.concatenate([np.arange(sink), mid, np.arange(n - window, n)])).astype(int)


def check_evicted(src, dst, budget, sink, window, k0, v0, w0, p0):
    """src's arrays are the host copies from before; dst's device arrays are compared with what they must hold."""
    want_k, want_v, want_w, want_p = k0.copy(), v0.copy(), w0.copy() if w0 is not None else None, p0.copy() if p0 is not None else None
    lens = []
    for b in range(src.B):
        n = int(np.clip(src.lens[b], 0, src.max_len))
        lens.append(min(n, budget))
        for h in range(src.nKV):
            kept = kept_slots(src.weight[b, h, :n], n, budget, sink, window)
            assert len(kept) == lens[-1]
            j = np.arange(len(kept))
            to = dst.table[b, j // PAGE]
            there = (to >= 0) & (to < k0.shape[0])
            page = src.table[b, kept // PAGE]
            known = (page >= 0) & (page < src.k.shape[0])
            for want, pool in ((want_k, src.k), (want_v, src.v)):
                rows = np.where(known[:, None], pool[np.where(known, page, 0), h, kept % PAGE], 0)
                want[to[there], h, j[there] % PAGE] = rows[there]
            if want_w is not None:
                want_w[b, h, :len(kept)] = src.weight[b, h, kept]
            if want_p is not None:
                want_p[b, h, :len(kept)] = src.position[b, h, kept]
    assert same(dst.dlen.numpy(), np.array(lens, np.int32))
    if want_w is not None:
        assert same(dst.dw.numpy().view(np.uint32), want_w.view(np.uint32))
    if want_p is not None:
        assert same(dst.dp.numpy(), want_p)
    pools = (src if dst.k is src.k else dst)
    assert same(pools.dk.numpy(), want_k) and same(pools.dv.numpy(), want_v)


def pair(gpu, lens, nKV, D, st, budget, seed=0, same_pool=True, **dst_over):
    """A source, and a destination of `budget` slots a sequence: in the source's pool, or in one of its own."""
    room = [min(max(n, 0), budget) for n in lens]
    need = sum(-(-r // PAGE) for r in room)
    src = Cache(gpu, lens, nKV, D, st, seed=seed, extra_pages=need + 2, weight=True, position=True)
    over = dict(weight=True, position=True)
    over.update(dst_over)
    dst = Cache(gpu, [1] * len(lens), nKV, D, st, seed=seed + 1, room=room, max_len=max(1, min(budget, src.max_len)), **over)
    if same_pool:
        at = 0
        for b, r in enumerate(room):
            n = -(-r // PAGE)
            dst.table[b, :n] = src.free[at:at + n]
            at += n
        dst.k, dst.v = src.k, src.v
    return src, dst


@pytest.mark.parametrize("budget,sink,window", [(100, 4, 32), (64, 0, 0), (1, 0, 0), (1, 1, 0), (7, 0, 7), (100, 50, 50), (1000, 4, 100), (333, 0, 1), (5000, 4, 4)])
@pytest.mark.parametrize("nKV,D,st", [(2, 128, 0), (3, 64, 1)])
@pytest.mark.parametrize("same_pool", [True, False])
def test_evict(gpu, budget, sink, window, nKV, D, st, same_pool):
    print(f"[case] {budget} {sink} {window} {nKV} {D} {st} {same_pool}", flush=True)
    lens = [0, 1, 63, 64, 100, 101, 999, 2500, 333]
    src, dst = pair(gpu, lens, nKV, D, st, budget, seed=budget, same_pool=same_pool)
    src.weight[:, :, ::5] = np.round(src.weight[:, :, ::5])      # ties
    src.weight[6] = 1.0                                          # nothing but ties
    src.weight[7, 0, 100:400] = [np.nan, np.inf, -np.inf, -0.0, 0.0, -1.5] * 50
    src.up(), dst.up()
    k0, v0 = (src.k.copy(), src.v.copy()) if same_pool else (dst.k.copy(), dst.v.copy())
    evict(gpu, src, dst, budget, sink, window)
    check_evicted(src, dst, budget, sink, window, k0, v0, dst.weight, dst.position)


def test_evict_long(gpu):
    src, dst = pair(gpu, [70001, 128, 33000], 1, 64, 0, 20000, seed=21)
    src.weight[0, 0, 1000:60000:2] = 0.0
    src.up(), dst.up()
    evict(gpu, src, dst, 20000, 4, 512)
    check_evicted(src, dst, 20000, 4, 512, src.k.copy(), src.v.copy(), dst.weight, dst.position)


def test_evict_without_arrays_and_bad_pages(gpu):
    """dst without weights and positions; a source page outside the pool copies as zeros, a target one takes nothing;
    lengths outside their bounds."""
    src, dst = pair(gpu, [200, 300, 64, 129], 2, 128, 0, 130, seed=31, weight=False, position=False)
    src.table[0, 1] = src.k.shape[0]
    src.table[2, 0] = -1
    dst.table[1, 1] = -3
    dst.table[3, 0] = 1 << 30
    src.lens[1], src.lens[3] = 1 << 29, -1
    src.table[1, :] = np.where(src.table[1, :] < 0, src.table[1, 0], src.table[1, :])
    src.up(), dst.up()
    evict(gpu, src, dst, 130, 4, 32)
    check_evicted(src, dst, 130, 4, 32, src.k.copy(), src.v.copy(), None, None)


def test_evict_from_shared_pages(gpu):
    """Two sequences over the same source pages (a shared prefix) are held at their own weights."""
    src, dst = pair(gpu, [500, 500], 2, 128, 0, 128, seed=41)
    src.table[1] = src.table[0]
    src.up(), dst.up()
    evict(gpu, src, dst, 128, 4, 32)
    check_evicted(src, dst, 128, 4, 32, src.k.copy(), src.v.copy(), dst.weight, dst.position)


# ------------------------------------------------------------------------------------------- sampling
def sample(mlxr, logits, t, k=None, p=None, low=None, u=None, stride=None, status=True, work=None):
    R, V = logits.shape
    stride = stride or V
    buf = np.full((R, stride), np.float32(1e30))
    buf[:, :V] = logits
    d = lambda x, ty: mlxr.DeviceArray.from_numpy(np.ascontiguousarray(np.broadcast_to(np.asarray(x, ty), (R,)))) if x is not None else None  # noqa: E731
    dl, dt, dk, dp, dm, du = mlxr.DeviceArray.from_numpy(buf), d(t, np.float32), d(k, np.int32), d(p, np.float32), d(low, np.float32), d(u, np.float32)
    tok, st = mlxr.DeviceArray.from_numpy(np.full(R + 1, -9, np.int32)), mlxr.DeviceArray.from_numpy(np.full(R + 1, -9, np.int32))
    work = work or workspace(mlxr, mlxr.lib.mlxr_k_sample_rows_work(R, V))
    o = lambda x: x.ptr if x else None  # noqa: E731
    mlxr.check(mlxr.lib.mlxr_k_sample_rows(dl.ptr, R, V, stride, dt.ptr, o(dk), o(dp), o(dm), du.ptr, tok.ptr, st.ptr if status else None,
                                           work.ptr, work.nbytes, None))
    mlxr.synchronize()
    assert same(dl.numpy(), buf), "logits written"
    tok, st = tok.numpy(), st.numpy()
    assert tok[R] == -9 and st[R] == -9
    return tok[:R], st[:R] if status else None


def reference_token(v, t, k, p, low, u):
    """(tokens that may come, status): one token, or those next to a border that the goal lies on. The kernel's weights
    are multiples of 2^-43 (off by 2^-44 each), its sums exact: a border may be off by V 2^-44."""
    v = np.asarray(v, np.float64)
    ok = ~np.isnan(v) & (v != -np.inf)
    if not ok.any() or v[ok].max() == np.inf:
        return {0}, 1
    idx = np.nonzero(ok)[0]
    order = idx[np.lexsort((idx, -v[idx]))]
    if not t > 0.001:
        return {int(order[0])}, 0
    if k is not None and k > 0:
        order = order[:k]
    w = np.exp((v[order] - v[order[0]]) / float(np.float32(t))) if np.isfinite(t) else np.ones(len(order))
    run = np.cumsum(w)
    slack = len(v) * 2.0 ** -44 + 1e-12 * run[-1]
    ends = [len(w)]
    if p is not None and p < 1:
        goal = float(np.float32(p)) * run[-1]
        ends = [max(1, min(len(w), int(np.searchsorted(run, goal + e)) + 1)) for e in (-slack, 0, slack)]
    if low is not None and low > 0:
        below = np.nonzero(w < float(np.float32(low)))[0]
        ends = [max(1, min(e, int(below[0]) if below.size else e)) for e in ends]
    may = set()
    for e in set(ends):
        goal = (float(np.float32(u)) if u == u else 0.0) * run[e - 1]
        first, last = (min(e - 1, int(np.searchsorted(run[:e], goal + d))) for d in (-slack, slack))
        may.update(int(i) for i in order[first:last + 1])   # every token whose border lies within the slack
    return may, 0


def check_tokens(gpu, logits, t, k=None, p=None, low=None, u=None, **kw):
    R = logits.shape[0]
    tok, st = sample(gpu, logits, t, k, p, low, u, **kw)
    at = lambda x, r: None if x is None else (x[r] if np.ndim(x) else x)  # noqa: E731
    doubtful = 0
    for r in range(R):
        may, status = reference_token(logits[r], at(t, r), at(k, r), at(p, r), at(low, r), at(u, r))
        assert tok[r] in may, (r, int(tok[r]), may, at(t, r), at(k, r), at(p, r), at(low, r), at(u, r))
        assert st is None or st[r] == status
        doubtful += len(may) > 1
    return tok, doubtful


def model_logits(rs, R, V, n=64):
    x = rs.standard_normal((R, V)).astype(np.float32) * 2
    x[np.arange(R)[:, None], rs.integers(0, V, (R, n))] = 6 + 8 * rs.random((R, n))
    return x


@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 1000, 4097, 32000, 151936])
def test_sample_parameters(gpu, V):
    print(f"[case] V={V}", flush=True)
    rs = np.random.default_rng(V)
    R = 48 if V < 100000 else 24
    x = model_logits(rs, R, V)
    u = rs.random(R).astype(np.float32)
    u[:3] = [0.0, 1 - 2.0 ** -24, 0.5]
    doubtful = 0
    for t, k, p, low in [(0.7, 40, 0.95, 0.0), (1.0, None, None, None), (0.0, 40, 0.9, None), (1.0, 0, 0.9, None), (1.3, None, None, 0.05), (0.001, None, None, None),
                         (0.5, 1, None, None), (2.0, 3000, 0.99, 0.001), (5.0, None, 0.999, None), (np.inf, None, None, None), (0.0011, None, None, None),
                         (1.0, 10 ** 9, 1.0, 0.0), (1.0, -3, 0.0, None), (1.0, None, 1e-9, None), (1.0, None, None, 1.0), (1.0, None, None, 7.0), (100.0, 700, 0.5, 0.9)]:
        doubtful += check_tokens(gpu, x, t, k, p, low, u)[1]
    assert doubtful < 17   # the reference decides nearly all


@pytest.mark.parametrize("V", [1500, 30000, 151936])
def test_sample_temperatures(gpu, V):
    """Temperatures around and above 1 over logits that reach far down (to -200, where weight may lie far behind the bins)."""
    print(f"[case] V={V}", flush=True)
    rs = np.random.default_rng(V)
    x = model_logits(rs, 12, V)
    x[4:8] = rs.uniform(-200, 0, (4, V))
    x[8:] -= rs.exponential(15, (4, V)).astype(np.float32)
    u = rs.random(12).astype(np.float32)
    u[[0, 5, 9]] = 1 - 2.0 ** -24
    doubtful = 0
    for t in (0.05, 0.999, 1.0, 1.001, 1.7, 3.0, 5.0, 8.0, 9.5, 40.0, 1e4):
        for k, p, low in [(None, 0.9, None), (None, None, None), (40, 0.95, None), (None, None, 0.03), (700, 0.99, 1e-6), (None, 0.999, 1e-5), (None, None, 1e-20)]:
            doubtful += check_tokens(gpu, x, t, k, p, low, u)[1]
    assert doubtful < 80   # of 924: the three rows drawn at 1 - 2^-24 end among tokens lighter than the slack


@pytest.mark.parametrize("V,stride", [(151936, 151936), (50257, 50258), (777, 779)])
def test_sample_mixed_rows(gpu, V, stride):
    rs = np.random.default_rng(7)
    R = 64
    x = model_logits(rs, R, V)
    t = rs.choice([0.0, 0.3, 0.7, 1.0, 1.5], R).astype(np.float32)
    k = rs.choice([0, 1, 5, 40, 200, 1024, 1025, 5000], R).astype(np.int32)
    p = rs.choice([1.0, 0.3, 0.9, 0.99], R).astype(np.float32)
    low = rs.choice([0.0, 0.01, 0.2], R).astype(np.float32)
    check_tokens(gpu, x, t, k, p, low, rs.random(R).astype(np.float32), stride=stride)


@pytest.mark.parametrize("V", [262145, 300001, 1 << 20])
def test_sample_large_vocabularies(gpu, V):
    print(f"[case] V={V}", flush=True)
    rs = np.random.default_rng(V)
    x = model_logits(rs, 4, V, 300)
    x[3] = rs.integers(0, 3, V)
    for t, k, p, low in [(0.7, 40, 0.95, 0.0), (1.0, None, 0.9, None), (1.0, None, None, None), (0.0, None, None, None), (1.0, None, None, 0.02), (1.0, 5000, 0.9, None)]:
        check_tokens(gpu, x, t, k, p, low, rs.random(4).astype(np.float32))


def test_sample_ties(gpu):
    """Equal logits are ranked by index, at every cut: rows of one value, of three, and of +0 and -0."""
    rs = np.random.default_rng(3)
    V = 5000
    x = np.zeros((12, V), np.float32)
    x[1] = -7.25
    x[2:6] = rs.choice([1.0, 2.0, 2.5], (4, V)).astype(np.float32)
    x[6] = np.where(np.arange(V) % 2, np.float32(0.0), np.float32(-0.0))
    x[7:] = rs.integers(-8, 8, (5, V)).astype(np.float32)
    for k, p, low in [(None, None, None), (100, None, None), (4000, 0.5, None), (None, 0.7, None), (None, None, 0.3), (1, None, None)]:
        for t in (1.0, 0.0):
            check_tokens(gpu, x, t, k, p, low, rs.random(12).astype(np.float32))


def test_sample_masked_rows(gpu):
    """Masks of -infinity, of the lowest float and of NaN; rows that leave one token, and none; infinite logits."""
    rs = np.random.default_rng(5)
    V = 3001
    x = np.full((10, V), -np.inf, np.float32)
    x[1, 2999] = -5.0                                         # one token
    x[2] = np.nan                                             # none
    x[3, :] = np.finfo(np.float32).min
    x[3, 17] = 3.0
    x[4] = rs.standard_normal(V); x[4, ::2] = np.nan
    x[5] = rs.standard_normal(V); x[5, ::3] = -np.inf
    x[6] = rs.standard_normal(V); x[6, 100] = np.inf
    x[7] = np.finfo(np.float32).min                           # all the lowest number: all equal
    x[8] = np.finfo(np.float32).max
    x[9, :50] = rs.standard_normal(50)
    for t, k, p, low in [(1.0, None, None, None), (0.0, None, None, None), (0.7, 100, 0.9, 0.01), (np.inf, None, 0.5, None), (1.0, 2900, None, None)]:
        _, _ = check_tokens(gpu, x, t, k, p, low, np.linspace(0, 1 - 2.0 ** -24, 10).astype(np.float32))
    assert list(sample(gpu, x, 1.0, u=0.5)[1]) == [1, 0, 1, 0, 0, 0, 1, 0, 0, 0]


def test_sample_odd_numbers(gpu):
    """u outside [0, 1) counts as its bounds and NaN as 0; NaN parameters are off; a NaN temperature is greedy; no status."""
    rs = np.random.default_rng(6)
    x = model_logits(rs, 4, 2000)
    lo = sample(gpu, x, 1.0, u=0.0)[0]
    assert same(sample(gpu, x, 1.0, u=-3.0)[0], lo) and same(sample(gpu, x, 1.0, u=np.nan)[0], lo)
    hi = sample(gpu, x, 1.0, k=50, u=1.0)[0]
    assert same(sample(gpu, x, 1.0, k=50, u=9.0)[0], hi)
    want = [int(np.lexsort((np.arange(2000), -r))[49]) for r in x]
    assert list(hi) == want
    assert same(sample(gpu, x, np.nan, u=0.9)[0], x.argmax(1).astype(np.int32))
    assert same(sample(gpu, x, 1.0, p=np.nan, low=np.nan, u=0.7)[0], sample(gpu, x, 1.0, u=0.7)[0])
    assert same(sample(gpu, x, 1.0, u=0.7, status=False)[0], sample(gpu, x, 1.0, u=0.7)[0])


def test_sample_distribution(gpu):
    """4096 draws of one row spread as its probabilities do (4.5 standard deviations)."""
    rs = np.random.default_rng(8)
    v = np.log(np.array([0.5, 0.2, 0.15, 0.1, 0.05], np.float32))
    R = 4096
    tok, _ = sample(gpu, np.tile(v, (R, 1)), 1.0, u=rs.random(R).astype(np.float32))
    for i, p in enumerate([0.5, 0.2, 0.15, 0.1, 0.05]):
        assert abs((tok == i).sum() - R * p) < 4.5 * np.sqrt(R * p * (1 - p))


def test_sample_many_rows_and_again(gpu):
    """More rows than the card has compute units, twice through one workspace that held other sizes: the same tokens."""
    rs = np.random.default_rng(9)
    x = model_logits(rs, 700, 1500)
    u = rs.random(700).astype(np.float32)
    work = workspace(gpu, max(gpu.lib.mlxr_k_sample_rows_work(700, 1500), gpu.lib.mlxr_k_sample_rows_work(3, 151936)))
    a = check_tokens(gpu, x, 0.9, 50, 0.9, None, u, work=work)[0]
    y = model_logits(rs, 3, 151936)
    check_tokens(gpu, y, 1.0, None, 0.9, None, u[:3], work=work)
    assert same(sample(gpu, x, 0.9, 50, 0.9, None, u, work=work)[0], a)


# ------------------------------------------------------------------------------------------- together
class Hip:
    """The few calls of the HIP runtime that a program with streams and graphs of its own makes."""

    def __init__(self, mlxr):
        self.lib = ctypes.CDLL("libamdhip64.so.7")   # the one that libmlxr runs on
        self.mlxr = mlxr

    def __call__(self, name, *args):
        assert getattr(self.lib, name)(*args) == 0, name

    def stream(self):
        s = ctypes.c_void_p()
        self("hipStreamCreateWithFlags", ctypes.byref(s), 1)   # non-blocking, the default priority
        return s

    def wait(self, s):
        self("hipStreamSynchronize", s)

    def capture(self, s, run):
        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        self("hipStreamBeginCapture", s, 2)   # relaxed
        try:
            run()
        finally:
            self("hipStreamEndCapture", s, ctypes.byref(graph))
        self("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
        return ex


class Step:
    """A batch's decode state, two sets of pages of one pool, and one step of it: append, attention, a token from the
    attention's output as logits, and where asked the eviction into the other set."""

    def __init__(self, gpu, seed=0, lens=(130, 40, 64), nH=8, nKV=2, D=128, top=256, budget=96):
        self.gpu, self.B, self.nH, self.nKV, self.D, self.top, self.budget = gpu, len(lens), nH, nKV, D, top, budget
        rs, B, per = np.random.default_rng(seed), len(lens), top // PAGE
        d = gpu.DeviceArray.from_numpy
        shape = (2 * B * per, nKV, PAGE, D)
        pages = rs.permutation(2 * B * per).astype(np.int32).reshape(2, B, per)
        self.k, self.v = (d(to_half(rs.standard_normal(shape), 0)) for _ in range(2))
        self.tables, self.table = pages, [d(pages[0]), d(pages[1])]
        self.len = [d(np.array(lens, np.int32)), gpu.DeviceArray.zeros(B, np.int32)]
        self.weight = [d(rs.exponential(1, (B, nKV, top)).astype(np.float32)), gpu.DeviceArray.zeros((B, nKV, top), np.float32)]
        self.position = [d(np.ascontiguousarray(np.broadcast_to(np.arange(top, dtype=np.int32), (B, nKV, top)))) for _ in range(2)]
        self.pos = d(np.array(lens, np.int32) - 1)
        self.inv_freq = (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
        self.inv, self.qkv = d(self.inv_freq), d(rs.standard_normal((B, (nH + 2 * nKV) * D)).astype(np.float32))
        self.q, self.out = gpu.DeviceArray.zeros((B, nH * D), np.float32), gpu.DeviceArray.zeros((B, nH * D), np.float32)
        self.t, self.u = d(np.full(B, 0.1, np.float32)), d(rs.random(B).astype(np.float32))
        self.tok, self.status = gpu.DeviceArray.zeros(B, np.int32), gpu.DeviceArray.zeros(B, np.int32)
        kv, lib = self.kv(0), gpu.lib
        self.wa = workspace(gpu, lib.mlxr_k_paged_attention_work(ctypes.byref(kv), nH))
        self.we = workspace(gpu, lib.mlxr_k_paged_evict_work(ctypes.byref(kv), budget))
        self.ws = workspace(gpu, lib.mlxr_k_sample_rows_work(B, nH * D))

    def kv(self, i):
        return self.gpu.PagedKV(k=self.k.ptr, v=self.v.ptr, table=self.table[i].ptr, len=self.len[i].ptr, weight=self.weight[i].ptr,
                                position=self.position[i].ptr, n_pages=self.k.shape[0], table_stride=self.top // PAGE, slot_stride=self.top,
                                max_len=self.top, B=self.B, nKV=self.nKV, D=self.D, st=0)

    def new_inputs(self, seed, i, more=1):
        rs = np.random.default_rng(seed)
        self.len[i].upload(self.len[i].numpy() + more)
        self.pos.upload(self.pos.numpy() + 1)
        self.qkv.upload(rs.standard_normal(self.qkv.shape).astype(np.float32))
        self.u.upload(rs.random(self.B).astype(np.float32))

    def run(self, i, evict=False, s=None):
        gpu, lib, kv, n = self.gpu, self.gpu.lib, self.kv(i), self.nH * self.D
        gpu.check(lib.mlxr_k_paged_append(ctypes.byref(kv), self.qkv.ptr, self.qkv.shape[1], self.inv.ptr, None, None, self.nH, self.D, 0, self.pos.ptr, 1e-6,
                                          self.q.ptr, n, s))
        gpu.check(lib.mlxr_k_paged_attention(ctypes.byref(kv), self.q.ptr, n, self.nH, 0, self.D ** -0.5, self.out.ptr, n, self.weight[i].ptr, 1.0,
                                             self.wa.ptr, self.wa.nbytes, s))
        gpu.check(lib.mlxr_k_sample_rows(self.out.ptr, self.B, n, n, self.t.ptr, None, None, None, self.u.ptr, self.tok.ptr, self.status.ptr, self.ws.ptr,
                                         self.ws.nbytes, s))
        if evict:
            to = self.kv(1 - i)
            gpu.check(lib.mlxr_k_paged_evict(ctypes.byref(kv), ctypes.byref(to), self.budget, 4, 16, self.we.ptr, self.we.nbytes, s))

    def state(self):
        return [x.numpy() for x in (self.k, self.v, *self.len, *self.weight, *self.position, self.q, self.out, self.tok, self.status)]

    def plain(self, i):
        """The step's attention output and weights from the state before it, in 64 bits (the new key and value rounded to bf16)."""
        lens, k, v = self.len[i].numpy(), bf16_to_f32(self.k.numpy()).astype(np.float64), bf16_to_f32(self.v.numpy()).astype(np.float64)
        w, x, pos, G = self.weight[i].numpy().astype(np.float64), self.qkv.numpy().astype(np.float64).reshape(self.B, -1, self.D), self.pos.numpy(), self.nH // self.nKV
        out = np.zeros((self.B, self.nH, self.D))
        for b, L in enumerate(lens):
            z = (x[b, :, :64] + 1j * x[b, :, 64:]) * np.exp(1j * pos[b] * self.inv_freq.astype(np.float64))
            rot = np.concatenate([z.real, z.imag], 1)
            w[b, :, L - 1] = 0
            j = np.arange(L)
            for h in range(self.nKV):
                kk, vv = (t[self.tables[i][b, j // PAGE], h, j % PAGE].copy() for t in (k, v))
                kk[-1], vv[-1] = bf16_to_f32(bf16_round(rot[self.nH + h])), bf16_to_f32(bf16_round(x[b, self.nH + self.nKV + h]))
                for g in range(h * G, h * G + G):
                    e = kk @ rot[g] * float(np.float32(self.D ** -0.5))
                    p = np.exp(e - e.max())
                    p /= p.sum()
                    out[b, g] = p @ vv
                    w[b, h, :L] += p
        return out.reshape(self.B, -1), w


def test_steps_together(gpu):
    """Ten steps of a batch, evicted twice into other pages: every step's output, weights and tokens are the formulas'."""
    s, i = Step(gpu), 0
    for n in range(10):
        s.new_inputs(100 + n, i)
        want, weight = s.plain(i)
        full = n in (3, 7)
        s.run(i, evict=full)
        gpu.synchronize()
        # a value of the new key may lie so near the middle of two bf16 numbers that it is rounded the other way: 2^-7 of it at
        # most, in few of the 128 terms of one score, so p of that key by some hundredths; nothing else is off by more than fp32
        lens, got, got_w = s.len[i].numpy(), s.out.numpy(), s.weight[i].numpy()
        assert np.abs(got - want).max() < 0.02 and np.abs(got - want).mean() < 1e-4
        for b, L in enumerate(lens):
            assert np.abs(got_w[b, :, :L] - weight[b, :, :L]).max() < 0.02
            assert int(s.tok.numpy()[b]) in reference_token(got[b], 0.1, None, None, None, s.u.numpy()[b])[0]
        if full:
            i = 1 - i
            assert same(s.len[i].numpy(), np.minimum(lens, 96).astype(np.int32))
            for b, L in enumerate(s.len[i].numpy()):   # the newest key is the last slot
                assert (s.position[i].numpy()[b, :, L - 1] == s.pos.numpy()[b]).all()


def test_step_captured(gpu):
    """The step in a HIP graph: replays with new inputs, eager work and synchronizations between them, give the eager
    step's bits."""
    hip = Hip(gpu)
    a, b, st = Step(gpu, seed=5), Step(gpu, seed=5), hip.stream()
    for s in (a, b):
        s.run(0, evict=True, s=st)
    hip.wait(st)
    graph = hip.capture(st, lambda: b.run(0, evict=True, s=st))
    for n in range(6):
        for s in (a, b):
            s.new_inputs(n, 0, more=1 if n < 4 else -3)
        a.run(0, evict=True, s=st)
        if n % 2:
            hip.wait(st)
        hip("hipGraphLaunch", graph, st)
        hip.wait(st)
        for x, y in zip(a.state(), b.state()):
            assert same(x, y), n
    hip("hipGraphExecDestroy", graph)
    hip("hipStreamDestroy", st)


def test_eviction_of_long_sequences_captured(gpu):
    """Lengths for which a launch asks for more LDS than it has by itself, in a HIP graph: every replay is the eager result."""
    hip = Hip(gpu)
    src, dst = pair(gpu, [20000, 31000, 40000], 1, 64, 0, 3000, seed=61)
    src.up(), dst.up()
    st, a = hip.stream(), src.desc()
    b = dst.desc(k=src.dk.ptr, v=src.dv.ptr, n_pages=src.k.shape[0])
    work = workspace(gpu, gpu.lib.mlxr_k_paged_evict_work(ctypes.byref(a), 3000))
    run = lambda: gpu.check(gpu.lib.mlxr_k_paged_evict(ctypes.byref(a), ctypes.byref(b), 3000, 4, 512, work.ptr, work.nbytes, st))  # noqa: E731
    graph = hip.capture(st, run)
    for n in range(3):
        src.weight = np.random.default_rng(62 + n).exponential(1.0, src.weight.shape).astype(np.float32)
        src.dw.upload(src.weight)
        hip("hipGraphLaunch", graph, st)
        hip.wait(st)
        check_evicted(src, dst, 3000, 4, 512, src.k.copy(), src.v.copy(), dst.weight, dst.position)
    hip("hipGraphExecDestroy", graph)
    hip("hipStreamDestroy", st)


def test_two_streams_at_once(gpu):
    """Two steps on two streams, each with its own workspaces, give what they give alone."""
    hip, alone = Hip(gpu), []
    for seed in (1, 2):
        s = Step(gpu, seed=seed)
        for _ in range(4):
            s.run(0, evict=True)
        gpu.synchronize()
        alone.append(s.state())
    both, streams = [Step(gpu, seed=seed) for seed in (1, 2)], [hip.stream(), hip.stream()]
    gpu.synchronize()
    for _ in range(4):
        for s, st in zip(both, streams):
            s.run(0, evict=True, s=st)
    for st in streams:
        hip.wait(st)
    for s, want in zip(both, alone):
        for x, y in zip(s.state(), want):
            assert same(x, y)
    for st in streams:
        hip("hipStreamDestroy", st)


def test_host_memory_is_refused(gpu):
    c = Cache(gpu, [64], 1, 128, 0).up()
    host = np.zeros(1 << 14, np.float32)
    kv = c.desc(k=(host.ctypes.data + 63) & ~63)
    q, work = gpu.DeviceArray.zeros(128, np.float32), gpu.DeviceArray.zeros(1 << 20, np.uint8)
    rc = gpu.lib.mlxr_k_paged_attention(ctypes.byref(kv), q.ptr, 128, 1, 0, 0.1, q.ptr, 128, None, 1.0, work.ptr, work.nbytes, None)
    assert rc == -10
