"""The batch's decode step at its edges: infinities and NaN in cache and queries, appends to pages outside the pool,
the order of NaN weights, draws next to a border, host memory in place of the device's. Helpers and tolerances are those of test_batch_gpu."""
import ctypes

import numpy as np
import pytest

from test_batch_gpu import (PAGE, Cache, Hip, attend, attention_reference, check_out, evict, model_logits, pair, queries, run_append, same, sample,
                            to_half, within)

pytestmark = pytest.mark.gpu
INF = np.float32(np.inf)
EIGHTH = next(x for x in (np.float32(0.125 / np.log2(np.e)) + np.float32(i * 2.0 ** -28) for i in range(-9, 9))
              if np.float32(x * np.float32(np.log2(np.e))) == 0.125)   # a scale that is 2^-3 in powers of two: no bits of its own


class Without:
    """A cache seen without some of its slots: `gone` [B][nKV][slot] take no part."""

    def __init__(self, c, gone):
        self.c, self.gone = c, gone

    def __getattr__(self, name):
        return getattr(self.c, name)

    def rows(self, pool, b, h, n):
        x, there = self.c.rows(pool, b, h, n)
        there = there & ~self.gone[b, h, :n]
        return np.where(there[:, None], x, 0), there


def put(c, pool, b, h, j, dims, value):
    pool[c.table[b, j // PAGE], h, j % PAGE, dims] = to_half(np.full(1, value, np.float32), c.st)[0]


def plain_weights(c, given, p, p_tol, G):
    want = given[:, :, :c.max_len] + p
    return want, p_tol + 2.0 ** -23 * (np.abs(given[:, :, :c.max_len]) + np.abs(want)) + (G + 2) * 2.0 ** -24 * p


# ------------------------------------------------------------------------------------------- infinities and NaN
@pytest.mark.parametrize("D,st", [(128, 0), (64, 0), (128, 1), (64, 1)])
@pytest.mark.parametrize("nKV,G,window", [(2, 4, 0), (1, 17, 0), (2, 1, 150)])
@pytest.mark.parametrize("exact", [True, False])
def test_attention_infinite_keys(gpu, D, st, nKV, G, window, exact):
    """Keys with infinite elements whose scores are -infinity take no part, whatever parts a query is split into: queries of
    few bits (parts of zero) and of many."""
    print(f"[case] {D} {st} {nKV} {G} {window} {exact}", flush=True)
    nH = nKV * G
    c = Cache(gpu, [1, 65, 700, 0, 2600, 64], nKV, D, st, seed=71, weight=True)
    q = queries(c, nH)
    heads = q[:, :nH * D].reshape(c.B, nH, D)
    heads[:, :, 3], heads[:, :, 5] = np.abs(heads[:, :, 3]) + 1, -np.abs(heads[:, :, 5]) - 1
    if exact:
        heads[:] = few_bits(heads)
    gone = np.zeros((c.B, nKV, c.max_len), bool)
    rs = np.random.default_rng(72)
    for b, L in enumerate(c.lens):
        for h in range(nKV):
            for j in rs.choice(L, min(L, 9), replace=False) if b != 5 else range(64):
                gone[b, h, j] = True
                put(c, c.k, b, h, j, 3, -INF)
                if j % 2:
                    put(c, c.k, b, h, j, 5, INF)
                if j % 3 == 0:
                    put(c, c.v, b, h, j, slice(None), INF if j % 2 else np.nan)   # of no account
    given = c.weight.copy()
    c.up()
    scale = float(EIGHTH) if exact else 0.09
    out, tol, p, p_tol = attention_reference(Without(c, gone), q, nH, window, scale)
    assert not out[[0, 3, 5]].any()
    check_out(attend(gpu, c, q, nH, window=window, scale=scale, weight_in=c.dw), c, nH, out, tol)
    want, w_tol = plain_weights(c, given.astype(np.float64), p, p_tol, G)
    got = c.dw.numpy()
    for b, L in enumerate(c.lens):
        assert within(np.abs(got[b, :, :L] - want[b, :, :L]), w_tol[b, :, :L]) <= 1
        assert same(got[b, :, L:], given[b, :, L:])


def few_bits(x):
    """A value of at most eight bits, which both cache types hold exactly."""
    return np.round(x * 16).astype(np.float32) / 16


@pytest.mark.parametrize("D,st", [(128, 0), (64, 1)])
@pytest.mark.parametrize("weight", [False, True])
def test_attention_infinite_values(gpu, D, st, weight):
    """An infinite value of a key that takes part gives that infinity, however small the key's share is, and two of
    different signs NaN; all other dims are as without."""
    c = Cache(gpu, [300, 64, 3000, 40, 129], 2, D, st, seed=73, weight=weight)
    q = queries(c, 8)
    plain = attention_reference(c, q, 8, 0, 0.09)
    put(c, c.v, 0, 0, 299, 7, INF)
    put(c, c.v, 1, 1, 0, 0, -INF)
    for j in (5, 1500, 2999):
        put(c, c.v, 2, 0, j, D - 1, INF)
    put(c, c.v, 2, 1, 10, 2, INF)
    put(c, c.v, 2, 1, 2900, 2, -INF)
    put(c, c.v, 3, 1, 39, slice(None), -INF)
    out, tol = (x.reshape(c.B, 8, D).copy() for x in plain[:2])
    for b, h, d, x in [(0, 0, 7, INF), (1, 1, 0, -INF), (2, 0, D - 1, INF), (2, 1, 2, np.nan), (3, 1, slice(None), -INF)]:
        out[b, 4 * h:4 * h + 4, d] = x
    c.up()
    given = c.weight.copy() if weight else None
    got = attend(gpu, c, q, 8, weight_in=c.dw)[:, :8 * D].reshape(c.B, 8, D)
    odd = ~np.isfinite(out)
    assert np.array_equal(got[odd], out[odd].astype(np.float32), equal_nan=True)
    assert within(np.abs(got[~odd] - out[~odd]), tol[~odd]) <= 1
    if weight:
        want, w_tol = plain_weights(c, given.astype(np.float64), plain[2], plain[3], 4)
        for b, L in enumerate(c.lens):
            assert within(np.abs(c.dw.numpy()[b, :, :L] - want[b, :, :L]), w_tol[b, :, :L]) <= 1


@pytest.mark.parametrize("st", [0, 1])
def test_attention_infinite_value_of_a_tiny_share(gpu, st):
    """Shares below what 32 bits hold (e^-200) are not nothing: an infinite value there is the result, in keys before and
    behind the heaviest one, in its run and in others."""
    c = Cache(gpu, [2000] * 5, 1, 128, st, seed=74)
    q = queries(c, 2)
    q[:, :256] = 0
    q[:, [0, 128]] = 20.0
    for b in range(5):
        for i in range(0, 2000, PAGE):
            c.k[c.table[b, i // PAGE], 0, :, 0] = to_half(np.float32(-10.0), st)
        put(c, c.k, b, 0, 1000, 0, 10.0)                      # scores 200 and -200 at a scale of 1
    for b, j in enumerate([999, 1001, 0, 1999]):
        put(c, c.v, b, 0, j, 9, INF)
    c.up()
    got = attend(gpu, c, q, 2, scale=1.0)[:, :256].reshape(5, 2, 128)
    assert (got[:4, :, 9] == INF).all()
    keep = np.arange(128) != 9
    for b in range(5):
        v = c.rows(c.v, b, 0, 2000)[0][1000]
        assert np.abs(got[b][:, keep] - v[keep]).max() <= 2.0 ** -22 * np.abs(v).max()   # one p of 1: products and a quotient
    assert np.isfinite(got[4]).all()


@pytest.mark.parametrize("st", [0, 1])
@pytest.mark.parametrize("length", [1, 64, 5000])
def test_attention_nan(gpu, st, length):
    """A NaN in a query or in a key that takes part is NaN in that row's result (and only there), in one run or many."""
    c = Cache(gpu, [length, length, length, 700], 2, 128, st, seed=75)
    q = queries(c, 8)
    q[0, 128 * 2 + 5] = np.nan             # head 2 of sequence 0
    clean = q.copy()
    clean[0, 128 * 2 + 5] = 0
    put(c, c.k, 1, 1, length - 1, 77, 0)
    out, tol = (x.reshape(4, 8, 128) for x in attention_reference(c, clean, 8, 0, 0.09)[:2])
    put(c, c.k, 1, 1, length - 1, 77, np.nan)
    c.up()
    got = attend(gpu, c, q, 8)[:, :1024].reshape(4, 8, 128)
    nan = np.zeros((4, 8), bool)
    nan[0, 2] = nan[1, 4:] = True
    assert np.isnan(got[nan]).all()
    assert within(np.abs(got[~nan] - out[~nan]), tol[~nan]) <= 1


@pytest.mark.parametrize("st", [0, 1])
@pytest.mark.parametrize("length", [1, 100, 5000])
def test_attention_infinite_queries(gpu, st, length):
    """A query's infinity against keys of the other sign scores -infinity at every one: zeros, and no weight. Against keys of
    both signs the row is NaN, as the formula is; the other rows are as they were."""
    c = Cache(gpu, [length, length, 70], 1, 64, st, seed=78, weight=True)
    q = queries(c, 3)
    for b in range(2):
        for i in range(0, length, PAGE):
            page = c.table[b, i // PAGE]
            n = min(PAGE, length - i)
            c.k[page, 0, :n, 11] = to_half(-1 - np.arange(n, dtype=np.float32), st)
    q2 = q.copy()
    q2[0, 64 + 11] = INF                                       # head 1 of sequence 0: all scores -infinity
    q2[1, 128 + 11] = -INF                                     # head 2 of sequence 1: all +infinity
    clean = q2.copy()
    clean[~np.isfinite(q2) & ~np.isnan(q2)] = 0
    out, tol, p, p_tol = attention_reference(c, clean, 3, 0, 0.09)
    c.up()
    given = c.weight.copy()
    got = attend(gpu, c, q2, 3, weight_in=c.dw)[:, :192].reshape(3, 3, 64)
    out, tol = out.reshape(3, 3, 64), tol.reshape(3, 3, 64)
    assert not got[0, 1].any() and np.isnan(got[1, 2]).all()
    rest = np.ones((3, 3), bool)
    rest[0, 1] = rest[1, 2] = False
    assert within(np.abs(got[rest] - out[rest]), tol[rest]) <= 1
    w = c.dw.numpy()
    assert np.isnan(w[1, 0, :length]).all()
    # sequence 0: heads 0 and 2 only
    kk = c.rows(c.k, 0, 0, length)[0]
    want = given[0, 0, :length].astype(np.float64)
    for h in (0, 2):
        s = float(np.float32(0.09)) * (kk @ q2[0, 64 * h:64 * h + 64].astype(np.float64))
        e = np.exp(s - s.max())
        want += e / e.sum()
    assert within(np.abs(w[0, 0, :length] - want), p_tol[0, 0, :length] + 2.0 ** -22 * want) <= 1


@pytest.mark.parametrize("st", [0, 1])
def test_attention_infinite_keys_in_long_runs(gpu, st):
    """More pages a run than a wave holds numbers of at once, some of them with a key that takes no part: 17003 pages, of 40
    in turn."""
    n, L, D = 40, 64 * 17003 - 5, 64
    c = Cache(gpu, [64 * n], 1, D, st, seed=79)
    table = np.resize(c.table[0, :n], 17003).astype(np.int32)
    q = queries(c, 2)
    q[0, [3, 64 + 3]] = 0.5
    for page in (2, 17, 39):
        put(c, c.k, 0, 0, 64 * page + 20, 3, -INF)
    gone = np.zeros(64 * n, bool)
    gone[[64 * 2 + 20, 64 * 17 + 20, 64 * 39 + 20]] = True
    c.up()
    dt, dl = gpu.DeviceArray.from_numpy(table.reshape(1, -1)), gpu.DeviceArray.from_numpy(np.array([L], np.int32))
    kv = c.desc(table=dt.ptr, len=dl.ptr, table_stride=17003, max_len=64 * 17003)
    got = attend(gpu, c, q, 2, desc=kv)[0, :2 * D].reshape(2, D)
    (k, _), (v, _) = c.rows(c.k, 0, 0, 64 * n), c.rows(c.v, 0, 0, 64 * n)
    times = np.bincount(np.arange(L) % (64 * n), minlength=64 * n)[~gone]
    k, v = k[~gone], v[~gone]
    U = 2.0 ** -24
    for h in range(2):
        x = q[0, h * D:(h + 1) * D].astype(np.float64)
        s = float(np.float32(0.09)) * (k @ x)
        p = np.exp(s - s.max())
        p /= (times * p).sum()
        # the terms of attention_reference's bound, each slot's share counted as often as it is there
        ds = 4 * np.sqrt(D) * U * 0.09 * np.sqrt((k ** 2) @ (x ** 2)) + 4 * U * np.abs(s) + 2 * U * np.abs(s).max()
        want, rel = (times * p) @ v, 2 * ds.max() + 8 * U
        tol = rel * ((times * p) @ np.abs(v)) + 4 * np.sqrt(L) * U * np.sqrt((times * p ** 2) @ (v ** 2)) + np.abs(want) * (4 * np.sqrt(L) * U * np.sqrt((times * p ** 2).sum()) + 2 * U)
        assert within(np.abs(got[h] - want), tol) <= 1


def test_append_past_f16_and_attention(gpu):
    """What passes f16's largest number is infinite in its cache: a key that scores -infinity then takes no part."""
    c = Cache(gpu, [200, 65], 1, 64, 1, seed=76, weight=True).up()
    qkv = np.random.default_rng(77).standard_normal((2, 4 * 64)).astype(np.float32)
    qkv[:, 128] = -1e5
    qkv[:, [0, 64]] = [0.75, 1.5]          # both query heads: positive, of few bits
    q, _ = run_append(gpu, c, qkv, 2, np.zeros(0, np.float32), None, None, 0, 0, None, 1e-6, False, q_pad=0)
    c.k, c.v = c.dk.numpy(), c.dv.numpy()
    gone = np.zeros((2, 1, c.max_len), bool)
    gone[0, 0, 199] = gone[1, 0, 64] = True
    out, tol, _, _ = attention_reference(Without(c, gone), q, 2, 0, float(EIGHTH))
    got = attend(gpu, c, q, 2, scale=float(EIGHTH))
    assert within(np.abs(got - out), tol) <= 1
    assert c.dw.numpy()[0, 0, 199] == 0 and c.dw.numpy()[1, 0, 64] == 0


# ------------------------------------------------------------------------------------------- append
def test_append_bad_pages_leave_everything(gpu):
    """An append to a page outside the pool writes nothing: no key, no value, no weight and no position."""
    c = Cache(gpu, [65, 64, 3], 2, 128, 0, seed=9, weight=True, position=True)
    c.table[0, 1], c.table[1, 0] = c.k.shape[0], -7
    c.up()
    qkv = np.random.default_rng(1).standard_normal((3, 6 * 128)).astype(np.float32)
    q, _ = run_append(gpu, c, qkv, 2, np.zeros(0, np.float32), None, None, 0, 0, None, 1e-6, False)
    assert same(q[:, :256], qkv[:, :256])
    w, p = c.weight.copy(), c.position.copy()
    w[2, :, 2], p[2, :, 2] = 0, 2
    assert same(c.dw.numpy(), w) and same(c.dp.numpy(), p)


# ------------------------------------------------------------------------------------------- eviction
def heaviest(w, n, budget, sink, window):
    """The kept slots: NaN below -infinity, equal ones by slot."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sink, n - window)
    nan = np.isnan(w[mid])
    mid = mid[np.lexsort((mid, -np.where(nan, 0, w[mid]).astype(np.float64), nan))][:budget - sink - window]
    return np.sort(np.concatenate([np.arange(sink), mid, np.arange(n - window, n)])).astype(int)


@pytest.mark.parametrize("budget,sink,window", [(100, 4, 32), (64, 0, 0), (260, 1, 9)])
def test_evict_nan_and_minus_infinity(gpu, budget, sink, window):
    """Cuts that fall among NaN weights (the lower slot stays), among those of -infinity, and between the two."""
    lens = [500, 500, 500, 300]
    src, dst = pair(gpu, lens, 2, 64, 0, budget, seed=81)
    room = budget - sink - window
    rs = np.random.default_rng(82)
    src.weight[0] = np.nan                                              # nothing else
    src.weight[1] = np.where(rs.random(src.weight[1].shape) < 0.5, np.nan, -INF)
    for h in range(2):                                                  # so many numbers above -infinity and NaN
        for b, above in ((2, room // 2), (3, 0)):
            n = lens[b]
            w = np.full(src.stride, np.nan, np.float32)
            order = rs.permutation(np.arange(sink, n - window))
            w[order[:above]] = rs.standard_normal(above)
            w[order[above:room]] = -INF                                 # the cut lies between these and NaN
            if h:
                w[order[above + 1:above + 2]] = np.nan                  # one too few: a NaN stays
            src.weight[b, h] = w
    src.up(), dst.up()
    k0 = src.k.copy()
    evict(gpu, src, dst, budget, sink, window)
    pos = dst.dp.numpy()
    for b, n in enumerate(lens):
        for h in range(2):
            kept = heaviest(src.weight[b, h, :n], n, budget, sink, window)
            assert same(pos[b, h, :len(kept)], src.position[b, h, kept]), (b, h)
            j = np.arange(len(kept))
            assert same(src.dk.numpy()[dst.table[b, j // PAGE], h, j % PAGE], k0[src.table[b, kept // PAGE], h, kept % PAGE])


# ------------------------------------------------------------------------------------------- sampling
STEP = 2.0 ** -43   # what a weight may be off by, of itself; the largest logit's is exact


def tokens_next_to(v, t, k, p, low, u):
    """The tokens that may come where every sum may be off by 2^-42 of itself (twice what the weights in it are)."""
    v = np.asarray(v, np.float64)
    idx = np.nonzero(~np.isnan(v) & (v != -np.inf))[0]
    order = idx[np.lexsort((idx, -v[idx]))]
    if not t > 0.001:
        return {int(order[0])}
    if k is not None and k > 0:
        order = order[:k]
    w = np.exp((v[order] - v[order[0]]) / float(np.float32(t))) if np.isfinite(t) else np.ones(len(order))
    run = np.cumsum(w.astype(np.longdouble))
    ends = {len(w)}
    if p is not None and p < 1:
        goal = np.longdouble(float(np.float32(p))) * run[-1]
        ends = {max(1, min(len(w), int(np.searchsorted(run, goal * (1 + e))) + 1)) for e in (-2 * STEP, 0, 2 * STEP)}
    if low is not None and low > 0:
        ends = {max(1, min(e, int((w >= float(np.float32(low)) * (1 + d)).sum()))) for e in ends for d in (-2 * STEP, 0, 2 * STEP)}
    may = set()
    for e in ends:
        goal = np.longdouble(float(np.float32(u))) * run[e - 1]
        first, last = (min(e - 1, int(np.searchsorted(run[:e], goal * (1 + d)))) for d in (-2 * STEP, 2 * STEP))
        may.update(int(i) for i in order[first:last + 1])
    return may


def check_near(gpu, x, t, k=None, p=None, low=None, u=None):
    tok, st = sample(gpu, x, t, k, p, low, u)
    at = lambda y, r: None if y is None else (y[r] if np.ndim(y) else y)  # noqa: E731
    doubtful = 0
    for r in range(x.shape[0]):
        may = tokens_next_to(x[r], at(t, r), at(k, r), at(p, r), at(low, r), at(u, r))
        assert int(tok[r]) in may, (r, int(tok[r]), sorted(may)[:9], t, k, p, low, at(u, r))
        doubtful += len(may) > 1
    assert not st.any()
    return doubtful


@pytest.mark.parametrize("V,t,far,k", [
    (151936, 1.0, -33.0, None), (151936, 0.5, -17.5, None), (1 << 20, 1.0, -34.0, None), (151936, 1.0, -40.0, None),
    (151936, 0.1, -3.5, None), (1 << 20, 3.0, -110.0, None), (1 << 20, 8.0, -280.0, None), (2000, 1.0, -33.0, None), (2000, 0.7, -23.0, 1500),
    (151936, 1.0, -33.0, 2000), (151936, 1.0, -33.0, 100000), (151936, 1.0, -36.0, 100000), (30000, 0.25, -8.25, 400)])
def test_sample_tail_counts(gpu, V, t, far, k):
    """Two equal logits above a tail that weighs less than 2^-24 in all: half of the sum is more than the first's weight,
    so a draw at 0.5 takes the second one. (The two weights are exact, and the tail's share is hundreds of steps of a
    64-bit sum at least.)"""
    print(f"[case] {V} {t} {far} {k}", flush=True)
    tail = (min(k or V, V) - 2) * np.exp(far / float(np.float32(t)))
    assert 2.0 ** -44 < tail < 2.0 ** -25
    x = np.full((2, V), np.float32(far))
    x[0, [7, V - 3]] = 0.0
    x[1] = np.float32(far) - np.random.default_rng(V).random(V).astype(np.float32) * np.float32(0.5 * t)   # no two alike, most of them
    x[1, [V // 2, V // 2 + 1]] = 0.0
    assert list(sample(gpu, x, t, k, u=0.5)[0]) == [V - 3, V // 2 + 1]


def test_sample_kept_tail_of_few_ranks(gpu):
    """The same with 48 ranks of about e^-33 behind the two: their share, 2^-42, is more than a 64-bit sum's steps."""
    V = 151936
    for t, scale in ((1.0, 1.0), (0.1, 0.1), (0.02, 0.02)):
        x = np.full((1, V), -2000.0, np.float32)
        x[0, 100:148] = -np.float32(33 * scale) - np.arange(48, dtype=np.float32) * np.float32(0.01 * scale)
        x[0, [5, 90000]] = 0.0
        for k in (50, 40, 3, None):
            assert list(sample(gpu, x, t, k, u=0.5)[0]) == [90000], (t, k)
        assert list(sample(gpu, x, t, 2, u=0.5)[0]) == [5]


@pytest.mark.parametrize("V", [4097, 151936, 1 << 20])
def test_sample_next_to_a_border(gpu, V):
    """Tokens against sums that may be off by 2^-42 of themselves only, at temperatures from 0.02 to 20."""
    print(f"[case] V={V}", flush=True)
    rs = np.random.default_rng(V + 1)
    x = model_logits(rs, 4, V)
    x[3] = np.round(x[3] * 4) / 4                     # thousands of equal ones
    doubtful = 0
    for t in (0.02, 0.1, 0.3, 0.7, 1.0, 1.9, 6.0, 20.0):
        u = rs.random(4).astype(np.float32)
        for k, p, low in [(40, 0.95, None), (None, None, None), (None, 0.9, None), (3000, None, None), (None, 0.999, 1e-6), (None, None, 1e-9)]:
            doubtful += check_near(gpu, x, t, k, p, low, u)
    assert doubtful <= 2


def test_sample_ties_of_little_weight(gpu):
    """Half a million equal logits of 1e-9 of the largest's weight each and as many of 7e-10: the draw next to 1 falls among
    the last 100 of them, on a token that the sums to 2^-42 decide."""
    V = 1 << 20
    x = np.full((2, V), np.float32(-20.7))
    x[:, ::2] = np.float32(-21.1)
    x[0, 12345] = 0.0
    x[1, [3, 777, 5000]] = 0.0
    assert check_near(gpu, x, 1.0, u=1 - 2.0 ** -24) == 0
    for u in (0.9996, 0.99925):                       # among the others: their weights' own error would count thousandfold
        assert check_near(gpu, x, 1.0, u=u) == 0
    assert check_near(gpu, x * np.float32(2), 2.0, k=1000000, u=1 - 2.0 ** -24) == 0
    assert check_near(gpu, x, 1.0, p=1 - 2.0 ** -23, u=1 - 2.0 ** -22) == 0


# ------------------------------------------------------------------------------------------- memory
class Calls:
    """The four calls over device memory, any one of whose pointers can be given another address."""

    def __init__(self, gpu):
        d = lambda x: gpu.DeviceArray.from_numpy(np.ascontiguousarray(x))  # noqa: E731
        rs = np.random.default_rng(91)
        pool, floats, table = rs.standard_normal((8, 2, PAGE, 128)), rs.random((2, 2, 128)).astype(np.float32), np.arange(8, dtype=np.int32).reshape(4, 2)
        a = dict(k=d(to_half(pool, 0)), v=d(to_half(pool, 0)), table=d(table[:2]), len=d(np.array([70, 128], np.int32)), weight=d(floats),
                 position=d(np.zeros((2, 2, 128), np.int32)))
        b = dict(a, table=d(table[2:]), len=d(np.zeros(2, np.int32)), weight=d(floats), position=d(np.zeros((2, 2, 128), np.int32)))
        x = dict(qkv=d(rs.standard_normal((2, 1024)).astype(np.float32)), inv=d(np.ones(64, np.float32)), qn=d(np.ones(128, np.float32)),
                 kn=d(np.ones(128, np.float32)), pos=d(np.array([69, 127], np.int32)), q=gpu.DeviceArray.zeros((2, 512), np.float32),
                 out=gpu.DeviceArray.zeros((2, 512), np.float32), work=gpu.DeviceArray.zeros(1 << 22, np.uint8))
        y = dict(logits=d(model_logits(rs, 3, 5000)), t=d(np.full(3, 0.8, np.float32)), k=d(np.full(3, 50, np.int32)), p=d(np.full(3, 0.9, np.float32)),
                 low=d(np.zeros(3, np.float32)), u=d(np.array([0.2, 0.5, 0.9], np.float32)), tokens=gpu.DeviceArray.zeros(3, np.int32),
                 status=gpu.DeviceArray.zeros(3, np.int32), work=gpu.DeviceArray.zeros(1 << 22, np.uint8))
        self.gpu, self.src, self.dst, self.x, self.y = gpu, a, b, x, y

    def cache(self, arrays, over):
        n = {k: over.get(k, v.ptr) for k, v in arrays.items()}
        return self.gpu.PagedKV(n_pages=8, table_stride=2, slot_stride=128, max_len=128, B=2, nKV=2, D=128, st=0, **n)

    def append(self, s=None, **over):
        o, kv = {k: over.get(k, v.ptr) for k, v in self.x.items()}, self.cache(self.src, over)
        return self.gpu.lib.mlxr_k_paged_append(ctypes.byref(kv), o["qkv"], 1024, o["inv"], o["qn"], o["kn"], 4, 128, 0, o["pos"], 1e-6, o["q"], 512, s)

    def attention(self, s=None, **over):
        o, kv = {k: over.get(k, v.ptr) for k, v in self.x.items()}, self.cache(self.src, over)
        return self.gpu.lib.mlxr_k_paged_attention(ctypes.byref(kv), o["q"], 512, 4, 0, 0.1, o["out"], 512, over.get("weight_in", kv.weight), 1.0, o["work"],
                                                   1 << 22, s)

    def evict(self, s=None, **over):
        to = {k[3:]: v for k, v in over.items() if k.startswith("to_")}
        a, b = self.cache(self.src, over), self.cache(self.dst, to)
        return self.gpu.lib.mlxr_k_paged_evict(ctypes.byref(a), ctypes.byref(b), 64, 4, 16, over.get("work", self.x["work"].ptr), 1 << 22, s)

    def sample(self, s=None, **over):
        o = {k: over.get(k, v.ptr) for k, v in self.y.items()}
        return self.gpu.lib.mlxr_k_sample_rows(o["logits"], 3, 5000, 5000, o["t"], o["k"], o["p"], o["low"], o["u"], o["tokens"], o["status"], o["work"], 1 << 22, s)


CACHE = ["k", "v", "table", "len", "weight", "position"]


@pytest.mark.parametrize("call,names", [
    ("append", CACHE + ["qkv", "inv", "qn", "kn", "pos", "q"]), ("attention", CACHE[:5] + ["q", "out", "weight_in", "work"]),
    ("evict", CACHE + ["to_" + x for x in CACHE] + ["work"]), ("sample", ["logits", "t", "k", "p", "low", "u", "tokens", "status", "work"])])
def test_host_memory_is_refused_everywhere(gpu, call, names):
    """Pageable host memory as any one of a call's pointers: refused, and nothing is launched."""
    c, host = Calls(gpu), np.zeros(1 << 20, np.uint8)
    at = (host.ctypes.data + 255) & ~255
    for name in names:
        print(f"[case] {call} {name}", flush=True)
        assert getattr(c, call)(**{name: at}) == -10, name
    assert not host.any()
    assert getattr(c, call)() == 0
    gpu.synchronize()


def test_pinned_memory_is_taken(gpu):
    """Random numbers in pinned host memory give the tokens that they give on the device."""
    c, hip = Calls(gpu), Hip(gpu)
    gpu.check(c.sample())
    gpu.synchronize()
    want = c.y["tokens"].numpy()
    p = ctypes.c_void_p()
    hip("hipHostMalloc", ctypes.byref(p), ctypes.c_size_t(4096), 0)
    u = c.y["u"].numpy()
    ctypes.memmove(p, u.ctypes.data, u.nbytes)
    c.y["tokens"].upload(np.full(3, -1, np.int32))
    gpu.check(c.sample(u=p.value))
    gpu.synchronize()
    assert same(c.y["tokens"].numpy(), want)
    hip("hipHostFree", p)


def test_calls_captured_in_the_strictest_mode(gpu):
    """Nothing that the calls ask of the runtime is forbidden in a capture of mode 'global'."""
    c, hip = Calls(gpu), Hip(gpu)
    s, graph, ex = hip.stream(), ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", s, 0)
    rc = [getattr(c, n)(s=s) for n in ("append", "attention", "evict", "sample")]
    hip("hipStreamEndCapture", s, ctypes.byref(graph))
    assert rc == [0, 0, 0, 0]
    hip("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
    for _ in range(3):
        hip("hipGraphLaunch", ex, s)
        hip.wait(s)
    out, tokens = c.x["out"].numpy(), c.y["tokens"].numpy()
    e = Calls(gpu)
    for n in ("append", "attention", "evict", "sample"):
        gpu.check(getattr(e, n)())
    gpu.synchronize()
    assert same(out, e.x["out"].numpy()) and same(tokens, e.y["tokens"].numpy())
    hip("hipGraphExecDestroy", ex)
    hip("hipStreamDestroy", s)
