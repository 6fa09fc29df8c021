"""The batch's decode step at its edges: NaN in cache and queries, appends to pages outside the pool. Helpers and
tolerances are those of test_batch_gpu."""
import numpy as np
import pytest

from test_batch_gpu import PAGE, Cache, attend, attention_reference, queries, run_append, same, to_half, within

pytestmark = pytest.mark.gpu


def put(c, pool, b, h, j, dims, value):
    pool[c.table[b, j // PAGE], h, j % PAGE, dims] = to_half(np.float32(value), c.st)


# ------------------------------------------------------------------------------------------- infinities and NaN
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
