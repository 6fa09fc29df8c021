"""The batch's decode step at its edges: appends to pages outside the pool. Helpers and tolerances are those of
test_batch_gpu."""
import numpy as np
import pytest

from test_batch_gpu import Cache, run_append, same

pytestmark = pytest.mark.gpu


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
