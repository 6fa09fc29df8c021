"""Refusals of the batch decode entry points (paged append, attention, eviction, sampling of rows): every check runs on
the host before a device is asked for anything, so none needs one. Pointers here are numbers that nothing follows."""
import ctypes

import numpy as np
import pytest

import mlxr

P = 1 << 20          # stands for a device address (aligned, never followed)
INVALID, UNSUPPORTED = -10, -4


def kv(**over):
    a = dict(k=P, v=P, table=P, len=P, weight=None, position=None, n_pages=4, table_stride=2, slot_stride=128, max_len=128, B=2, nKV=2, D=128, st=0)
    a.update(over)
    return mlxr.PagedKV(**a)


def append(c=None, **over):
    a = dict(qkv=P, row_stride=8 * 128, inv_freq=P, qn=None, kn=None, nH=4, rot_dim=128, traditional=0, positions=None, eps=1e-6, q_out=P + 65536,
             q_stride=512, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_append(ctypes.byref(c or kv()), *a.values())


def attention(c=None, **over):
    a = dict(q=P, q_stride=512, nH=4, window=0, scale=0.1, out=P, out_stride=512, weight_in=None, decay=1.0, work=P, work_bytes=1 << 40, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_attention(ctypes.byref(c or kv()), *a.values())


def evict(src=None, dst=None, **over):
    a = dict(budget=100, sink=4, window=32, work=P, work_bytes=1 << 40, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_evict(ctypes.byref(src or kv(weight=P)), ctypes.byref(dst or kv(table=2 * P, len=2 * P, weight=2 * P)), *a.values())


def sample(**over):
    a = dict(logits=P, rows=2, V=100, stride=100, temperature=P, top_k=None, top_p=None, min_p=None, u=P, tokens=P, status=None, work=P,
             work_bytes=1 << 40, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_sample_rows(*a.values())


KV_BAD = [("k", None), ("v", None), ("table", None), ("len", None), ("D", 96), ("D", 256), ("st", 2), ("st", -1), ("B", 0), ("B", 65536), ("nKV", 0),
          ("nKV", 2048), ("n_pages", 0), ("table_stride", 0), ("max_len", 0), ("max_len", 129), ("max_len", 1 << 25), ("k", P + 8), ("v", P + 2), ("len", P + 2), ("table", P + 1)]


@pytest.mark.parametrize("field,value", KV_BAD)
def test_cache_descriptions_are_checked(field, value):
    c = kv(**{field: value})
    want = (INVALID, UNSUPPORTED)
    assert append(c) in want and attention(c) in want
    assert evict(kv(weight=P, **{field: value})) in want
    assert mlxr.lib.mlxr_last_error()
    assert mlxr.lib.mlxr_k_paged_attention_work(ctypes.byref(c), 4) < 0
    assert mlxr.lib.mlxr_k_paged_evict_work(ctypes.byref(c), 100) < 0


@pytest.mark.parametrize("over", [dict(weight=P, slot_stride=127), dict(position=P, slot_stride=0), dict(weight=P + 2)])
def test_slot_arrays_are_checked(over):
    assert append(kv(**over)) == INVALID and attention(kv(**over)) == INVALID


def test_null_cache():
    lib = mlxr.lib
    assert lib.mlxr_k_paged_append(None, P, 1024, P, None, None, 4, 128, 0, None, 1e-6, P, 512, None) == INVALID
    assert lib.mlxr_k_paged_attention(None, P, 512, 4, 0, 0.1, P, 512, None, 1.0, P, 1 << 40, None) == INVALID
    assert lib.mlxr_k_paged_evict(None, None, 100, 4, 32, P, 1 << 40, None) == INVALID
    assert lib.mlxr_k_paged_attention_work(None, 4) < 0 and lib.mlxr_k_paged_evict_work(None, 4) < 0


@pytest.mark.parametrize("over", [dict(qkv=None), dict(q_out=None), dict(inv_freq=None), dict(qn=P), dict(kn=P), dict(nH=0), dict(nH=3), dict(nH=8192),
                                  dict(rot_dim=-2), dict(rot_dim=130), dict(rot_dim=63), dict(row_stride=1023), dict(q_stride=511),
                                  dict(q_out=P), dict(qkv=P + 2), dict(positions=P + 1)])
def test_append_refuses(over):
    assert append(**over) == INVALID


@pytest.mark.parametrize("over", [dict(q=None), dict(out=None), dict(nH=0), dict(nH=5), dict(window=-1), dict(scale=float("nan")), dict(decay=float("nan")),
                                  dict(weight_in=P), dict(q_stride=508), dict(q_stride=514), dict(out_stride=510), dict(q=P + 4), dict(out=P + 8),
                                  dict(work=None), dict(work=P + 16), dict(work_bytes=16), dict(q=P, out=P, q_stride=512, out_stride=516)])
def test_attention_refuses(over):
    assert attention(**over) == INVALID


@pytest.mark.parametrize("over", [dict(budget=0), dict(budget=-1), dict(sink=-1), dict(window=-1), dict(sink=50, window=51), dict(sink=2**31 - 1, window=2**31 - 1),
                                  dict(work=None), dict(work=P + 128), dict(work_bytes=8)])
def test_evict_refuses(over):
    assert evict(**over) == INVALID


@pytest.mark.parametrize("src,dst", [(dict(weight=None), {}), ({}, dict(B=3)), ({}, dict(nKV=1)), ({}, dict(D=64)), ({}, dict(st=1)), ({}, dict(position=P)),
                                     ({}, dict(max_len=99)), ({}, dict(len=P)), ({}, dict(table=P)), ({}, dict(weight=P))])
def test_evict_refuses_pairs(src, dst):
    a, b = dict(weight=P), dict(table=2 * P, len=2 * P, weight=2 * P)
    a.update(src)
    b.update(dst)
    assert evict(kv(**a), kv(**b)) == INVALID


@pytest.mark.parametrize("over", [dict(logits=None), dict(temperature=None), dict(u=None), dict(tokens=None), dict(rows=0), dict(rows=65536), dict(V=0),
                                  dict(V=(1 << 20) + 1, stride=1 << 21), dict(stride=99), dict(logits=P + 2), dict(top_k=P + 2), dict(status=P + 2),
                                  dict(work=None), dict(work=P + 8), dict(work_bytes=4)])
def test_sample_rows_refuses(over):
    assert sample(**over) == INVALID


def test_work_sizes():
    lib = mlxr.lib
    for f in (lambda: lib.mlxr_k_sample_rows_work(0, 10), lambda: lib.mlxr_k_sample_rows_work(1, 0), lambda: lib.mlxr_k_sample_rows_work(70000, 10),
              lambda: lib.mlxr_k_paged_attention_work(ctypes.byref(kv()), 3), lambda: lib.mlxr_k_paged_evict_work(ctypes.byref(kv()), 0)):
        assert f() < 0
    assert lib.mlxr_k_sample_rows_work(256, 151936) > 0
    # large batches: sizes are counted in 64 bits
    big = kv(B=4096, nKV=8, max_len=131072, table_stride=2048, slot_stride=131072, weight=P)
    assert lib.mlxr_k_paged_evict_work(ctypes.byref(big), 131072) >= 4096 * 8 * 131072 * 4
    assert lib.mlxr_k_paged_attention_work(ctypes.byref(big), 32) > 0


def test_batches_too_large_to_count():
    """More pages or heads than the kernels count in 32 bits are refused, whatever the workspace."""
    c = kv(B=60000, nKV=8, max_len=1 << 24, table_stride=1 << 18, slot_stride=1 << 24)
    assert attention(c, nH=8, q_stride=1024, out_stride=1024) == UNSUPPORTED
    assert mlxr.lib.mlxr_k_paged_attention_work(ctypes.byref(c), 8) < 0
    c = kv(B=65535, nKV=1024, table_stride=1, slot_stride=64, max_len=64)
    assert append(c, nH=1024, row_stride=3 * 1024 * 128, q_stride=1024 * 128) == UNSUPPORTED


@pytest.mark.skipif(mlxr.device_count() > 0, reason="what a call without a device says")
def test_good_arguments_without_a_device():
    assert append() == attention() == evict() == sample() == -1
    assert "GPU" in mlxr.lib.mlxr_last_error().decode()
