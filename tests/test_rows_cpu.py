"""Refusals of the entry points for any number of new tokens a sequence (pages from lengths, append of rows, attention of
rows): every check runs on the host before a device is asked for anything. Pointers here are numbers that nothing follows."""
import ctypes

import pytest

import mlxr
from test_batch_cpu import INVALID, KV_BAD, P, UNSUPPORTED, kv


def reserve(c=None, **over):
    a = dict(want=2 * P, free_pages=3 * P, n_free=4 * P, rows=100, len_out=P, n_free_out=4 * P, start=5 * P, count=6 * P, seq=7 * P, slot=8 * P, work=9 * P,
             work_bytes=1 << 40, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_reserve(ctypes.byref(c or kv(table=10 * P)), *a.values())


def append(c=None, **over):
    a = dict(qkv=P, row_stride=8 * 128, rows=7, seq=P, slot=P, positions=None, inv_freq=P, rope_scale=1.0, qn=None, kn=None, nH=4, rot_dim=128, traditional=0,
             eps=1e-6, q_out=P + 65536, q_type=0, q_stride=512, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_append_rows(ctypes.byref(c or kv()), *a.values())


def attention(c=None, **over):
    a = dict(start=P, count=P, rows=9, q=P, q_type=0, q_stride=512, nH=4, window=0, scale=0.1, out=P, out_stride=512, work=P, work_bytes=1 << 40, stream=None)
    a.update(over)
    return mlxr.lib.mlxr_k_paged_attention_rows(ctypes.byref(c or kv()), *a.values())


@pytest.mark.parametrize("field,value", KV_BAD)
def test_cache_descriptions_are_checked(field, value):
    c, want = kv(**{field: value}), (INVALID, UNSUPPORTED)
    assert append(c) in want and attention(c) in want and reserve(kv(**{"table": 10 * P, field: value})) in want
    assert mlxr.lib.mlxr_last_error()
    assert mlxr.lib.mlxr_k_paged_attention_rows_work(ctypes.byref(c), 4, 9, 0) < 0
    assert mlxr.lib.mlxr_k_paged_reserve_work(ctypes.byref(c), 9) < 0


def test_null_cache():
    lib = mlxr.lib
    assert lib.mlxr_k_paged_reserve(None, P, P, P, 1, P, P, P, P, P, P, P, 1 << 40, None) == INVALID
    assert lib.mlxr_k_paged_append_rows(None, P, 1024, 1, P, P, None, P, 1.0, None, None, 4, 128, 0, 1e-6, P, 0, 512, None) == INVALID
    assert lib.mlxr_k_paged_attention_rows(None, P, P, 1, P, 0, 512, 4, 0, 0.1, P, 512, P, 1 << 40, None) == INVALID
    assert lib.mlxr_k_paged_reserve_work(None, 1) < 0 and lib.mlxr_k_paged_attention_rows_work(None, 4, 1, 0) < 0


@pytest.mark.parametrize("over", [*({x: None} for x in ("want", "free_pages", "n_free", "len_out", "n_free_out", "start", "count", "seq", "slot", "work")),
                                  *({x: 11 * P + 2} for x in ("want", "free_pages", "n_free", "len_out", "n_free_out", "start", "count", "seq", "slot")),
                                  dict(rows=-1), dict(rows=(1 << 22) + 1), dict(work=9 * P + 16), dict(work_bytes=16),
                                  dict(want=P), dict(len_out=2 * P), dict(start=6 * P), dict(seq=8 * P), dict(slot=3 * P), dict(count=10 * P), dict(start=P),
                                  dict(n_free=3 * P), dict(n_free=8 * P), dict(n_free_out=5 * P), dict(free_pages=10 * P), dict(len_out=10 * P)])
def test_reserve_refuses(over):
    assert reserve(**over) == INVALID


@pytest.mark.parametrize("over", [dict(qkv=None), dict(q_out=None), dict(seq=None), dict(slot=None), dict(inv_freq=None), dict(qn=P), dict(kn=P), dict(nH=0), dict(nH=3),
                                  dict(nH=8192), dict(rot_dim=-2), dict(rot_dim=130), dict(rot_dim=63), dict(row_stride=1023), dict(q_stride=511), dict(q_out=P),
                                  dict(q_out=P, q_type=1, q_stride=1024), dict(qkv=P + 2), dict(q_out=P + 2), dict(q_out=P + 1, q_type=1), dict(positions=P + 1),
                                  dict(seq=P + 2), dict(slot=P + 3), dict(rows=0), dict(rows=(1 << 22) + 1), dict(q_type=2), dict(q_type=-1),
                                  dict(rope_scale=float("nan"))])
def test_append_refuses(over):
    assert append(**over) == INVALID


@pytest.mark.parametrize("over", [dict(start=None), dict(count=None), dict(q=None), dict(out=None), dict(nH=0), dict(nH=5), dict(window=-1), dict(scale=float("nan")),
                                  dict(scale=float("inf")), dict(scale=2.0 ** 127), dict(scale=-(2.0 ** 127)), dict(q_stride=508), dict(q_stride=514), dict(out_stride=510), dict(q=P + 4), dict(out=P + 8),
                                  dict(work=None), dict(work=P + 16), dict(work_bytes=16), dict(out_stride=516), dict(rows=0), dict(rows=(1 << 22) + 1),
                                  dict(q_type=2), dict(q_type=1, q_stride=516, out_stride=516), dict(start=P + 2), dict(count=P + 1)])
def test_attention_refuses(over):
    assert attention(**over) == INVALID


def test_slot_arrays_are_checked():
    for over in (dict(weight=P, slot_stride=127), dict(position=P, slot_stride=0), dict(weight=P + 2)):
        assert append(kv(**over)) == INVALID and attention(kv(**over)) == INVALID


def test_sizes_past_32_bits():
    lib = mlxr.lib
    big = kv(B=65535, max_len=1 << 24, table_stride=1 << 18, slot_stride=1 << 24)
    assert reserve(kv(table=10 * P, B=65535, max_len=1 << 24, table_stride=1 << 18)) == UNSUPPORTED
    assert lib.mlxr_k_paged_reserve_work(ctypes.byref(big), 1) < 0
    for B in (4095, 4096):   # 2^30 pages
        c = kv(table=10 * P, B=B, max_len=1 << 24, table_stride=1 << 18)
        assert (lib.mlxr_k_paged_reserve_work(ctypes.byref(c), 1) < 0) == (B == 4096)
    assert lib.mlxr_k_paged_reserve_work(ctypes.byref(kv(B=65535)), 1 << 22) >= 65536 * 16
    assert attention(kv(nKV=1), nH=4096, q_stride=4096 * 128, out_stride=4096 * 128, rows=1 << 22) == UNSUPPORTED
    assert lib.mlxr_k_paged_attention_rows_work(ctypes.byref(kv(nKV=1)), 4096, 1 << 22, 0) < 0
    assert lib.mlxr_k_paged_attention_rows_work(ctypes.byref(big), 8, 1 << 22, 1) > 0


@pytest.mark.skipif(mlxr.device_count() > 0, reason="what a call without a device says")
def test_good_arguments_without_a_device():
    assert reserve() == append() == attention() == -1
    assert reserve(len_out=11 * P, n_free_out=12 * P) == reserve(rows=0) == -1
    assert attention(q_type=1) == append(q_type=1) == append(q_out=P, q_stride=1024) == -1
    assert "GPU" in mlxr.lib.mlxr_last_error().decode()
