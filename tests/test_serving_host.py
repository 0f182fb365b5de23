"""Refusals of the paged-cache serving operators that need no GPU: the C entries'
argument checks run before any CUDA call, the Python ones before the C entry."""
import ctypes as C

import pytest
import torch

from lama32_mojo_b200 import _lib, ops

ONE = 4096  # an address no check looks behind


def pages(**kw):
    d = dict(k=ONE, v=ONE, k_scale=ONE, v_scale=ONE, num_pages=4, n_kv=2, page=32, head_dim=64)
    d.update(kw)
    return C.byref(_lib.q8_kv8_pages(*[d[f] for f, _ in _lib.q8_kv8_pages._fields_]))


def refused(status, word):
    assert status == _lib.Q8_ERR_ARG
    assert word in _lib.last_error()


def test_kv8_entries_refuse():
    L = _lib.lib()

    def append(k=ONE, ld=128, dtype=0, rows=1, starts=ONE, ctx=ONE, S=1, kv=None, table=ONE, width=1):
        return L.q8op_kv8_append(k, ld, k, ld, dtype, rows, starts, ctx, S, kv or pages(), table, width, None)

    def attend(q=ONE, ld=256, dtype=0, rows=1, heads=4, kv=None, width=1, out=ONE, S=1):
        return L.q8op_kv8_attention(q, ld, dtype, rows, ONE, ONE, S, heads, kv or pages(), ONE, width, out, ld, ONE, 1 << 30, None)

    refused(append(k=None), "rows need")
    refused(append(ld=127), "rows need")
    refused(append(dtype=3), "dtype")
    refused(append(starts=None), "null")
    refused(append(ctx=None), "null")
    refused(append(table=None), "null")
    refused(append(rows=-1), "shape")
    refused(append(S=-1), "shape")
    refused(append(width=0), "shape")
    refused(append(width=1 << 27), "positions")
    refused(attend(width=1 << 27), "positions")
    for bad in (dict(page=24), dict(page=0), dict(head_dim=96), dict(num_pages=0), dict(n_kv=0), dict(k=None),
                dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=ONE + 8)):
        assert append(kv=pages(**bad)) == _lib.Q8_ERR_ARG
        assert attend(kv=pages(**bad)) == _lib.Q8_ERR_ARG
    assert L.q8op_kv8_append(ONE, 128, ONE, 128, 0, 1, ONE, ONE, 1, None, ONE, 1, None) == _lib.Q8_ERR_ARG
    refused(attend(heads=3), "heads")
    refused(attend(heads=0), "heads")
    refused(attend(ld=255), "rows need")
    refused(attend(out=None), "rows need")
    refused(attend(dtype=-1), "dtype")
    assert append(rows=0) == attend(rows=0) == append(S=0) == attend(S=0) == _lib.Q8_OK
    refused(L.q8op_kv8_read(pages(), ONE, ONE, 1, ONE, 1, None, ONE, 1, None), "null")
    refused(L.q8op_kv8_read(pages(), ONE, ONE, 1, ONE, 1, ONE + 4, ONE, 1, None), "unaligned")
    refused(L.q8op_kv8_read(pages(), ONE, None, 1, ONE, 1, ONE, ONE, 1, None), "null")


def test_page_entries_refuse():
    L = _lib.lib()

    def trunc(S=1, width=1, num=4, page=16, table=ONE, refs=ONE, ctx=ONE, new=ONE):
        return L.q8op_kv_truncate(table, S, width, ctx, refs, num, page, new, None)

    for bad in (dict(S=8193), dict(S=-1), dict(width=0), dict(num=0), dict(page=0), dict(table=None),
                dict(refs=None), dict(ctx=None), dict(new=None), dict(S=8000, width=1 << 20),
                dict(width=1 << 20, page=1 << 12)):
        refused(trunc(**bad), "q8op_kv_truncate")
    assert trunc(S=0) == _lib.Q8_OK
    refused(L.q8op_kv_fork(ONE, 1, 1, ONE, ONE, 4, 16, ONE, ONE, 8193, None), "pairs")
    refused(L.q8op_kv_fork(ONE, 1, 1, ONE, ONE, 4, 16, None, ONE, 1, None), "null")
    assert L.q8op_kv_fork(ONE, 1, 1, ONE, ONE, 4, 16, None, None, 0, None) == _lib.Q8_OK
    refused(L.q8op_kv_reserve(ONE, 1, 1, ONE, ONE, 4, 16, ONE, ONE, ONE, None, ONE, None), "null")
    refused(L.q8op_kv_compact(ONE, 1, 1, ONE, 4, ONE, ONE, None, None), "null")
    arr, size = (C.c_void_p * 1)(ONE), (C.c_int64 * 1)(64)
    refused(L.q8op_kv_copy_pages(arr, size, 65, 4, ONE, ONE, 1, None), "pools")
    refused(L.q8op_kv_copy_pages(arr, size, 1, 0, ONE, ONE, 1, None), "shape")
    refused(L.q8op_kv_copy_pages(arr, size, 1, 4, None, ONE, 1, None), "null")
    refused(L.q8op_kv_copy_pages((C.c_void_p * 1)(None), size, 1, 4, ONE, ONE, 1, None), "pool 0")
    refused(L.q8op_kv_copy_pages(arr, (C.c_int64 * 1)(0), 1, 4, ONE, ONE, 1, None), "pool 0")
    assert L.q8op_kv_copy_pages(arr, size, 1, 4, ONE, ONE, 0, None) == _lib.Q8_OK


def test_speculative_entries_refuse():
    L = _lib.lib()
    refused(L.q8op_probs(ONE, 1, 10, 9, 1.0, ONE, 10, None), "shape")
    refused(L.q8op_probs(ONE, 1, 10, 10, 1.0, ONE, 9, None), "shape")
    refused(L.q8op_probs(ONE, 1, 0, 10, 1.0, ONE, 10, None), "shape")
    refused(L.q8op_probs(ONE, 1, 10, 10, float("nan"), ONE, 10, None), "NaN")
    refused(L.q8op_probs(None, 1, 10, 10, 1.0, ONE, 10, None), "null")
    assert L.q8op_probs(None, 0, 10, 10, 1.0, None, 10, None) == _lib.Q8_OK
    refused(L.q8op_verify(ONE, 9, ONE, 10, 1, ONE, ONE, 1, 1, 10, ONE, ONE, ONE, None), "shape")
    refused(L.q8op_verify(ONE, 10, ONE, 9, 1, ONE, ONE, 1, 1, 10, ONE, ONE, ONE, None), "shape")
    refused(L.q8op_verify(ONE, 10, ONE, 10, 1, ONE, None, 1, 1, 10, ONE, ONE, ONE, None), "null")
    refused(L.q8op_verify(None, 10, ONE, 10, 1, ONE, ONE, 1, 1, 10, ONE, ONE, ONE, None), "null")
    assert L.q8op_verify(None, 10, None, 10, 0, None, None, 0, 0, 10, None, None, None, None) == _lib.Q8_OK
    refused(L.q8op_rope_kv_append(ONE, 512, 1, ONE, None, 4, 2, 64, ONE, None, None, 1e-6, ONE, ONE, 16, ONE, 1, None),
            "null")


def test_python_entries_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.KV8Pages(*(torch.zeros((1, 1, 16, 64), dtype=torch.int8),) * 2, *(torch.zeros((1, 1, 1)),) * 2)
    for call in (lambda: ops.kv_truncate(t, i[:1], i, 16, i[:1]), lambda: ops.kv_fork(t, i[:1], i, 16, i, i),
                 lambda: ops.kv_reserve(t, i[:1], i, 16, i[:1]), lambda: ops.kv_compact(t, i),
                 lambda: ops.kv_copy_pages([torch.zeros((2, 4))], i, i), lambda: ops.probs(torch.zeros((1, 4)), 1.0),
                 lambda: ops.verify(torch.zeros((1, 4)), None, i[:1], i, torch.zeros(1)),
                 lambda: ops.kv8_attention(torch.zeros((1, 64)), i, i[:1], 1, None, t),
                 lambda: ops.rope(torch.zeros((1, 256)), i[:1], 2, 1, 64, torch.zeros(32))):
        with pytest.raises(ValueError):
            call()
    assert ops.kv_copy_pages([], i, i) is None
