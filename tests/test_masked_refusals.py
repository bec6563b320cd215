"""Refusals of the masked and paged operators that need no GPU: the C ABI's argument errors, and CPU tensors."""
import ctypes

import pytest
import torch

from ditto_b200 import _lib, ops


@pytest.fixture
def address():
    buf = ctypes.create_string_buffer(4096)
    address.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255            # never dereferenced by calls that are refused


def _masked(p, **changes):
    s = _lib.Strides3(64 * 2 * 32, 64 * 2, 64)
    a = dict(q=p, k=p, v=p, out=p, lse=p, q_strides=s, k_strides=s, v_strides=s, out_strides=s, batch=1, M=32, L=32, heads=2, kv_heads=2, head_dim=64,
             dtype=0, causal=1, scale=1.0, cap=0.0)
    return ctypes.byref(_lib.MaskedArgs(**{**a, **changes}))


def test_masked_argument_errors(address):
    lib, p = _lib.load(), address
    invalid = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=p + 2), dict(batch=0), dict(M=-1), dict(L=0), dict(scale=0.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan")), dict(causal=2), dict(heads=0), dict(kv_heads=0),
               dict(q_strides=_lib.Strides3(1, 64, 8)), dict(k_strides=_lib.Strides3(0, 64, 64)), dict(out_strides=_lib.Strides3(64, -64, 64)),
               dict(causal=0, prefix=p), dict(documents=p, M=33)]
    unsupported = [dict(dtype=7), dict(heads=3), dict(heads=256, kv_heads=1), dict(head_dim=60), dict(head_dim=136)]
    for changes, code in [(c, _lib.ERR_INVALID_ARG) for c in invalid] + [(c, _lib.ERR_UNSUPPORTED) for c in unsupported]:
        assert lib.ditto_b200_masked_attention(_masked(p, **changes), None, 0, None, None) == code, changes
        strides = _lib.Strides3(64 * 2 * 32, 64 * 2, 64)
        assert lib.ditto_b200_masked_attention_backward(_masked(p, **changes), p, strides, p, p, p, None, 0, None, None) == code, changes
    assert lib.ditto_b200_masked_attention(None, None, 0, None, None) == _lib.ERR_INVALID_ARG
    for lse, grad, dq in ((None, p, p), (p, None, p), (p, p, None), (p, p + 8, p)):
        assert lib.ditto_b200_masked_attention_backward(_masked(p, lse=lse), grad, _lib.Strides3(64, 64, 64), dq, p, p, None, 0, None,
                                                        None) == _lib.ERR_INVALID_ARG
    assert lib.ditto_b200_masked_workspace_bytes(_masked(p, M=0), 0) == 0


def test_paged_argument_errors(address):
    lib, p = _lib.load(), address
    base = dict(q=p, key_pages=p, value_pages=p, out=p, q_strides=_lib.Strides2(128, 64), out_strides=_lib.Strides2(128, 64),
                key_strides=_lib.Strides3(2048, 128, 64), value_strides=_lib.Strides3(2048, 128, 64), table=p, lengths=p, table_stride=4, tokens=3, batch=3,
                pages=10, page=16, table_cols=4, heads=2, kv_heads=2, head_dim=64, dtype=0, scale=1.0, cap=0.0)
    invalid = [dict(q=None), dict(key_pages=None), dict(out=None), dict(table=None), dict(lengths=None), dict(tokens=0), dict(batch=0), dict(pages=0),
               dict(page=0), dict(table_cols=0), dict(table_stride=0), dict(tokens=4), dict(value_pages=p + 1), dict(q_strides=_lib.Strides2(128, 4)),
               dict(key_strides=_lib.Strides3(2048, 128, 0)), dict(scale=-1.0), dict(cap=-1.0)]
    unsupported = [dict(page=24), dict(page=192), dict(page=8), dict(dtype=3), dict(heads=3), dict(head_dim=132), dict(table_cols=2 ** 30)]
    for changes, code in [(c, _lib.ERR_INVALID_ARG) for c in invalid] + [(c, _lib.ERR_UNSUPPORTED) for c in unsupported]:
        assert lib.ditto_b200_paged_attention(ctypes.byref(_lib.PagedArgs(**{**base, **changes})), None, 0, None, None) == code, changes
    append = dict(keys=p, values=p, key_pages=p, value_pages=p, k_strides=_lib.Strides2(128, 64), v_strides=_lib.Strides2(128, 64),
                  key_strides=_lib.Strides3(2048, 128, 64), value_strides=_lib.Strides3(2048, 128, 64), table=p, lengths=p, table_stride=4, tokens=3, batch=3,
                  pages=10, page=5, table_cols=4, kv_heads=2, head_dim=64)
    for changes, code in ((dict(keys=None), -1), (dict(value_pages=None), -1), (dict(table=None), -1), (dict(tokens=4), -1), (dict(page=0), -1),
                          (dict(kv_heads=0), -1), (dict(keys=p + 4), -1), (dict(k_strides=_lib.Strides2(128, 1)), -1), (dict(head_dim=12), -2)):
        assert lib.ditto_b200_cache_append(ctypes.byref(_lib.AppendArgs(**{**append, **changes})), None, None) == code, changes


def test_cache_argument_errors(address):
    lib, p = _lib.load(), address
    base = (ctypes.c_void_p * 2)(p, p)
    pools = dict(base=ctypes.cast(base, ctypes.c_void_p), count=2, pages=10, page_bytes=64, stride_bytes=64)
    tables = dict(table=p, lengths=p, references=p, stride=4, sequences=3, cols=4, page=16, pages=10)
    good_p, good_t = _lib.PoolsArgs(**pools), _lib.TablesArgs(**tables)
    bad_base = (ctypes.c_void_p * 2)(p, p + 8)
    for changes in (dict(base=None), dict(count=0), dict(pages=0), dict(page_bytes=0), dict(page_bytes=24), dict(stride_bytes=48), dict(stride_bytes=72),
                    dict(base=ctypes.cast(bad_base, ctypes.c_void_p)), dict(pages=11)):
        bad = ctypes.byref(_lib.PoolsArgs(**{**pools, **changes}))
        if "pages" not in changes or changes["pages"] == 0:
            assert lib.ditto_b200_cache_copy(bad, p, p, 1, None, None) == _lib.ERR_INVALID_ARG, changes
        assert lib.ditto_b200_cache_fork(bad, ctypes.byref(good_t), p, p, 1, p, 4096, None, None) == _lib.ERR_INVALID_ARG, changes
        assert lib.ditto_b200_cache_compact(bad, ctypes.byref(good_t), p, 4, p, p, 4096, None, None) == _lib.ERR_INVALID_ARG, changes
    for changes in (dict(table=None), dict(references=None), dict(sequences=0), dict(cols=0), dict(pages=0), dict(stride=3)):
        bad = ctypes.byref(_lib.TablesArgs(**{**tables, **changes}))
        assert lib.ditto_b200_cache_free(bad, p, 1, None, None) == _lib.ERR_INVALID_ARG, changes
        assert lib.ditto_b200_cache_reserve(bad, p, p, 4096, None, None) == _lib.ERR_INVALID_ARG, changes
        assert lib.ditto_b200_cache_fork(ctypes.byref(good_p), bad, p, p, 1, p, 4096, None, None) == _lib.ERR_INVALID_ARG, changes
    for changes in (dict(page=0), dict(lengths=None)):
        bad = ctypes.byref(_lib.TablesArgs(**{**tables, **changes}))
        assert lib.ditto_b200_cache_reserve(bad, p, p, 4096, None, None) == _lib.ERR_INVALID_ARG, changes
    t = ctypes.byref(good_t)
    assert lib.ditto_b200_cache_reserve(t, p, p, 8, None, None) == _lib.ERR_WORKSPACE
    assert lib.ditto_b200_cache_fork(ctypes.byref(good_p), t, p, p, 2, p, 8, None, None) == _lib.ERR_WORKSPACE
    assert lib.ditto_b200_cache_compact(ctypes.byref(good_p), t, p, 4, p, None, 0, None, None) == _lib.ERR_WORKSPACE
    assert lib.ditto_b200_cache_compact(ctypes.byref(good_p), t, p, 3, p, p, 4096, None, None) == _lib.ERR_INVALID_ARG
    assert lib.ditto_b200_cache_free(t, None, 1, None, None) == _lib.ERR_INVALID_ARG
    assert lib.ditto_b200_cache_free(t, p, 0, None, None) == _lib.ERR_INVALID_ARG
    assert lib.ditto_b200_cache_workspace_bytes(t, 100) >= 301 * 4


def test_cpu_tensors():
    x, table, lengths = torch.zeros(2, 16, 4, 64, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.masked_attention(x, x, x), lambda: ops.masked_attention_backward(x, x, x, x, x, x[..., 0].float()),
                 lambda: ops.paged_attention(x[:, 0], x, x, table, lengths), lambda: ops.cache_append(x[:, 0], x[:, 0], x, x, table, lengths),
                 lambda: ops.cache_copy([x], lengths, lengths), lambda: ops.cache_reserve(table, lengths, lengths, lengths, 16),
                 lambda: ops.cache_fork([x], table, lengths, lengths, lengths, lengths, 16), lambda: ops.cache_free(table, lengths, lengths, lengths),
                 lambda: ops.cache_compact([x], table, lengths)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
