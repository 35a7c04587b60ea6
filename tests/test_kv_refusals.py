"""What the calls of the paged key-value cache refuse, on the CPU: the checks come before anything touches a device, so a context that
is nothing but zeros will do."""
import ctypes as C

import numpy as np
import pytest

import tensorwarp_amd as T
from tensorwarp_amd import _lib

A, B = 0x1000, 0x2000   # addresses that are never read: every call here is refused, or has nothing to do


@pytest.fixture()
def ctx():
    return C.cast(C.create_string_buffer(1 << 14), C.c_void_p)


def cache(**kw):
    c = dict(k_dev=A, v_dev=A, k_scales_dev=None, v_scales_dev=None, dtype=_lib.F16, pages=10, page_tokens=16, kv_heads=2, head_dim=64)
    c.update(kw)
    return _lib.KvCacheStruct(**c)


def seqs(**kw):
    s = dict(tables_dev=A, lengths_dev=A, starts_dev=A, seqs=3, table_stride=4)
    s.update(kw)
    return _lib.KvSeqsStruct(**s)


def append(ctx, c=None, s=None, qkv=A, dtype=_lib.F32, rows=3, stride=0, heads=4, cos_sin=A, positions=8, rotary=64, q=B):
    return _lib.load().twm_kv_append(ctx, c or cache(), s or seqs(), qkv, dtype, rows, stride, heads, cos_sin, positions, rotary, 0, q)


def decode(ctx, c=None, s=None, q=A, stride=0, heads=4, scale=0.125, window=0, out=B, out_stride=0):
    return _lib.load().twm_attn_decode(ctx, c or cache(), s or seqs(), q, stride, heads, scale, window, out, out_stride)


def prompt(ctx, c=None, s=None, q=A, stride=0, rows=3, heads=4, scale=0.125, window=0, out=B, out_stride=0):
    return _lib.load().twm_attn_prompt(ctx, c or cache(), s or seqs(), q, stride, rows, heads, scale, window, out, out_stride)


def copy(ctx, caches=None, sources=(1,), targets=(2,), count=None):
    caches = [cache()] if caches is None else caches
    array = (_lib.KvCacheStruct * len(caches))(*caches)
    pages = [(C.c_uint32 * len(x))(*x) for x in (sources, targets)]
    return _lib.load().twm_kv_copy_pages(ctx, array, len(caches) if count is None else count, pages[0], pages[1], len(sources))


def refused(rc, code, text):
    assert rc == code, (rc, _lib.load().twm_last_error())
    assert text in _lib.load().twm_last_error(), _lib.load().twm_last_error()
    assert _lib.load().twm_last_error_kind() == 0


CALLS = [append, decode, prompt]


def test_null_contexts_and_descriptions(ctx):
    for call in CALLS + [copy]:
        refused(call(None), _lib.INVALID_HANDLE, b"null context")
    lib = _lib.load()
    refused(lib.twm_attn_decode(ctx, None, seqs(), A, 0, 4, 0.1, 0, B, 0), _lib.INVALID_HANDLE, b"null cache")
    refused(lib.twm_attn_decode(ctx, cache(), None, A, 0, 4, 0.1, 0, B, 0), _lib.INVALID_HANDLE, b"null sequences")
    refused(lib.twm_kv_copy_pages(ctx, None, 1, A, A, 1), _lib.INVALID_HANDLE, b"null cache")
    refused(lib.twm_kv_copy_pages(ctx, cache(), 1, None, A, 1), _lib.INVALID_HANDLE, b"null pointer")


@pytest.mark.parametrize("call", CALLS)
def test_caches(ctx, call):
    for dtype in (_lib.F32, _lib.I32, -1):
        refused(call(ctx, c=cache(dtype=dtype)), _lib.UNSUPPORTED_OP, b"f16 or e4m3")
    for dim in (0, 32, 80, 96, 512):
        refused(call(ctx, c=cache(head_dim=dim)), _lib.UNSUPPORTED_OP, b"64, 128 and 256")
    for page in (0, 1, 8, 24, 48, 512):
        refused(call(ctx, c=cache(page_tokens=page)), _lib.UNSUPPORTED_OP, b"16, 32, 64, 128 and 256")
    for heads in (0, 1025):
        refused(call(ctx, c=cache(kv_heads=heads)), _lib.SHAPE_ERROR, b"key-value heads")
    refused(call(ctx, c=cache(pages=(1 << 28) + 1)), _lib.SHAPE_ERROR, b"beyond 2^28")
    for name in ("k_dev", "v_dev"):
        refused(call(ctx, c=cache(**{name: None})), _lib.INVALID_HANDLE, b"null pointer")
        refused(call(ctx, c=cache(**{name: A + 8})), _lib.SHAPE_ERROR, b"16-byte aligned")
    for name in ("k_scales_dev", "v_scales_dev"):
        refused(call(ctx, c=cache(dtype=_lib.U8, **{name: A + 2})), _lib.SHAPE_ERROR, b"aligned to its elements")


@pytest.mark.parametrize("call", CALLS)
def test_sequences(ctx, call):
    refused(call(ctx, s=seqs(seqs=(1 << 20) + 1)), _lib.SHAPE_ERROR, b"sequences are beyond 2^20")
    refused(call(ctx, s=seqs(table_stride=(1 << 26) + 1)), _lib.SHAPE_ERROR, b"2^30 tokens")
    for name in ("tables_dev", "lengths_dev"):
        refused(call(ctx, s=seqs(**{name: None})), _lib.INVALID_HANDLE, b"null pointer")
        refused(call(ctx, s=seqs(**{name: A + 2})), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(call(ctx, s=seqs(starts_dev=A + 1)), _lib.SHAPE_ERROR, b"aligned to its elements")
    for heads in (0, 1, 3, 1026):
        refused(call(ctx, heads=heads), _lib.SHAPE_ERROR, b"query heads")
    assert call(ctx, s=seqs(seqs=0)) == _lib.OK


def test_rows(ctx):
    refused(prompt(ctx, s=seqs(starts_dev=None)), _lib.INVALID_HANDLE, b"null pointer")
    for call in (append, prompt):
        refused(call(ctx, rows=(1 << 20) + 1), _lib.SHAPE_ERROR, b"rows are beyond 2^20")
        assert call(ctx, rows=0) == _lib.OK
    for call in (decode, prompt):
        for scale in (0.0, -1.0, float("nan"), float("inf")):
            refused(call(ctx, scale=scale), _lib.SHAPE_ERROR, b"scale")
        refused(call(ctx, stride=255), _lib.SHAPE_ERROR, b"row stride")
        refused(call(ctx, out_stride=255), _lib.SHAPE_ERROR, b"row stride")
        for name in ("q", "out"):
            refused(call(ctx, **{name: None}), _lib.INVALID_HANDLE, b"null pointer")
            refused(call(ctx, **{name: A + 1}), _lib.SHAPE_ERROR, b"aligned to its elements")


def test_append(ctx):
    refused(append(ctx, dtype=_lib.U8), _lib.UNSUPPORTED_OP, b"f16 or f32")
    refused(append(ctx, s=seqs(starts_dev=None), rows=4), _lib.SHAPE_ERROR, b"one row each")
    for rotary in (8, 40, 80, 128):
        refused(append(ctx, rotary=rotary), _lib.SHAPE_ERROR, b"rotary_dim")
    refused(append(ctx, stride=511), _lib.SHAPE_ERROR, b"row stride")
    for name in ("qkv", "cos_sin", "q"):
        refused(append(ctx, **{name: None}), _lib.INVALID_HANDLE, b"null pointer")
    refused(append(ctx, qkv=A + 2), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(append(ctx, qkv=A + 1, dtype=_lib.F16), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(append(ctx, cos_sin=A + 2), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(append(ctx, q=A + 1), _lib.SHAPE_ERROR, b"aligned to its elements")


def test_copies(ctx):
    refused(copy(ctx, sources=(10,)), _lib.SHAPE_ERROR, b"of 10")
    refused(copy(ctx, targets=(10,)), _lib.SHAPE_ERROR, b"of 10")
    refused(copy(ctx, sources=(1, 2), targets=(3, 3)), _lib.SHAPE_ERROR, b"page 3 is a target and named again")
    refused(copy(ctx, sources=(1, 2), targets=(2, 5)), _lib.SHAPE_ERROR, b"page 2 is a target and named again")
    refused(copy(ctx, sources=(4,), targets=(4,)), _lib.SHAPE_ERROR, b"page 4 is a target and named again")
    refused(copy(ctx, sources=(1, 2), targets=(2, 1)), _lib.SHAPE_ERROR, b"named again")
    for other in (cache(pages=11), cache(dtype=_lib.U8), cache(page_tokens=32), cache(kv_heads=3), cache(head_dim=128)):
        refused(copy(ctx, caches=[cache(), other]), _lib.SHAPE_ERROR, b"one shape")
    refused(copy(ctx, caches=[cache(), cache(k_dev=None)]), _lib.INVALID_HANDLE, b"null pointer")
    refused(copy(ctx, count=(1 << 20) + 1), _lib.SHAPE_ERROR, b"beyond 2^20")
    assert copy(ctx, sources=(), targets=()) == _lib.OK and copy(ctx, caches=[]) == _lib.OK


@pytest.mark.parametrize("page", [-1, 1 << 32, -(1 << 32), 1 << 40])
def test_page_numbers_that_32_bits_do_not_hold(page):
    # (refused before anything is asked of a device)
    layers = T.kv_layers([])
    for sources, targets in (([page], [1]), ([1], [page]), (np.array([0, page]), np.array([1, 2]))):
        with pytest.raises(ValueError, match="outside the pool"):
            T.kv_copy_pages(None, layers, sources, targets)


def test_what_is_no_list_of_pages():
    layers = T.kv_layers([])
    for sources, targets in ((np.zeros((1, 1), np.int32), [1]), (np.array([0.5]), [1]), ([0], np.array([1.0])), ([0, 1], [2]), (np.arange(2), [5])):
        with pytest.raises(ValueError):
            T.kv_copy_pages(None, layers, sources, targets)
    with pytest.raises(TypeError):
        T.kv_copy_pages(None, layers, [0.5], [1])
