"""A paged key-value cache and the attention that reads it: thin calls into libtwmarlin_hip.so like those of quantize.py.  The
arrays and what the calls do with them are described in include/twmarlin.h.

Arrays are GpuTensors, or anything with .ptr, .dtype ("f32", "f16", "i32", "u8" for e4m3 codes) and .numel.  The library takes addresses: what an
array holds, how much, and whether a number fits 32 bits is checked here (ValueError), before the call.
"""
import array

import numpy as np

from . import _lib
from .fp8 import _DTYPES
from .quantize import _check

_CACHE_DTYPES = {"f16": _lib.F16, "u8": _lib.U8}


def _array(what, t, dtype, least):
    """The address of an array of `least` elements or more."""
    if t.dtype != dtype:
        raise ValueError("%s is %s, not %s" % (what, t.dtype, dtype))
    if getattr(t, "numel", least) < least:
        raise ValueError("%s has %d elements of %d" % (what, t.numel, least))
    return t.ptr


def _optional(what, t, dtype, least):
    return None if t is None else _array(what, t, dtype, least)


def _numbers(**numbers):
    for name, x in numbers.items():
        if x >> 32:   # (of a number below zero too)
            raise ValueError("%s: %d does not fit 32 bits" % (name, x))


def _last(rows, width, stride):
    """Elements up to the end of the last row."""
    return (rows - 1) * (stride or width) + width if rows else 0


# The calls look at everything in one expression, whose sizes are a little above what is needed where rows are apart, and only at what does not
# pass one by one (which alone would cost the smallest call 0.6 us of 4.3; so 0.2).
_ANY = 1 << 80   # elements of an array that does not say


class KvCache:
    """One layer's keys and values, [pages][kv_heads][page_tokens][head_dim] each, f16 or e4m3 codes (u8, with scales f32
    [kv_heads] or None).  The arrays stay the caller's; pages follows from their size."""

    def __init__(self, k, v, page_tokens, kv_heads, head_dim, k_scales=None, v_scales=None):
        _numbers(page_tokens=page_tokens, kv_heads=kv_heads, head_dim=head_dim)
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        pages = min(k.numel, v.numel) // max(1, page_tokens * kv_heads * head_dim)
        dtype = _CACHE_DTYPES.get(k.dtype, -1) if k.dtype == v.dtype else -1
        self.struct = _lib.KvCacheStruct(k.ptr, v.ptr, _optional("k_scales", k_scales, "f32", kv_heads), _optional("v_scales", v_scales, "f32", kv_heads),
                                         dtype, pages, page_tokens, kv_heads, head_dim)
        self.kv_heads, self.head_dim = kv_heads, head_dim


class KvSequences:
    """The sequences of a call: tables i32 [seqs][table_stride], lengths i32 [seqs], starts i32 [seqs + 1] (None: one row each)."""

    def __init__(self, tables, lengths, seqs, table_stride, starts=None):
        _numbers(seqs=seqs, table_stride=table_stride)
        self.tables, self.lengths, self.starts, self.seqs = tables, lengths, starts, seqs
        self.struct = _lib.KvSeqsStruct(_array("tables", tables, "i32", seqs * table_stride), _array("lengths", lengths, "i32", seqs),
                                        _optional("starts", starts, "i32", seqs + 1 if seqs else 0), seqs, table_stride)


def kv_append(device, cache, seqs, qkv, rows, q_heads, q_out, cos_sin=None, positions=0, rotary_dim=0, interleaved=False, qkv_stride=0):
    """Rotates q and k of `rows` fused rows [q | k | v] (f32 or f16), stores q as f16 rows and k and v in the cache."""
    dim, kind = cache.head_dim, qkv.dtype
    width, all_heads = q_heads * dim, q_heads * dim + 2 * cache.kv_heads * dim
    if ((rows | q_heads | positions | rotary_dim | qkv_stride) >> 32 or q_out.dtype != "f16" or getattr(q_out, "numel", _ANY) < rows * width
            or getattr(qkv, "numel", _ANY) < rows * (qkv_stride or all_heads)
            or cos_sin is not None and (cos_sin.dtype != "f32" or getattr(cos_sin, "numel", _ANY) < positions * rotary_dim)):
        _numbers(rows=rows, q_heads=q_heads, positions=positions, rotary_dim=rotary_dim, qkv_stride=qkv_stride)
        _array("qkv", qkv, kind, _last(rows, all_heads, qkv_stride))
        _array("q_out", q_out, "f16", rows * width)
        _optional("cos_sin", cos_sin, "f32", positions * rotary_dim)
    _check(device._l.twm_kv_append(device.handle, cache.struct, seqs.struct, qkv.ptr, _DTYPES.get(kind, -1), rows, qkv_stride, q_heads,
                                   None if cos_sin is None else cos_sin.ptr, positions, rotary_dim, 1 if interleaved else 0, q_out.ptr))


def _refuse(cache, q, rows, q_heads, out, window, q_stride, out_stride):
    _numbers(rows=rows, q_heads=q_heads, window=window, q_stride=q_stride, out_stride=out_stride)
    _array("q", q, "f16", _last(rows, q_heads * cache.head_dim, q_stride))
    _array("out", out, "f16", _last(rows, q_heads * cache.head_dim, out_stride))


def attention_decode(device, cache, seqs, q, q_heads, out, scale=None, window=0, q_stride=0, out_stride=0):
    """One new token per sequence: q f16 [seqs, q_heads * head_dim] -> out likewise; scale None: head_dim ** -0.5."""
    dim, rows = cache.head_dim, seqs.seqs
    if ((q_heads | window | q_stride | out_stride) >> 32 or q.dtype != "f16" or out.dtype != "f16"
            or getattr(q, "numel", _ANY) < rows * (q_stride or q_heads * dim) or getattr(out, "numel", _ANY) < rows * (out_stride or q_heads * dim)):
        _refuse(cache, q, rows, q_heads, out, window, q_stride, out_stride)
    scale = dim ** -0.5 if scale is None else scale
    _check(device._l.twm_attn_decode(device.handle, cache.struct, seqs.struct, q.ptr, q_stride, q_heads, scale, window, out.ptr, out_stride))


def attention_prompt(device, cache, seqs, q, rows, q_heads, out, scale=None, window=0, q_stride=0, out_stride=0):
    """Several new tokens per sequence, packed, each of which sees the tokens up to itself."""
    dim = cache.head_dim
    if ((rows | q_heads | window | q_stride | out_stride) >> 32 or q.dtype != "f16" or out.dtype != "f16"
            or getattr(q, "numel", _ANY) < rows * (q_stride or q_heads * dim) or getattr(out, "numel", _ANY) < rows * (out_stride or q_heads * dim)):
        _refuse(cache, q, rows, q_heads, out, window, q_stride, out_stride)
    scale = dim ** -0.5 if scale is None else scale
    _check(device._l.twm_attn_prompt(device.handle, cache.struct, seqs.struct, q.ptr, q_stride, rows, q_heads, scale, window, out.ptr, out_stride))


def kv_layers(caches):
    """A model's caches, one per layer, as kv_copy_pages() takes them; keeps them alive."""
    layers = (_lib.KvCacheStruct * len(caches))(*[c.struct for c in caches])
    layers.caches = list(caches)
    return layers


def _page_numbers(pages):
    """Page numbers for the library, an address and how many; what keeps them alive comes first."""
    try:
        if not isinstance(pages, np.ndarray):
            numbers = array.array("I", pages)
            return (numbers,) + numbers.buffer_info()
        if pages.ndim != 1 or pages.dtype.kind not in "iu":
            raise ValueError("kv_copy_pages: pages are a list of whole numbers")
        if pages.size == 0 or (pages.min() >= 0 and pages.max() <= 0xFFFFFFFF):
            numbers = np.ascontiguousarray(pages, np.uint32)
            return numbers, numbers.ctypes.data, numbers.size
    except OverflowError:
        pass
    raise ValueError("kv_copy_pages: a page's number is outside the pool")


def kv_copy_pages(device, layers, sources, targets):
    """Page sources[i] to page targets[i] in every layer (kv_layers())."""
    _from, source, count = _page_numbers(sources)
    _to, target, targeted = _page_numbers(targets)
    if count != targeted:
        raise ValueError("kv_copy_pages: as many targets as sources")
    _check(device._l.twm_kv_copy_pages(device.handle, layers, len(layers), source, target, count))
