"""A paged key-value cache and the attention that reads it: thin calls into libtwmarlin_hip.so like those of quantize.py.  The
arrays and what the calls do with them are described in include/twmarlin.h.

Arrays are GpuTensors, or anything with .ptr, .dtype ("f32", "f16", "i32", "u8" for e4m3 codes) and .numel.
"""
import array

import numpy as np

from . import _lib
from .fp8 import _dtype, _ptr
from .quantize import _check

_CACHE_DTYPES = {"f16": _lib.F16, "u8": _lib.U8}


class KvCache:
    """One layer's keys and values, [pages][kv_heads][page_tokens][head_dim] each, f16 or e4m3 codes (u8, with scales f32
    [kv_heads] or None).  The arrays stay the caller's; pages follows from their size."""

    def __init__(self, k, v, page_tokens, kv_heads, head_dim, k_scales=None, v_scales=None):
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        pages = min(k.numel, v.numel) // max(1, page_tokens * kv_heads * head_dim)
        dtype = _CACHE_DTYPES.get(k.dtype, -1) if k.dtype == v.dtype else -1
        self.struct = _lib.KvCacheStruct(k.ptr, v.ptr, _ptr(k_scales), _ptr(v_scales), dtype, pages, page_tokens, kv_heads, head_dim)
        self.head_dim = head_dim


class KvSequences:
    """The sequences of a call: tables i32 [seqs][table_stride], lengths i32 [seqs], starts i32 [seqs + 1] (None: one row each)."""

    def __init__(self, tables, lengths, seqs, table_stride, starts=None):
        self.tables, self.lengths, self.starts = tables, lengths, starts
        self.struct = _lib.KvSeqsStruct(tables.ptr, lengths.ptr, _ptr(starts), seqs, table_stride)


def kv_append(device, cache, seqs, qkv, rows, q_heads, q_out, cos_sin=None, positions=0, rotary_dim=0, interleaved=False, qkv_stride=0):
    """Rotates q and k of `rows` fused rows [q | k | v] (f32 or f16), stores q as f16 rows and k and v in the cache."""
    _check(device._l.twm_kv_append(device.handle, cache.struct, seqs.struct, qkv.ptr, _dtype(qkv), rows, qkv_stride, q_heads, _ptr(cos_sin),
                                   positions, rotary_dim, int(interleaved), q_out.ptr))


def attention_decode(device, cache, seqs, q, q_heads, out, scale=None, window=0, q_stride=0, out_stride=0):
    """One new token per sequence: q f16 [seqs, q_heads * head_dim] -> out likewise; scale None: head_dim ** -0.5."""
    scale = cache.head_dim ** -0.5 if scale is None else scale
    _check(device._l.twm_attn_decode(device.handle, cache.struct, seqs.struct, q.ptr, q_stride, q_heads, scale, window, out.ptr, out_stride))


def attention_prompt(device, cache, seqs, q, rows, q_heads, out, scale=None, window=0, q_stride=0, out_stride=0):
    """Several new tokens per sequence, packed, each of which sees the tokens up to itself."""
    scale = cache.head_dim ** -0.5 if scale is None else scale
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
